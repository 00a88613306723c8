"""What the roundings of 8-bit cache attention may amount to, kernel by kernel, with bounds from what a row sees (kv8_bound)."""
import pytest

from kv8_bound import exact_attention, filled, ints, randn, starts, worst

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,group,n,seq_pages", [(1, 4, 300, 32), (1, 7, 1500, 80), (3, 4, 400, 32), (2, 16, 2000, 80),
                                                    (1, 20, 900, 32)])
def test_few_f16_rows_hold_weights_in_two_halves(qh, gpu, rows, group, n, seq_pages, hd):
    """f16 calls with few rows round the result once and little before that. A result differs from the rounded exact one
    where an error e from before lies between it and a border of rounding, at odds of e over a step, which is 2^-11 to 2^-10
    of the value. Two halves (2^-22), scores and sums in f32 leave e near 2^-19 of it, so at most one in a hundred; one half
    leaves 2^-12.3 (root mean square of a rounding), so one in four and more. One in twenty lies between."""
    import torch
    k, v = randn(1, n, 2, hd).half(), randn(2, n, 2, hd).half()
    c = filled(qh, k, v, [n], page=32, seq_pages=seq_pages)
    q = randn(3, rows, 2 * group, hd).half()
    got = c.attention(0, q, start=starts([rows]), seqs=ints([0]))
    want, bound = exact_attention(c, 0, q, [0], [rows], two=True)
    ratio, at = worst(got, want, bound)
    assert ratio <= 1, (ratio, at)
    same = (got == want.half()).double().mean().item()
    assert same >= 0.95, same
    if rows == 1:
        assert torch.equal(c.attention(0, q, seqs=ints([0])), got)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,heads,n,seq_pages,kernel,split", [
    (1, 7, 900, 32, 0, False), (1, 7, 5000, 160, 1, True), (3, 4, 9000, 300, 1, True), (60, 4, 300, 12, 2, False),
    (60, 4, 5000, 160, 2, True), (620, 4, 5000, 160, 2, True), (9000, 4, 600, 20, 2, False)])
def test_each_weight_in_f32_by_every_kernel(qh, gpu, rows, heads, n, seq_pages, kernel, split, hd):
    """hd positions spread over the sequence hold one-hot values, all others zeros, so that a result's channels are the weights of
    those positions. Small scores: a weight's relative error is that of its two halves (2^-22), its exponential, products and
    division (16 roundings) and its row's sum (four additions a tile of 64 and lane, and 32 to meet)."""
    import torch
    k, v = randn(1, n, 1, hd), torch.zeros(n, 1, hd, device="cuda")
    at = torch.linspace(0, n - 1, hd, device="cuda").long()
    v[at, 0, torch.arange(hd, device="cuda")] = 1
    c = filled(qh, k, v, [n], seq_pages=seq_pages)
    plan = c.attention_plan(heads, 1, rows)
    assert (plan.kernel, plan.splits > 1) == (kernel, split)
    keys, values = c.read(0, n, start=ints([0, n]), seqs=ints([0]))
    assert torch.equal(values, v)
    q = randn(2, rows, heads, hd) * 1e-3
    got = c.attention(0, q, start=ints([0, rows]), seqs=ints([0]), causal=False).double()
    e = torch.exp((q.double().view(-1, hd) @ keys[:, 0].double().t().contiguous()) * hd ** -0.5)
    want = (e / e.sum(1, keepdim=True))[:, at].view(got.shape)
    bound = want * (2.0 ** -22 + (16 + 4 * -(-n // 64) + 32) * 2.0 ** -24) + 2.0 ** -30 * want.amax()
    ratio, i = worst(got, want, bound)
    assert ratio <= 1, (ratio, i, float(got[i]), float(want[i]))
