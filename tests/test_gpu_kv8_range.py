"""Attention over the 8-bit cache where value scales lie far apart: blocks that a row does not see, or gives no weight to, do
not take bits from it. Bounds (kv8_bound) use only what a row sees."""
import numpy as np
import pytest

from kv8_bound import exact_attention, filled, ints, randn, starts, worst

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(gpu):
    return gpu


def check(c, q, counts, seqs=None, single=False, causal=True):
    import torch
    seqs = list(range(len(counts))) if seqs is None else seqs
    got = c.attention(0, q, start=None if single else starts(counts), seqs=ints(seqs), causal=causal)
    want, bound = exact_attention(c, 0, q, seqs, counts, causal)
    assert torch.isfinite(got).all()
    ratio, at = worst(got, want, bound)
    assert ratio <= 1, (ratio, at, float(got[at]), float(want[at]))


# the largest values over the others: f16 rows reach no further than 2^26 (6e4 over 1e-3)
RATIOS = [("float32", 2.0 ** 14), ("float32", 2.0 ** 22), ("float32", 1e10), ("float32", 1e20), ("float16", 2.0 ** 15)]


@pytest.mark.parametrize("dtype,ratio", RATIOS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,heads,seq_pages", [(3, 2, 40), (4, 2, 80), (70, 2, 40), (300, 2, 80), (300, 40, 40)])
def test_a_large_value_behind_the_row(qh, dtype, ratio, hd, rows, heads, seq_pages):
    """The last token holds a value `ratio` times the others: the rows before it do not see it. Tables on both sides of the
    few-row kernels' and the splits' rules."""
    import torch
    n, t = 317, getattr(torch, dtype)
    k, v = randn(1, n, 2, hd), randn(2, n, 2, hd) * (1.0 if dtype == "float32" else 2.0 ** -6)
    v[-1] *= ratio
    c = filled(qh, k.to(t), v.to(t), [n], seq_pages=seq_pages)
    check(c, randn(3, rows, heads, hd).to(t), [rows])


@pytest.mark.parametrize("dtype,ratio", RATIOS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,seq_pages,at", [(1, 40, 5), (1, 90, 70), (6, 90, 40), (90, 40, 33), (300, 90, 130), (1, 40, 316)])
def test_a_large_value_without_weight(qh, dtype, ratio, hd, rows, seq_pages, at):
    """A visible block with a value `ratio` times the others and scores so low that it counts for nothing: first,
    in the middle and last, with tiles of ordinary values behind it."""
    import torch
    n, t = 317, getattr(torch, dtype)
    k, v = randn(1, n, 1, hd), randn(2, n, 1, hd) * (1.0 if dtype == "float32" else 2.0 ** -6)
    q = randn(3, rows, 4, hd)
    q[..., 0] = 8.0 * hd ** 0.5  # the first channel says: a score of 8 times the key's
    k[..., 0] = 0.0
    k[at // 16 * 16:at // 16 * 16 + 16, :, 0] = -25.0  # e^-200, for the block that the value gives its scale
    v[at] *= ratio
    c = filled(qh, k.to(t), v.to(t), [n], seq_pages=seq_pages)
    check(c, q.to(t), [rows])
    if rows == 1:
        check(c, q.to(t), [1], single=True)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("rows,seq_pages", [(1, 40), (1, 90), (6, 90), (90, 40), (400, 90)])
def test_values_of_every_size_in_any_order(qh, dtype, rows, seq_pages):
    """Blocks of 16 tokens whose values are 2^-40 to 2^40 apart (2^-12 to 2^12 in f16), zeros among them, with scores that
    prefer small ones, large ones or none."""
    import torch
    n, hd, t, far = 640, 64, getattr(torch, dtype), 40 if dtype == "float32" else 12
    rng = np.random.default_rng(7)
    for slope in (-1.0, -0.3, 0.0, 0.7):
        size = rng.integers(-far, far + 1, n // 16)
        k, v = randn(1, n, 2, hd), randn(2, n, 2, hd)
        lift = torch.from_numpy(np.repeat(size, 16).astype(np.float32)).to("cuda").view(-1, 1)
        v *= torch.exp2(lift).unsqueeze(-1)
        v[16 * 7:16 * 8] = 0
        v[:16] = 0
        k[..., 0] = lift * slope * float(np.log(2.0))
        k[16 * 7:16 * 8, :, 0] = 10.0  # zeros that nearly all the weight goes to in some rows
        q = randn(3, rows, 4, hd)
        q[..., 0] = hd ** 0.5
        c = filled(qh, k.to(t), v.to(t), [n], seq_pages=seq_pages)
        check(c, q.to(t), [rows])
        check(c, q.to(t), [rows], causal=False)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,n,seq_pages", [(1, 300, 32), (4, 300, 32), (1, 2500, 90), (4, 2500, 90), (90, 300, 32), (90, 2500, 90),
                                              (90, 2500, 32)])
def test_values_near_the_end_of_the_range(qh, rows, n, seq_pages, hd):
    """Values whose sum is past f32's largest number, and their weighted mean is not; in whole rows, shares, halves of a
    workgroup and splits."""
    import torch
    k, v = randn(1, n, 2, hd) * 0.1, 2.9e38 * (1 - 0.2 * torch.sigmoid(randn(2, n, 2, hd)))
    v[:, :, ::2] *= -1
    c = filled(qh, k, v, [n], page=32 if n <= 32 * seq_pages else 128, seq_pages=seq_pages)
    q = randn(3, rows, 6, hd)
    check(c, q, [rows])
    if rows == 1:
        check(c, q, [1], single=True)


def test_tokens_that_are_cut_off_leave_their_scale(qh):
    """A draft of large values and one of a NaN, cut off inside their blocks: the tokens that stay keep the scale (the NaN), as
    the definition says, until the block is stored anew; other blocks are as if the draft had never been."""
    import torch
    hd = 64
    k, v = randn(1, 40, 1, hd), randn(2, 40, 1, hd)
    c = filled(qh, k[:20], v[:20], [20], seq_pages=4)
    read = lambda m: c.read(0, m, start=ints([0, m]), seqs=ints([0]))[0]
    before = read(20)
    one, two = k[20:26] * 1000, k[20:26].clone()
    two[1, 0, 5] = float("nan")

    def draft(rows, keep):
        c.resize(ints([0]), ints([26]))
        c.append(0, rows, v[20:26], start=ints([0, 6]), seqs=ints([0]))
        c.resize(ints([0]), ints([keep]))

    draft(one, 20)
    after = read(20)
    assert torch.equal(after[:16], before[:16])
    step = (one.abs().amax().double() / 127).float()
    want = torch.trunc(before[16:].double() / step + torch.copysign(torch.tensor(0.5), before[16:])) * step
    assert torch.allclose(after[16:].double(), want, rtol=2.0 ** -22, atol=0)
    draft(two, 20)
    assert torch.equal(read(20)[:16], before[:16]) and torch.isnan(read(20)[16:]).all()
    c.resize(ints([0]), ints([16]))  # from the block's first token again
    c.resize(ints([0]), ints([20]))
    c.append(0, k[16:20], v[16:20], start=ints([0, 4]), seqs=ints([0]))
    assert torch.equal(read(20), before)


@pytest.mark.parametrize("rows,seq_pages", [(1, 40), (1, 90), (6, 40), (90, 40)])
@pytest.mark.parametrize("at", [3, 15, 40, 63, 64, 300])
def test_a_large_value_of_one_token(qh, rows, seq_pages, at):
    """One token's value 1e10 times the others' and its score too low to count, wherever it lies; stored with the prompt, or
    token by token, so that earlier codes of its block are rounded to zero and later ones are zero from the start; read from a
    copy; and gone again with the tokens from it on."""
    import torch
    n, hd = 317, 64
    k, v, q = randn(1, n, 2, hd), randn(2, n, 2, hd), randn(3, rows, 6, hd)
    k[..., 0], q[..., 0] = 0.0, 8.0 * hd ** 0.5
    k[at, :, 0] = -25.0
    v[at] *= 1e10
    whole = filled(qh, k, v, [n], seq_pages=seq_pages)
    check(whole, q, [rows])
    c = qh.KV8Cache(1, 40, 32, 2, hd, 3, seq_pages)
    c.pages.fill_(0x7f)
    first = max(0, at - 9)
    for a, b in [(0, first)] * (first > 0) + [(i, i + 1) for i in range(first, min(n, at + 20))] + [(min(n, at + 20), n)] * (at + 20 < n):
        c.resize(ints([0]), ints([b]))
        c.append(0, k[a:b], v[a:b], start=ints([0, b - a]), seqs=ints([0]))
    check(c, q, [rows], seqs=[0])
    c.fork(ints([0, 0]), ints([1, 2]), copy=True)
    check(c, q, [rows], seqs=[2])
    if at >= 15 and at % 16:
        c.resize(ints([1]), ints([at]))  # the block of the cut keeps the scale, and only zeros
        m = min(rows, at)
        check(c, q[:m], [m], seqs=[1])


def test_reads_do_not_see_the_mark(qh):
    """The values read back beside a large one: zeros, not zeros of another sign of scale; and a block that grows again from
    them takes its scale's size."""
    import torch
    k = torch.zeros(20, 1, 64, device="cuda")
    k[:, 0, 0] = 1.0
    v = k.clone()
    v[3] *= 1e6
    c = filled(qh, k[:17], v[:17], [17], seq_pages=2)
    got = c.read(0, 17, start=ints([0, 17]))[1]
    assert (got[:16] >= 0).all() and float(got[3, 0, 0]) == 1e6 and float(got[:16].sum()) == 1e6 and float(got[16, 0, 0]) == 1.0
    c.resize(ints([0]), ints([10]))
    c.resize(ints([0]), ints([12]))
    c.append(0, k[10:12], -v[10:12], start=ints([0, 2]))
    got = c.read(0, 12, start=ints([0, 12]))[1]
    assert float(got[3, 0, 0]) == 1e6 and float(got.abs().sum()) == 1e6
