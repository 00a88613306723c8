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
