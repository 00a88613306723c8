"""Attention over the 8-bit cache by each of its kernels, in both types and head sizes: every case states the kernel it is meant
to reach and checks that it does, so that a change of the rules cannot leave one untested."""
import pytest

from kv8_bound import exact_attention, filled, ints, randn, starts, worst

pytestmark = pytest.mark.gpu

WHOLE, SHARES, TILES = 0, 1, 2
SHORT = [(37 * i) % 301 for i in range(140)]
MANY = [(37 * i) % 201 for i in range(100)]
MANY[3], MANY[40], MANY[97], MANY[99] = 4100, 2500, 3001, 1

# name, head_dims, query heads, KV heads, lengths, rows of each entry (None: single tokens), kernel (kind, rows, waves, split)
CASES = [
    ("whole, 8 waves", (64, 128), 14, 2, [700, 1, 130, 0], None, (WHOLE, 16, 8, False)),
    ("whole, 8 waves, drafts", (64, 128), 10, 2, [700, 3, 130, 64], [3, 3, 0, 5], (WHOLE, 16, 8, False)),
    ("whole, 4 waves", (64, 128), 8, 2, SHORT, None, (WHOLE, 16, 4, False)),
    ("whole, 4 waves, drafts", (64, 128), 8, 2, SHORT, [i % 5 for i in range(140)], (WHOLE, 16, 4, False)),
    ("shares, 8 waves", (64, 128), 14, 2, [5000, 3, 2500, 0], None, (SHARES, 16, 8, True)),
    ("shares, 8 waves, drafts", (64, 128), 14, 2, [5000, 3, 2500, 70], [4, 3, 1, 2], (SHARES, 16, 8, True)),
    ("shares, 4 waves", (64, 128), 16, 4, MANY, None, (SHARES, 16, 4, True)),
    ("shares, 4 waves, drafts", (64, 128), 16, 4, MANY, [i % 4 for i in range(100)], (SHARES, 16, 4, True)),
    ("tiles of 128 rows", (128,), 32, 8, [900, 300, 330, 700], [700, 1, 330, 129], (TILES, 128, 4, False)),
    ("tiles, 4 waves", (64, 128), 32, 8, [500, 300, 131, 700], [300, 1, 131, 203], (TILES, 64, 4, False)),
    ("tiles, 4 waves, split", (64, 128), 14, 2, [1500, 700, 211], [300, 161, 201], (TILES, 64, 4, True)),
    ("tiles, 8 waves", (64, 128), 8, 2, [500, 64, 130], [77, 20, 33], (TILES, 64, 8, False)),
    ("tiles, 8 waves, split", (64, 128), 8, 2, [3000, 64, 1300], [77, 20, 33], (TILES, 64, 8, True)),
    ("tiles, single tokens of many heads", (64, 128), 80, 2, [700, 1, 130], None, (TILES, 64, 8, True)),
]


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("case", [(c[0], hd) + c[2:] for c in CASES for hd in c[1]], ids=lambda c: f"{c[0]}, {c[1]}")
def test_kernel(qh, gpu, case, dtype):
    import torch
    _, hd, heads, kv, lens, counts, (kind, tile, waves, split) = case
    t = getattr(torch, dtype)
    n = sum(lens)
    c = filled(qh, (randn(1, n, kv, hd) * 1.5).to(t), randn(2, n, kv, hd).to(t), lens)
    single = counts is None
    counts = [1] * len(lens) if single else counts
    rows = sum(counts)
    plan = c.attention_plan(heads, len(lens), rows, single)
    assert (plan.kernel, plan.rows, plan.waves, plan.splits > 1, plan.launches) == (kind, tile, waves, split, 1)
    q = randn(3, rows, heads, hd).to(t)
    few = plan.kernel != TILES
    for causal in (True, False):
        got = c.attention(0, q, start=None if single else starts(counts), seqs=ints(range(len(lens))), causal=causal)
        want, bound = exact_attention(c, 0, q, range(len(lens)), counts, causal, two=few or dtype == "float32")
        ratio, at = worst(got, want, bound)
        assert ratio <= 1, (causal, ratio, at, float(got[at]), float(want[at]))
        # and on the whole: half an f16 step of a result is 2^-11 of it at most, 2^-10 / sqrt(12) in the mean square; weights in
        # one f16 add as much again; in f32 a lost half of a weight or of a query would be 2^-13 of the results and more, and
        # scores, sums and halves that are kept stay a hundred times below
        off = ((got.double() - want).norm() / want.norm()).item()
        assert off <= (2.0 ** -17 if dtype == "float32" else 2.0 ** -10 / 12 ** 0.5 * (1.05 if few else 1.5)), (causal, off)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("case", [(c[0], hd) + c[2:] for c in CASES for hd in c[1]], ids=lambda c: f"{c[0]}, {c[1]}")
def test_kernel_with_value_scales_far_apart(qh, gpu, case, dtype):
    """The same with blocks whose values are up to 2^60 apart (2^18 in f16), the largest last and, for some rows, out of sight,
    and scores that grow or fall along the sequence."""
    import torch
    _, hd, heads, kv, lens, counts, kernel = case
    t, far, n = getattr(torch, dtype), 30 if dtype == "float32" else 9, sum(lens)
    k, v = randn(1, n, kv, hd), randn(2, n, kv, hd)
    at = torch.cat([torch.arange(m, device="cuda") for m in lens])
    size = (at // 16 * 37 + 11) % (2 * far + 1) - far
    ends = torch.tensor(lens, device="cuda").repeat_interleave(torch.tensor(lens, device="cuda"))
    size = torch.where(at // 16 == (ends - 1) // 16, far, size)
    v *= torch.exp2(size.float()).view(-1, 1, 1)
    k[..., 0] = (at.float() / 50).view(-1, 1)
    c = filled(qh, k.to(t), v.to(t), lens)
    single = counts is None
    counts = [1] * len(lens) if single else counts
    q = randn(3, sum(counts), heads, hd)
    q[..., 0] = torch.linspace(-2, 2, heads, device="cuda")
    q = q.to(t)
    for causal in (True, False):
        got = c.attention(0, q, start=None if single else starts(counts), seqs=ints(range(len(lens))), causal=causal)
        want, bound = exact_attention(c, 0, q, range(len(lens)), counts, causal, two=kernel[0] != TILES or dtype == "float32")
        ratio, at_ = worst(got, want, bound)
        assert ratio <= 1, (causal, ratio, at_, float(got[at_]), float(want[at_]))


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("case", [(c[0], hd) + c[2:] for c in CASES for hd in c[1]], ids=lambda c: f"{c[0]}, {c[1]}")
def test_kernel_with_single_large_values(qh, gpu, case, dtype):
    """Single tokens whose values are so large that the others of their blocks have only zeros for codes, and whose scores are so
    low that they count for nothing (every seventh has a score like the others'): the zeros beside them have their share of the
    weights, and ordinary values elsewhere keep all their bits."""
    import torch
    _, hd, heads, kv, lens, counts, kernel = case
    t, n = getattr(torch, dtype), sum(lens)
    k, v = randn(1, n, kv, hd), randn(2, n, kv, hd) * (1 if dtype == "float32" else 2.0 ** -9)
    k[..., 0] = 0.0
    at = torch.cat([torch.arange(m, device="cuda") for m in lens])
    large = at % 97 == 5
    v[large] *= 1e12 if dtype == "float32" else 2.0 ** 16
    k[large & (at % 7 != 0), :, 0] = -25.0
    c = filled(qh, k.to(t), v.to(t), lens)
    single = counts is None
    counts = [1] * len(lens) if single else counts
    q = randn(3, sum(counts), heads, hd)
    q[..., 0] = 8.0 * hd ** 0.5
    q = q.to(t)
    for causal in (True, False):
        got = c.attention(0, q, start=None if single else starts(counts), seqs=ints(range(len(lens))), causal=causal)
        want, bound = exact_attention(c, 0, q, range(len(lens)), counts, causal, two=kernel[0] != TILES or dtype == "float32")
        ratio, at_ = worst(got, want, bound)
        assert ratio <= 1, (causal, ratio, at_, float(got[at_]), float(want[at_]))
