"""Attention of packed prompts (qh_attention) against its formula in 64 bits: types, head layouts, lengths, entries without rows
or keys, strides, hidden values that are not finite, scales, and values far apart.

Bounds, relative to sum_j p_j |v_j| of a result (call it A), for scores of a row that reach X = scale sum_i |q_i k_i|:
* a score is off by what products drop and sums round: f32 2^-22 (products, six of nine) + 2^-24 (hd + 8) (sums of 6 hd terms
  whose parts fall off quickly, at most one rounding per 32 x 32 x 16 step and operand) of X, f16 the sums alone; the exponent
  (score times log2 e less the base) rounds twice more, 2^-23 of |x| <= X log2 e + 2^7, and exp2 is off by 2^-22: a weight is
  off by d = ln 2 times that in all;
* weights go in as f16 (half a step, 2^-11, and below 2^-14 of the base's 2^-6 by 2^-25 of it: 2^-31 of the largest weight each)
  or in three bf16 (2^-24); the sum takes the rounded ones in f16;
* the second product drops 2^-22 (f32), its sums and the join round 2^-24 for each of the keys / 16 steps and more;
* the result rounds once: 2^-11 or 2^-24 of itself.
The test's bound is the sum of these."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16}


def formula(q, k, v, start, kstart, causal, scale):
    """(result, bound, rows that belong to an entry) in 64 bits on the CPU or GPU, a head at a time."""
    half = q.dtype is torch.float16
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    err, mine = out.clone(), torch.zeros(rows, dtype=torch.bool, device=q.device)
    for a, b, c, d in zip(start[:-1], start[1:], kstart[:-1], kstart[1:]):
        m, l = b - a, d - c
        mine[a:b] = True
        if m <= 0 or l <= 0:
            continue
        see = torch.ones(m, l, dtype=torch.bool, device=q.device)
        if causal:
            see = torch.arange(l, device=q.device) <= torch.arange(l - m, l, device=q.device).view(m, 1)
        none = ~see.any(1)
        for h in range(heads):
            x, y = q[a:b, h].double(), k[c:d, h // group].double()
            z = v[c:d, h // group].double()
            s = (x @ y.t().contiguous() * scale).masked_fill(~see, -math.inf)
            s[none] = 0.0
            p = torch.softmax(s, 1)
            p[none] = 0.0
            p[~see] = 0.0
            # hidden values have no part, whatever they are
            o = p @ torch.where(torch.isfinite(z), z, torch.zeros_like(z))
            strange = (~torch.isfinite(z)).double()
            if bool(strange.any()):
                for j in strange.any(1).nonzero().view(-1).tolist():
                    o = o + torch.where(see[:, j:j + 1] & (strange[j:j + 1] > 0), z[j:j + 1].expand(m, hd), torch.zeros_like(o))
            out[a:b, h] = o
            top = (x.abs() @ y.abs().t().contiguous()).masked_fill(~see, 0.0).amax(1, keepdim=True) * abs(scale)
            dx = top * 2.0 ** -24 * (hd + 8) + (0.0 if half else top * 2.0 ** -22)
            dx = dx + 2.0 ** -23 * (top * 1.4427 + 128) * math.log(2) + 2.0 ** -22
            mass = p @ z.abs().nan_to_num(0.0, 0.0, 0.0)
            big = z.abs().nan_to_num(0.0, 0.0, 0.0).amax(0, keepdim=True)
            peak = p.amax(1, keepdim=True)
            each = 2 * dx + (2.0 ** -10 if half else 2.0 ** -21) + 2.0 ** -24 * (l / 8 + 40)
            err[a:b, h] = each * mass + (peak * l * 2.0 ** -30 * big if half else 0.0) + (2.0 ** -11 if half else 2.0 ** -24) * o.abs()
    return out, err + (2.0 ** -25 if half else 2.0 ** -140), mine


def check(got, want, err, mine):
    got, want = got.double()[mine], want[mine]
    there = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    off = (got[there] - want[there]).abs() / err[mine][there]
    assert off.numel() == 0 or off.max() <= 1.0, off.max()


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def starts(counts):
    return [0] + np.cumsum(counts).tolist()


def case(qh, gpu, dtype, heads, kv, hd, rows, keys=None, causal=True, scale=None, seed=0, wide=1.0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    t, st = TYPES[dtype], starts(rows)
    kst = st if keys is None else starts(keys)
    q = torch.randn(st[-1], heads, hd, generator=gen, device=gpu).mul(wide).to(t)
    k = torch.randn(kst[-1], kv, hd, generator=gen, device=gpu).to(t)
    v = torch.randn(kst[-1], kv, hd, generator=gen, device=gpu).to(t)
    got = qh.attention(q, k, v, ints(st, gpu), None if keys is None else ints(kst, gpu), causal=causal, scale=scale)
    check(got, *formula(q, k, v, st, kst, causal, hd ** -0.5 if scale is None else scale))
    return q, k, v, got


LAYOUTS = [(1, 1, 64), (4, 4, 64), (14, 2, 64), (40, 2, 64), (8, 1, 128), (32, 8, 128), (3, 3, 128), (9, 3, 64)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", LAYOUTS)
def test_layouts(qh, gpu, dtype, heads, kv, hd):
    case(qh, gpu, dtype, heads, kv, hd, [1, 77, 0, 200, 33])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [500], [1025], [1] * 50, [0, 0, 5, 0],
                                  [3, 64, 1, 129, 32, 7], [2] * 63, [3] * 64, [5, 0, 1, 33] * 40])
def test_lengths(qh, gpu, dtype, hd, rows):
    case(qh, gpu, dtype, 4, 2, hd, rows, seed=len(rows) + rows[-1])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [([1], [1]), ([1], [1000]), ([5, 40], [70, 40]), ([64, 3], [65, 300]), ([130], [2000]),
                                       ([20, 7], [5, 0]), ([200], [3]), ([1, 1, 1], [17, 64, 129]), ([33, 0, 9], [31, 64, 900]),
                                       ([1] * 9, [333] * 9), ([3, 0, 2] * 30, [5, 70, 1] * 30)])
def test_keys_of_their_own(qh, gpu, dtype, hd, causal, rows, keys):
    """New rows behind kept ones, other states' keys, and more rows than keys: the first of them see nothing then."""
    case(qh, gpu, dtype, 6, 2, hd, rows, keys, causal, seed=sum(keys))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_long(qh, gpu, dtype):
    case(qh, gpu, dtype, 4, 1, 64, [3001])
    case(qh, gpu, dtype, 2, 2, 128, [2500, 1700])
    case(qh, gpu, dtype, 2, 1, 128, [7], [20011])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("off", [0, 1])
def test_many_rows(qh, gpu, dtype, hd, off):
    """Calls whose row tiles are as many as the compute units, which workgroups of eight waves take: ragged lengths, values that
    are not finite behind rows and between entries, and rows that begin anywhere (keys on multiples of 16 bytes go another way)."""
    t, heads = TYPES[dtype], 16
    st = [0, 700, 700, 763, 2900, 4300]
    gen = torch.Generator(device=gpu).manual_seed(hd + off)
    buf = torch.randn(4300 * 3 * heads * hd + off, generator=gen, device=gpu).to(t)
    row = buf[off:].view(4300, 3, heads, hd)
    q, k, v = row[:, 0], row[:, 1], row[:, 2]
    v[699, 3, 5], v[1500, 2, hd - 1], v[2899, 0, 0] = math.nan, math.inf, -math.inf
    assert 4300 // 256 * heads >= 256
    check(qh.attention(q, k, v, ints(st, gpu)), *formula(q, k, v, st, st, True, hd ** -0.5))
    v[1500, 2, hd - 1] = 0.5
    check(qh.attention(q, k, v, ints(st, gpu), causal=False), *formula(q, k, v, st, st, False, hd ** -0.5))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-8, -1e-30])
def test_scales(qh, gpu, dtype, scale):
    case(qh, gpu, dtype, 4, 2, 64, [50, 129], scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_large_scores(qh, gpu, dtype, hd):
    """Scores of some hundreds: a row's base moves many times, and most weights vanish."""
    case(qh, gpu, dtype, 4, 2, hd, [300, 70], wide=30.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("up", [True, False])
def test_scores_that_rise_or_fall(qh, gpu, dtype, up):
    """Scores that grow (or fall) tile by tile by more than the slack of a base."""
    n, hd = 700, 64
    q = torch.ones(n, 2, hd, device=gpu)
    ramp = torch.linspace(0, 12, n, device=gpu)
    k = torch.randn(n, 1, hd, device=gpu) * 0.1 + (ramp if up else ramp.flip(0)).view(n, 1, 1)
    v = torch.randn(n, 1, hd, device=gpu)
    q, k, v = (x.to(TYPES[dtype]) for x in (q, k, v))
    got = qh.attention(q, k, v)
    check(got, *formula(q, k, v, [0, n], [0, n], True, hd ** -0.5))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_have_no_part(qh, gpu, dtype, hd, bad):
    """Keys and values that are not finite where rows do not see them: later positions, other sequences, and behind the last.
    Rows that see such a value have it in that dim alone; a row that sees such a key is NaN (or leaves it out)."""
    gen = torch.Generator(device=gpu).manual_seed(hd)
    st = [0, 70, 70, 199, 230]
    q, k, v = (torch.randn(240, 2, hd, generator=gen, device=gpu).to(TYPES[dtype]) for _ in range(3))
    v[100, 0, 5] = bad          # in the middle of the third entry: rows from it on see it
    v[198, 1, hd - 1] = bad     # its last position
    v[0, 0, 0] = bad            # the first position of the first: every row of it
    v[230:], k[230:], q[230:] = bad, bad, bad   # behind the last entry
    want = formula(q, k, v, st, st, True, hd ** -0.5)
    check(qh.attention(q, k, v, ints(st, gpu)), *want)
    k2 = k.clone()
    k2[150, 1] = bad
    got = qh.attention(q, k2, v, ints(st, gpu))
    keep = torch.ones(240, 2, dtype=torch.bool, device=gpu)
    keep[150:199, 1] = False
    keep[230:] = False
    a, b = got.double()[keep], want[0][keep]
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    there = torch.isfinite(b)
    assert bool(((a[there] - b[there]).abs() <= want[1][keep][there]).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_that_are_not_finite_stay_alone(qh, gpu, dtype):
    q, k, v = (torch.randn(150, 4, 64, device=gpu).to(TYPES[dtype]) for _ in range(3))
    clean = qh.attention(q, k, v)
    q[17, 2], q[100, 0, 3] = math.nan, math.inf
    got = qh.attention(q, k, v)
    other = torch.ones(150, 4, dtype=torch.bool, device=gpu)
    other[17, 2] = other[100, 0] = False
    assert torch.equal(got[other], clean[other]) and bool(torch.isnan(got[~other]).all())


def test_far_apart_values(qh, gpu):
    """f32: hidden values and keys 1e30 times the others, and values of 1e-30 next to ones, take nothing from a row."""
    q, k, v = (torch.randn(200, 2, 64, device=gpu) for _ in range(3))
    v[120:] *= 1e30
    v[:60, :, ::2] *= 1e-30
    got = qh.attention(q, k, v)
    check(got, *formula(q, k, v, [0, 200], [0, 200], True, 0.125))
    small = qh.attention(q * 1e-15, k * 1e15, v)
    check(small, *formula(q * 1e-15, k * 1e15, v, [0, 200], [0, 200], True, 0.125))
    ends = torch.full((80, 2, 64), 3.4e38, device=gpu)
    check(qh.attention(q[:80], k[:80], ends), *formula(q[:80], k[:80], ends, [0, 80], [0, 80], True, 0.125))


def test_large_f16_values(qh, gpu):
    q, k = (torch.randn(200, 2, 64, device=gpu).half() for _ in range(2))
    v = torch.full((200, 2, 64), 65504.0, device=gpu).half()
    assert bool((qh.attention(q, k, v) == 65504.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_strides(qh, gpu, dtype, hd):
    """Views of one fused row at an odd offset, and rows outside the entries left as they were."""
    t, heads, kv, rows = TYPES[dtype], 6, 2, 150
    width = (heads + 2 * kv) * hd + 5
    buf = torch.randn(rows * width + 3, device=gpu).to(t)
    row = buf[3:].view(rows, width)
    q = row[:, :heads * hd].view(rows, heads, hd)
    k = row[:, heads * hd:(heads + kv) * hd].view(rows, kv, hd)
    v = row[:, (heads + kv) * hd:(heads + 2 * kv) * hd].view(rows, kv, hd)
    obuf = torch.full((rows * (heads * hd + 7) + 1,), 7.0, dtype=t, device=gpu)
    out = obuf[1:].view(rows, heads * hd + 7)[:, :heads * hd].view(rows, heads, hd)
    st = [10, 60, 60, 140]
    got = qh.attention(q, k, v, ints(st, gpu), out=out)
    assert got is out
    check(out, *formula(q, k, v, st, st, True, hd ** -0.5))
    held = torch.full_like(obuf, 7.0)
    held[1:].view(rows, heads * hd + 7)[10:140, :heads * hd] = out[10:140].reshape(130, heads * hd)
    assert torch.equal(held, obuf)


def test_far_rows(qh, gpu):
    """Rows past 4 GiB of the first one."""
    ld = (1 << 28) + 8
    buf = torch.zeros(9 * ld, dtype=torch.float16, device=gpu)
    row = buf.view(9, ld)
    q, k, v = (row[:, 64 * i:64 * i + 64].view(9, 1, 64) for i in range(3))
    for x in (q, k, v):
        x.copy_(torch.randn(9, 1, 64, device=gpu))
    out = row[:, 256:320].view(9, 1, 64)
    qh.attention(q, k, v, out=out)
    assert torch.equal(out, qh.attention(q.contiguous(), k.contiguous(), v.contiguous()))


def test_starts_of_any_kind(qh, gpu):
    """Starts past the rows, below 0 or out of order: rows stay inside, and an entry that ends before it begins is empty."""
    q, k, v = (torch.randn(40, 2, 64, device=gpu) for _ in range(3))
    out = torch.full_like(q, 7.0)
    qh.attention(q, k, v, ints([-5, 20, 20, 1000], gpu), out=out)
    check(out, *formula(q, k, v, [0, 20, 20, 40], [0, 20, 20, 40], True, 0.125))
    out.fill_(7.0)
    qh.attention(q, k, v, ints([30, 10], gpu), out=out)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_same_bits_every_time_and_alone(qh, gpu, dtype):
    """A sequence's rows do not depend on what else is in the batch, and calls give the same bits again."""
    q, k, v = (torch.randn(400, 4, 64, device=gpu).to(TYPES[dtype]) for _ in range(3))
    st = [0, 100, 229, 400]
    got = qh.attention(q, k, v, ints(st, gpu))
    assert torch.equal(got, qh.attention(q, k, v, ints(st, gpu)))


def test_captured_and_on_another_stream(qh, gpu):
    q, k, v = (torch.randn(300, 4, 64, device=gpu) for _ in range(3))
    st = ints([0, 120, 300], gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = qh.attention(q, k, v, st)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, qh.attention(q, k, v, st))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = qh.attention(q, k, v, st)
        graphs.append((g, out))
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        st.copy_(ints([0, 50 * i + 1, 300], gpu))
        want = qh.attention(q, k, v, st)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


def test_refuses(qh, gpu):
    q, k, v = (torch.randn(10, 4, 64, device=gpu) for _ in range(3))
    st = ints([0, 10], gpu)
    for call in (lambda: qh.attention(q.double(), k, v), lambda: qh.attention(q, k.half(), v), lambda: qh.attention(q, k[:, :3], v[:, :3]),
                 lambda: qh.attention(q, k, v[:9]), lambda: qh.attention(q[..., :32], k[..., :32], v[..., :32]),
                 lambda: qh.attention(q, k, v, st.long()), lambda: qh.attention(q, k, v, st.cpu()),
                 lambda: qh.attention(q, k[:5], v[:5], st), lambda: qh.attention(q, k, v, st, ints([0, 5, 10], gpu)),
                 lambda: qh.attention(q, k, v, st, out=q), lambda: qh.attention(q, k, v, kstart=st),
                 lambda: qh.attention(q.cpu(), k.cpu(), v.cpu(), st.cpu()), lambda: qh.attention(q, k, v, st, scale=math.nan),
                 lambda: qh.attention(q.transpose(0, 1), k, v, st)):
        with pytest.raises(qh.QHError):
            call()
