"""The row operators (qh_rmsnorm, qh_rope) against their formulas in 64 bits, over types, widths, strides and positions.

Tolerances: a result is rounded once, half a step of its type (2^-24 relative in f32, 2^-11 in f16, and half the smallest
subnormal); what a rotation adds before that is derived where it is used. Codes and scales are equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25}


def guarded(rows, width, ld, off, dtype, dev, fill=7.0):
    """A [rows][width] view with row stride ld that begins `off` elements into a buffer of `fill`, and the buffer."""
    buf = torch.full((off + max(rows, 1) * ld + 19,), fill, dtype=dtype, device=dev)
    return buf[off:off + rows * ld].view(rows, ld)[:, :width] if rows else buf[:0].view(0, width), buf


def untouched(buf, view, fill=7.0):
    """Everything of the buffer outside the view still holds `fill`."""
    keep = torch.ones_like(buf, dtype=torch.bool)
    if view.numel():
        off = view.storage_offset()
        ld = view.stride(0) if view.shape[0] > 1 else view.shape[1]
        for r in range(view.shape[0]):
            keep[off + r * ld:off + r * ld + view.shape[1]] = False
    return bool((buf[keep] == fill).all())


def norm_formula(h, w, eps):
    h = h.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()


def check_rounded(got, want, dtype):
    err = (got.double() - want).abs()
    assert bool((err <= STEP[dtype] * (1 + 2 ** -20) * want.abs() + TINY[dtype]).all()), err.max()


def codes_of(oracle, y32):
    q, d = oracle.quantize_q8(y32.cpu().numpy())
    return q, d


WIDTHS = [1, 2, 3, 7, 8, 31, 32, 33, 64, 255, 256, 257, 512, 513, 896, 1024, 1025, 2048, 2049, 4096, 4864, 5120, 8192, 8193, 16384,
          16391, 32768]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", WIDTHS)
def test_norm(qh, oracle, gpu, dtype, n):
    t = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(n)
    rows = 5 if n > 64 else 131
    x = torch.randn(rows, n, generator=gen, device=gpu).mul(3).to(t)
    res = torch.randn(rows, n, generator=gen, device=gpu).to(t)
    w = torch.randn(n, generator=gen, device=gpu)
    h = (x.float() + res.float()).to(t)
    want = norm_formula(h, w, 1e-6)
    total, y = qh.rmsnorm(x, w, 1e-6, residual=res)
    assert torch.equal(total, h)
    check_rounded(y, want, t)
    check_rounded(qh.rmsnorm(x, w, 1e-6), norm_formula(x, w, 1e-6), t)
    if n % 32 == 0:
        total, q, d = qh.rmsnorm_q8(x, w, 1e-6, residual=res)
        assert torch.equal(total, h)
        # the normalized rows in f32, rounded once: a 64-bit result next to a border of two f32 values is the only other way
        wq, wd = codes_of(oracle, want.float())
        assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(d.cpu().numpy(), wd)
        if t is torch.float32:  # and those of the call's own rows through qh_quantize_q8
            q2, d2 = qh.quantize_q8(y)
            assert torch.equal(q, q2) and torch.equal(d, d2)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n,ld,off", [(1, 96, 96, 1), (4, 96, 101, 3), (3, 1001, 1003, 5), (7, 33, 40, 2), (2, 2048, 5000, 9),
                                          (0, 64, 64, 0), (1, 1, 1, 1), (70, 5, 7, 1)])
@pytest.mark.parametrize("place", ["new", "x", "residual"])
def test_norm_strides(qh, gpu, dtype, rows, n, ld, off, place):
    t = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(rows + n)
    x, xb = guarded(rows, n, ld, off, t, gpu)
    r, rb = guarded(rows, n, ld + 2, off + 1, t, gpu)
    y, yb = guarded(rows, n, ld + 1, off + 2, t, gpu)
    s, sb = guarded(rows, n, ld + 3, off, t, gpu)
    x.copy_(torch.randn(rows, n, generator=gen, device=gpu))
    r.copy_(torch.randn(rows, n, generator=gen, device=gpu))
    x0, r0 = x.clone(), r.clone()
    w = torch.rand(n, generator=gen, device=gpu) + 0.5
    h = (x0.float() + r0.float()).to(t)
    to = {"new": s, "x": x, "residual": r}[place]
    total, got = qh.rmsnorm(x, w, 1e-5, residual=r, sum=to, out=y)
    assert total is to and got is y and torch.equal(to, h)
    check_rounded(y, norm_formula(h, w, 1e-5), t)
    for view, buf in ((x, xb), (r, rb), (y, yb), (s, sb)):
        assert untouched(buf, view)
    if place != "x":
        assert torch.equal(x, x0)
    if place != "residual":
        assert torch.equal(r, r0)


def test_norm_many_rows(qh, gpu):
    x = torch.randn(70001, 36, device=gpu)
    w = torch.randn(36, device=gpu)
    check_rounded(qh.rmsnorm(x, w), norm_formula(x, w, 1e-6), torch.float32)


def test_norm_far_rows(qh, gpu):
    """Rows past 4 GiB of their first one."""
    ld = (1 << 30) + 8
    buf = torch.empty(2 * ld, dtype=torch.float32, device=gpu)
    x = buf.view(2, ld)[:, :96]
    x.copy_(torch.randn(2, 96, device=gpu))
    w = torch.ones(96, device=gpu)
    want = norm_formula(x, w, 0.0)
    out = buf.view(2, ld)[:, 128:224]
    qh.rmsnorm(x, w, 0.0, out=out)
    check_rounded(out, want, torch.float32)


@pytest.mark.parametrize("n", [32, 896, 8192])
def test_norm_special_values(qh, gpu, n):
    """Squares past f32's range, zeros, infinities and NaN: the formula's results in 64 bits."""
    x = torch.randn(7, n, device=gpu)
    x[0] *= 1e38
    x[1] = 0.0
    x[2] *= 1e-30
    x[3, 5] = math.inf
    x[4, n - 1] = math.nan
    x[5] = 3.4e38
    w = torch.ones(n, device=gpu)
    for eps in (0.0, 1e-6):
        want = norm_formula(x, w, eps)
        got = qh.rmsnorm(x, w, eps)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        there = ~torch.isnan(want)
        check_rounded(got[there], want[there], torch.float32)
        q, d = qh.rmsnorm_q8(x, w, eps)
        q2, d2 = qh.quantize_q8(got)
        assert torch.equal(q, q2) and np.array_equal(d.cpu().numpy().view(np.uint32), d2.cpu().numpy().view(np.uint32))


def test_norm_sum_past_f16(qh, gpu):
    x = torch.full((2, 64), 40000.0, dtype=torch.float16, device=gpu)
    total, y = qh.rmsnorm(x, torch.ones(64, device=gpu), residual=x.clone())
    assert bool(torch.isinf(total).all()) and bool(torch.isnan(y).all())


# ------------------------------------------------------------------------------------------------------------- rope

def rope_formula(x, pos, turns, rot, interleaved, magnitude):
    """The rotation in 64 bits, and the bound of an f32 one's error before its rounding to x's type: cosine and sine are off
    by at most 4 * 2^-24 times the magnitude (argument, last two steps of the series, product with the magnitude: less than
    one each of values up to 1), one product is rounded by itself (2^-24 of it), and the sum once (2^-24)."""
    x = x.double()
    t = pos.double().view(-1, 1) * turns.double()
    angle = 2 * math.pi * (t - torch.round(t))
    c, s = (magnitude * torch.cos(angle)).unsqueeze(1), (magnitude * torch.sin(angle)).unsqueeze(1)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * c - b * s, a * s + b * c
    off = 2.0 ** -24 * ((a.abs() + b.abs()) * 4 * abs(magnitude) + torch.maximum(a.abs(), b.abs()) * abs(magnitude))
    out, err = x.clone(), torch.zeros_like(x)
    for v, (u, w) in ((out, (first, second)), (err, (off + 2.0 ** -24 * first.abs(), off + 2.0 ** -24 * second.abs()))):
        if interleaved:
            v[..., 0:rot:2], v[..., 1:rot:2] = u, w
        else:
            v[..., :rot // 2], v[..., rot // 2:rot] = u, w
    return out, err


def check_rope(got, x, pos, turns, rot, interleaved, magnitude=1.0):
    want, err = rope_formula(x, pos, turns, rot, interleaved, magnitude)
    if x.dtype is torch.float16:
        err = err + 2.0 ** -11 * (want.abs() + err) + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= err + 2.0 ** -149).all())
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (128, 128), (128, 48), (128, 2), (80, 80), (80, 22), (96, 50), (256, 256),
                                    (256, 254), (2, 2), (7, 4), (5, 2), (33, 30)])
def test_rope(qh, gpu, dtype, interleaved, hd, rot):
    t = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(hd + rot)
    rope = qh.Rope(hd, rot_dim=rot, interleaved=interleaved, theta=1e4, device=gpu)
    for rows, heads, kv in ((1, 1, 1), (3, 5, 1), (65, 14, 2)):
        q = torch.randn(rows, heads, hd, generator=gen, device=gpu).to(t)
        k = torch.randn(rows, kv, hd, generator=gen, device=gpu).to(t)
        pos = torch.randint(-3000, 200000, (rows,), generator=gen, device=gpu, dtype=torch.int32)
        pos[0] = 0 if rows > 1 else 77
        q2, k2 = rope(q, k, pos=pos)
        check_rope(q2, q, pos, rope.turns, rot, interleaved)
        check_rope(k2, k, pos, rope.turns, rot, interleaved)
        if rows > 1:
            assert torch.equal(q2[0], q[0]) and torch.equal(k2[0], k[0])  # position 0 turns nothing
        assert torch.equal(rope(q, pos=pos), q2)
        for a, b in ((q, q2), (k, k2)):  # in place, alone
            mine = a.clone()
            assert rope(mine, pos=pos, q_out=mine) is mine and torch.equal(mine, b)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_a_fused_row(qh, gpu, dtype, interleaved):
    """q and k as views of rows that hold queries, keys and values, at an odd offset, in place: the rest is left."""
    t, rows, heads, kv, hd = TYPES[dtype], 37, 6, 2, 64
    width = (heads + 2 * kv) * hd + 3
    buf = torch.randn(rows * width + 1, device=gpu).to(t)
    row = buf[1:].view(rows, width)
    q, k = row[:, :heads * hd].view(rows, heads, hd), row[:, heads * hd:(heads + kv) * hd].view(rows, kv, hd)
    before, q0, k0 = buf.clone(), q.clone(), k.clone()
    pos = torch.arange(rows, dtype=torch.int32, device=gpu) * 911
    rope = qh.Rope(hd, rot_dim=40, interleaved=interleaved, device=gpu)
    rope(q, k, pos=pos, q_out=q, k_out=k)
    check_rope(q, q0, pos, rope.turns, 40, interleaved)
    check_rope(k, k0, pos, rope.turns, 40, interleaved)
    after = buf[1:].view(rows, width)[:, (heads + kv) * hd:]
    assert torch.equal(after, before[1:].view(rows, width)[:, (heads + kv) * hd:]) and buf[0] == before[0]


@pytest.mark.parametrize("rows", [1, 2047, 2049, 9001])
def test_rope_rows(qh, gpu, rows):
    q = torch.randn(rows, 3, 64, device=gpu)
    pos = torch.arange(rows, dtype=torch.int32, device=gpu)
    rope = qh.Rope(64, device=gpu)
    check_rope(rope(q, pos=pos), q, pos, rope.turns, 64, False)


def test_rope_most_heads(qh, gpu):
    """4,096 heads, nearly all of each a copy: the most items that a token can have."""
    q, k = torch.randn(2, 4000, 256, device=gpu), torch.randn(2, 96, 256, device=gpu)
    rope = qh.Rope(256, rot_dim=2, device=gpu)
    pos = ints_of([5, -7], gpu)
    q2, k2 = rope(q, k, pos=pos)
    check_rope(q2, q, pos, rope.turns, 2, False)
    check_rope(k2, k, pos, rope.turns, 2, False)


def ints_of(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def test_rope_of_no_rows(qh, gpu):
    rope = qh.Rope(64, device=gpu)
    q = torch.empty(0, 4, 64, device=gpu)
    assert rope(q, pos=torch.empty(0, dtype=torch.int32, device=gpu)).shape == (0, 4, 64)


@pytest.mark.parametrize("scaling", [None, "linear", "base", "parts"])
def test_rope_far_positions(qh, gpu, scaling):
    """Positions up to int32's ends: the angle in 64 bits is off by 2^-53 of its turns (2^31 / 2 pi at most), 2^-22 of a turn,
    so these are checked against the same table's exact angle in whole numbers."""
    rope = qh.Rope(128, scaling=scaling, factor=8.0, context=32768.0, magnitude=1.25, device=gpu)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 123456789, -99999999], dtype=torch.int32, device=gpu)
    q = torch.randn(5, 2, 128, device=gpu)
    got = rope(q, pos=pos).double().cpu()
    from fractions import Fraction
    x = q.double().cpu()
    for r, p in enumerate(pos.tolist()):
        for i, f in enumerate(rope.turns.tolist()):
            exact = Fraction(f) * p
            angle = 2 * math.pi * float(exact - round(exact))
            c, s = 1.25 * math.cos(angle), 1.25 * math.sin(angle)
            # a product of 64 bits is off by 2^-53 of it
            slack = 2 * math.pi * 2.0 ** -53 * abs(p * f) * 1.25 + 2.0 ** -24 * 6 * 1.25
            for h in range(2):
                a, b = x[r, h, i].item(), x[r, h, i + 64].item()
                lim = slack * (abs(a) + abs(b)) + 2.0 ** -24 * 1.25 * (abs(a) + abs(b))
                assert abs(got[r, h, i].item() - (a * c - b * s)) <= lim
                assert abs(got[r, h, i + 64].item() - (a * s + b * c)) <= lim


def test_rope_own_table_and_back(qh, gpu):
    """A table of one's own, and the opposite positions: turned there and back is where it was, within both roundings."""
    turns = torch.rand(24, dtype=torch.float64) * 0.3
    rope = qh.Rope(64, rot_dim=48, turns=turns, device=gpu)
    q = torch.randn(50, 4, 64, device=gpu)
    pos = torch.randint(0, 100000, (50,), dtype=torch.int32, device=gpu)
    there = rope(q, pos=pos)
    check_rope(there, q, pos, turns.to(gpu), 48, False)
    again = rope(there, pos=-pos)
    lim = 2.0 ** -24 * 2 * 8 * 2 * q.double().abs().amax(-1, keepdim=True)
    assert bool(((again.double() - q.double()).abs() <= lim).all())


def test_rope_infinite_values_stay_in_their_pair(qh, gpu):
    q = torch.randn(4, 2, 64, device=gpu)
    q[1, 0, 3], q[2, 1, 40] = math.inf, math.nan
    pos = torch.arange(4, dtype=torch.int32, device=gpu)
    out = qh.Rope(64, rot_dim=48, device=gpu)(q, pos=pos)
    bad = ~torch.isfinite(out)
    assert sorted(map(tuple, bad.nonzero().tolist())) == [(1, 0, 3), (1, 0, 27), (2, 1, 16), (2, 1, 40)]


def test_rows_refuse_what_does_not_fit(qh, gpu):
    x, w = torch.randn(4, 64, device=gpu), torch.ones(64, device=gpu)
    pos = torch.zeros(4, dtype=torch.int32, device=gpu)
    rope = qh.Rope(64, device=gpu)
    bad = [lambda: qh.rmsnorm(x.double(), w), lambda: qh.rmsnorm(x.t(), w), lambda: qh.rmsnorm(x, w[:63]),
           lambda: qh.rmsnorm(x, w.cpu()), lambda: qh.rmsnorm(x.cpu(), w.cpu()), lambda: qh.rmsnorm(x, w, residual=x.half()),
           lambda: qh.rmsnorm(x, w, residual=x[:3]), lambda: qh.rmsnorm(x, w, out=x), lambda: qh.rmsnorm_q8(x[:, :33], w[:33]),
           lambda: qh.rmsnorm(x[0], w), lambda: qh.rmsnorm(x, w.half()),
           lambda: rope(x.view(4, 2, 32), pos=pos), lambda: rope(x.view(4, 1, 64), pos=pos.long()),
           lambda: rope(x.view(4, 1, 64), pos=pos[:3]), lambda: rope(x.view(4, 1, 64), x.view(4, 1, 64).half(), pos=pos),
           lambda: rope(x.view(4, 1, 64).cpu(), pos=pos.cpu()), lambda: rope(x.view(4, 1, 64).double(), pos=pos),
           lambda: rope(x.view(4, 1, 64), pos=pos, q_out=x.view(4, 1, 64)[:2]),
           lambda: qh.Rope(64, scaling="other", device=gpu), lambda: qh.Rope(64, rot_dim=65, device=gpu),
           lambda: qh.Rope(64, turns=torch.zeros(31, dtype=torch.float64), device=gpu),
           lambda: qh.Rope(64, turns=torch.zeros(32), device=gpu)]
    for call in bad:
        with pytest.raises(qh.QHError):
            call()


def test_rows_captured_and_on_other_streams(qh, gpu):
    """Both in a graph, replayed with new inputs and eager calls between the replays, and eagerly on a side stream."""
    x, res, w = torch.randn(9, 896, device=gpu), torch.randn(9, 896, device=gpu), torch.randn(896, device=gpu)
    q, pos = torch.randn(9, 14, 64, device=gpu), torch.arange(9, dtype=torch.int32, device=gpu)
    rope = qh.Rope(64, device=gpu)

    def both():
        return (*qh.rmsnorm_q8(x, w, residual=res), rope(q, pos=pos))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        pos.add_(1000 * i)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
