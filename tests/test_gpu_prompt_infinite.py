"""Attention of packed prompts (qh_attention) where rows see values that are infinite: the formula gives the infinity in that dim
however small its weight is, NaN where both infinities or a NaN are seen, and nothing of it where it is hidden. Weights below f16's,
and f32's, smallest next to the row's others; infinities in the first tiles, in tiles that all rows see and in the last; a base that moves
after one; keys shared out between workgroups, whose parts are joined."""
import math

import pytest
import torch

from test_gpu_prompt import TYPES, check, formula, ints

pytestmark = pytest.mark.gpu


def inputs(gpu, dtype, rows, keys, heads, kv, hd, low, off=0):
    """Random q, k, v; the keys named by `low` (a slice) score about 200 less than the others for every row. off: elements before k
    and v, which then lie on no multiple of 16 bytes."""
    gen = torch.Generator(device=gpu).manual_seed(hd + keys)
    q = torch.randn(rows, heads, hd, generator=gen, device=gpu) * 0.5
    buf = torch.randn(keys * 2 * kv * hd + off, generator=gen, device=gpu) * 0.5
    q[..., 0] = 40.0
    buf = buf.to(TYPES[dtype])
    row = buf[off:].view(keys, 2 * kv, hd)
    k, v = row[:, :kv], row[:, kv:]
    k[..., 0] = 0.0
    k[low, :, 0] = -5.0 * hd ** 0.5
    return q.to(TYPES[dtype]), k, v


# rows, keys, which keys weigh nothing: one row tile and several; more keys than rows (shared out), a batch that fills the card
SHAPES = [(200, 200, slice(0, 70)), (130, 700, slice(0, 400)), (1, 3000, slice(0, 1500)), (40, 1100, slice(500, 900)),
          (2100, 2100, slice(0, 1000))]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys,low", SHAPES)
def test_infinite_values_of_small_weights(qh, gpu, dtype, hd, off, causal, rows, keys, low):
    heads, kv = (32, 16) if rows > 2000 else (4, 2)
    q, k, v = inputs(gpu, dtype, rows, keys, heads, kv, hd, low, off)
    a, b = low.start, low.stop
    v[a, 0, 0], v[a + 3, 0, 1], v[b - 1, 0, hd - 1] = math.inf, -math.inf, math.inf   # weigh nothing
    v[a + 5, 1, 3], v[b - 2, 1, 3] = math.inf, -math.inf                              # both in one dim: NaN where both are seen
    v[a + 6, 1, 4], v[b - 1, 1, 5] = math.nan, math.inf
    v[b, 1, 7], v[keys - 1, 1, 8] = -math.inf, math.inf                               # weighs as much as others, and the last
    st, kst = [0, rows], [0, keys]
    got = qh.attention(q, k, v, ints(st, gpu), ints(kst, gpu), causal=causal)
    check(got, *formula(q, k, v, st, kst, causal, hd ** -0.5))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_infinite_value_before_a_base_that_moves(qh, gpu, dtype, hd):
    """An infinity that weighs as much as its neighbours, and keys of far larger scores behind it: what was summed is scaled by 0."""
    for rows, keys in ((64, 1000), (900, 900)):
        q, k, v = inputs(gpu, dtype, rows, keys, 4, 2, hd, slice(0, 0))
        for at, up in ((100, 5.0), (400, 10.0), (650, 15.0)):
            k[at:, :, 0] = up * hd ** 0.5
        v[2, 0, 1], v[130, 0, 2], v[420, 1, hd - 2] = math.inf, -math.inf, math.inf
        st, kst = [0, rows], [0, keys]
        for causal in (True, False):
            got = qh.attention(q, k, v, ints(st, gpu), ints(kst, gpu), causal=causal)
            check(got, *formula(q, k, v, st, kst, causal, hd ** -0.5))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_batch_of_entries_with_and_without(qh, gpu, dtype):
    """Entries next to each other, one of which sees an infinity of no weight: the others' rows as they are without it."""
    st = [0, 90, 180, 400]
    q, k, v = inputs(gpu, dtype, 400, 400, 4, 2, 64, slice(90, 150))
    clean = qh.attention(q, k, v, ints(st, gpu))
    v[95, 1, 9], v[399, 0, 0] = -math.inf, math.inf
    got = qh.attention(q, k, v, ints(st, gpu))
    check(got, *formula(q, k, v, st, st, True, 0.125))
    assert torch.equal(got[:95], clean[:95]) and torch.equal(got[180:399], clean[180:399])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [(150, 150), (3, 2500), (70, 900), (2100, 2100)])
@pytest.mark.parametrize("share", [0.001, 0.3, 1.0])
def test_many_values_that_are_not_finite(qh, gpu, dtype, hd, causal, rows, keys, share):
    """Infinities of both signs and NaN all over, up to every value; large keys among the last, so that early ones weigh nothing."""
    heads, kv = (32, 16) if rows > 2000 else (4, 2)
    q, k, v = inputs(gpu, dtype, rows, keys, heads, kv, hd, slice(0, keys // 2))
    gen = torch.Generator(device=gpu).manual_seed(rows)
    there = torch.rand(v.shape, generator=gen, device=gpu) < share
    kinds = torch.tensor([math.nan, math.inf, -math.inf, math.inf, -math.inf, math.inf], device=gpu).to(v.dtype)
    # dims of +infinity alone, of both, and of all three
    kind = kinds[torch.randint(0, 6, v.shape, generator=gen, device=gpu)]
    kind[..., ::3] = math.inf
    kind[..., 1::3] = kind[..., 1::3].nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf)
    v.copy_(torch.where(there, kind, v))
    st, kst = [0, rows], [0, keys]
    got = qh.attention(q, k, v, ints(st, gpu), ints(kst, gpu), causal=causal)
    check(got, *formula(q, k, v, st, kst, causal, hd ** -0.5))
