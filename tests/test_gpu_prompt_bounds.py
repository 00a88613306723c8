"""Attention of packed prompts (qh_attention): f32 values near the type's smallest, and a sequence alone against the same one in a batch.

Small f32 values. The largest weight of a row is 2^-L at least, with 2^L at most 2^10 times the keys (so that f32's largest values do not
overflow), and their products are summed in f32: where a sum falls below 2^-126 each of the 6 products of a key may round by 2^-150,
6 keys 2^-150 in all, and the division by a sum of weights of 2^-L and more makes that 6 keys 2^-150 2^10 keys < keys^2 2^-137. The
three bf16 of a value below 2^-110 end at bf16's smallest, 2^-133: a value is off by 2^-132 at most. Both come on top of the bound that
holds for other values."""
import pytest
import torch

from test_gpu_prompt import TYPES, check, formula, ints, starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,keys", [(1, 1), (3, 70), (150, 200), (40, 1000), (5, 5000)])
@pytest.mark.parametrize("wide", [0.0, 1.0, 20.0])
@pytest.mark.parametrize("size", [-80, -95, -105, -115, -125, -135])
def test_small_f32_values(qh, gpu, hd, rows, keys, wide, size):
    """Values of one small size, under equal weights, ordinary ones and one that outweighs the others."""
    gen = torch.Generator(device=gpu).manual_seed(keys)
    q = torch.randn(rows, 4, hd, generator=gen, device=gpu) * wide
    k = torch.randn(keys, 2, hd, generator=gen, device=gpu)
    v = torch.randn(keys, 2, hd, generator=gen, device=gpu) * 2.0 ** size
    got = qh.attention(q, k, v, ints([0, rows], gpu), ints([0, keys], gpu))
    want, err, mine = formula(q, k, v, [0, rows], [0, keys], True, hd ** -0.5)
    check(got, want, err + keys ** 2 * 2.0 ** -137 + 2.0 ** -132, mine)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("rows,behind", [([300, 1, 77, 512, 40], 0), ([1500, 1500, 800], 0), ([4, 4, 60, 1], 700)])
def test_a_sequence_alone(qh, gpu, dtype, heads, kv, hd, rows, behind):
    """What else is in a batch decides how keys are shared out and rows are cut into tiles, and with them the order of sums: a
    sequence's rows alone and in the batch are within the bounds of both of each other."""
    gen = torch.Generator(device=gpu).manual_seed(len(rows))
    keys = [m + behind for m in rows]
    st, kst = starts(rows), starts(keys)
    shapes = ((st[-1], heads, hd), (kst[-1], kv, hd), (kst[-1], kv, hd))
    q, k, v = (torch.randn(shape, generator=gen, device=gpu).to(TYPES[dtype]) for shape in shapes)
    got = qh.attention(q, k, v, ints(st, gpu), ints(kst, gpu))
    want, err, mine = formula(q, k, v, st, kst, True, hd ** -0.5)
    check(got, want, err, mine)
    for i in range(len(rows)):
        a, b, c, d = st[i], st[i + 1], kst[i], kst[i + 1]
        alone = qh.attention(q[a:b], k[c:d], v[c:d], ints([0, b - a], gpu), ints([0, d - c], gpu))
        check(alone, got[a:b].double(), 2 * err[a:b], mine[a:b])
