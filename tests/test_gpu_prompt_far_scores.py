"""Attention of packed prompts (qh_attention) with scores so large that their own rounding is more than 1: a key whose score stands out by
far more than that takes the whole weight, keys of one score share it, and nothing becomes NaN.

Scores here are multiples of one power of two with few bits, so that they are exact in f32 (and so is the order); the largest is ahead of
the next by 2^-7 of itself and 2^10 at least, so that no other key has a weight. What is left is the rounding of the weight and the result:
f16 2^-11 twice, f32 2^-22 of the second product's missing parts and a few of 2^-24; and for n keys of one score the rounding of their sum,
n 2^-24 in all."""
import pytest
import torch

from test_gpu_prompt import TYPES, ints

pytestmark = pytest.mark.gpu

SIZES = {"f16": [2.0 ** 8, 2.0 ** 12, 2.0 ** 15], "f32": [2.0 ** 8, 2.0 ** 15, 2.0 ** 30, 2.0 ** 55]}
CASES = [(t, s) for t in SIZES for s in SIZES[t]]


def close(got, want, dtype, n=1):
    tol = (2.0 ** -10 if dtype == "f16" else 2.0 ** -21) + n * 2.0 ** -24
    assert bool(torch.isfinite(got).all())
    # for one key the result is that key's value; for several, of their largest (dims may cancel)
    big = want.abs() if n == 1 else want.abs().amax().expand_as(want) * n ** 0.5
    assert bool(((got.double() - want).abs() <= tol * big + 2.0 ** -24).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [(1, 100), (200, 200), (20, 2000), (2100, 2100)])
@pytest.mark.parametrize("dtype,size", CASES)
def test_one_key_stands_out(qh, gpu, hd, off, causal, rows, keys, dtype, size):
    """Keys' scores from 33/64 to 61/64 of the largest in steps of 1/64, one of 1 and one of 1/2; the heads by turns take the largest and,
    with negative queries, the smallest. Rows whose best key is alone are compared, the others have to be finite."""
    t, heads, kv = TYPES[dtype], 4, 2
    if rows > 2000:
        heads, kv = 32, 16
    gen = torch.Generator(device=gpu).manual_seed(keys)
    q = torch.full((rows, heads, hd), size, device=gpu).to(t)
    q[:, 1::2] *= -1
    level = torch.randint(33, 62, (keys,), generator=gen, device=gpu) / 64.0
    level[17 if causal else int(torch.randint(20, keys, (1,), generator=gen, device=gpu))] = 1.0
    level[3] = 0.5
    buf = torch.empty(keys * 2 * kv * hd + off, device=gpu).to(t)
    row = buf[off:].view(keys, 2 * kv, hd)
    k, v = row[:, :kv], row[:, kv:]
    k.copy_((size * level).to(t).view(keys, 1, 1).expand_as(k))
    v.copy_(torch.randn(v.shape, generator=gen, device=gpu).to(t))
    got = qh.attention(q, k, v, ints([0, rows], gpu), ints([0, keys], gpu), causal=causal)
    assert bool(torch.isfinite(got).all())
    vis = torch.arange(keys - rows + 1, keys + 1, device=gpu) if causal else torch.full((rows,), keys, device=gpu)
    for h in range(heads):
        x = (level if h % 2 == 0 else -level).expand(rows, -1).masked_fill(torch.arange(keys, device=gpu) >= vis.view(-1, 1), -9.0)
        top = x.topk(2, dim=1)
        alone = top.values[:, 0] > top.values[:, 1]
        close(got[alone, h], v[top.indices[:, 0], h // (heads // kv)][alone].double(), dtype)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype,size", CASES)
def test_keys_of_one_score_share(qh, gpu, hd, sign, dtype, size):
    """Every key the same, with a score that is no power of two: the mean of the values; with far larger ones behind, the mean of those."""
    gen = torch.Generator(device=gpu).manual_seed(hd)
    keys, t = 700, TYPES[dtype]
    v = torch.randn(keys, 1, hd, generator=gen, device=gpu).to(t)
    q = torch.full((3, 2, hd), size * 1.25, device=gpu).to(t)
    k = torch.full((keys, 1, hd), sign * size * 1.375, device=gpu).to(t)
    for scale in (None, 0.1, -0.3):
        got = qh.attention(q, k, v, ints([0, 3], gpu), ints([0, keys], gpu), causal=False, scale=scale)
        close(got, v.double().mean(0).expand(3, 2, hd), dtype, keys)
    k[500:] = sign * size * 1.5
    got = qh.attention(q, k, v, ints([0, 3], gpu), ints([0, keys], gpu), causal=False)
    part = v[500:] if sign > 0 else v[:500]
    close(got, part.double().mean(0).expand(3, 2, hd), dtype, len(part))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("keys", [150, 1500])
def test_rows_next_to_far_ones(qh, gpu, hd, dtype, keys):
    """Rows of ordinary scores have the same bits whether their neighbours' scores are ordinary or far, from the first key on or later."""
    gen = torch.Generator(device=gpu).manual_seed(keys)
    q, k, v = (torch.randn(n, 4, hd, generator=gen, device=gpu).to(TYPES[dtype]) for n in (150, keys, keys))
    q[..., 1] = 0.0
    k[..., 1] = 0.0
    k[keys // 2:, :, 1] = 30000.0  # of weight for queries that have this dim alone
    starts = ints([0, 150], gpu), ints([0, keys], gpu)
    clean = qh.attention(q, k, v, *starts)
    q[7, 1, 1], q[40:43, :, 1] = 20000.0, -20000.0
    q[90, 2] *= 16000.0
    got = qh.attention(q, k, v, *starts)
    same = torch.ones(150, 4, dtype=torch.bool, device=gpu)
    same[7, 1] = same[40:43] = same[90, 2] = False
    assert torch.equal(got[same], clean[same])
    assert bool(torch.isfinite(got).all())
