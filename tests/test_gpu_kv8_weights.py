"""Every single attention weight of the 8-bit cache, read off through values that are one-hot per position."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("hd,n", [(64, 33), (64, 49), (64, 64), (128, 128), (128, 100)])
def test_each_weight_in_f32(qh, gpu, hd, n, single):
    """Small scores, so that a weight's relative error is the rounding of its two halves, its exponential and the sum:
    2^-22 and 16 + n roundings of 2^-24 at most."""
    import torch
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    heads = 40
    c = qh.KV8Cache(1, 8, 32, 1, hd, 1, 8)
    c.resize(ints([0]), ints([n]))
    k = torch.randn(n, 1, hd, device="cuda", generator=gen)
    v = torch.zeros(n, 1, hd, device="cuda")
    v[torch.arange(n), 0, torch.arange(n)] = 1
    c.append(0, k, v, start=ints([0, n]))
    keys, values = c.read(0, n, start=ints([0, n]))
    assert torch.equal(values, v)  # 127 * (1 / 127 rounded) rounds to 1
    rows = 1 if single else n
    q = torch.randn(rows, heads, hd, device="cuda", generator=gen) * 1e-3
    got = c.attention(0, q, start=None if single else ints([0, n]))[:, :, :n].double().cpu().numpy()
    s = np.einsum("rhd,nd->rhn", q.double().cpu().numpy(), keys[:, 0].double().cpu().numpy()) * hd ** -0.5
    see = np.arange(n)[None, None] <= np.arange(n - rows, n)[:, None, None]
    e = np.where(see, np.exp(s), 0.0)
    want = e / e.sum(-1, keepdims=True)
    bound = want * (2.0 ** -22 + (16 + n) * 2.0 ** -24) + 2.0 ** -30
    assert (np.abs(got - want) <= bound).all(), (np.argwhere(np.abs(got - want) > bound)[:5], np.abs(got - want).max())
