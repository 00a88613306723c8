"""qh_attention refuses bad arguments on the host; no kernel is launched."""
import ctypes as C
import math

import pytest

Q, K, V, O, S, W = (C.c_void_p(x) for x in (1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20))


def attend(qh, q=Q, k=K, v=V, out=O, dtype=0, heads=4, kv=2, hd=64, ldq=256, ldk=128, ldv=128, ldo=256, start=S, kstart=None, n=2,
           n_tok=9, n_keys=9, causal=1, scale=0.125, ws=W, ws_bytes=1 << 40):
    return qh.lib().qh_attention(q, k, v, out, dtype, heads, kv, hd, ldq, ldk, ldv, ldo, start, kstart, n, n_tok, n_keys, causal,
                                 scale, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, 1), ({"k": None}, 1), ({"v": None}, 1), ({"out": None}, 1), ({"dtype": 2}, 2), ({"heads": 3}, 3), ({"heads": 0}, 3),
    ({"kv": 0}, 3), ({"kv": 257, "heads": 257}, 3), ({"hd": 80}, 3), ({"hd": 256}, 3), ({"ldq": 255}, 1), ({"ldk": 127}, 1),
    ({"ldv": 127}, 1), ({"ldo": 255}, 1), ({"start": None}, 1), ({"n": -1}, 1), ({"n_tok": -1}, 1), ({"n_keys": -1}, 1),
    ({"n_keys": 10}, 1), ({"causal": 2}, 1), ({"scale": math.nan}, 1), ({"scale": math.inf}, 1), ({"scale": -2e38}, 1),
    ({"q": C.c_void_p(4098)}, 4), ({"dtype": 1, "k": C.c_void_p(4097)}, 4), ({"out": Q}, 1), ({"out": K}, 1), ({"out": V}, 1),
    ({"ws": C.c_void_p(8)}, 4), ({"n_tok": 1 << 30, "n_keys": 1 << 30}, 3), ({"n": 1 << 23}, 3), ({"heads": 1 << 17, "kv": 1}, 3),
    ({"n_keys": (1 << 30) + 1, "kstart": S}, 3),
])
def test_refusals(qh, change, code):
    assert attend(qh, **change) == code
    assert qh.lib().qh_last_error()


def test_nothing_to_do(qh):
    assert attend(qh, n=0) == 0 and attend(qh, n_tok=0, n_keys=0, q=None, k=None, v=None, out=None) == 0


def test_workspace(qh):
    f = qh.lib().qh_attention_workspace_bytes
    for shape in ((2, 4, 2, 64, 1, 9, 9), (0, 3, 2, 64, 1, 9, 9), (0, 4, 2, 80, 1, 9, 9), (0, 4, 2, 64, -1, 9, 9), (0, 4, 2, 64, 0, 9, 9),
                  (0, 4, 2, 64, 1, 0, 9)):
        assert f(*shape) == 0, shape
