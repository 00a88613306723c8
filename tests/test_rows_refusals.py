"""The row operators' entry points refuse bad arguments on the host, and the rotation's table is right; no kernel is
launched."""
import ctypes as C
import math

import numpy as np
import pytest

P = C.c_void_p(4096)
A, B, D, E = (C.c_void_p(x) for x in (8192, 16384, 32768, 65536))


def norm(qh, x=P, res=A, w=P, dtype=0, ldx=64, ldr=64, n_tok=3, n=64, eps=1e-6, sum=A, lds=64, y=None, ldy=64, q=B, d=D):
    return qh.lib().qh_rmsnorm(x, res, w, dtype, ldx, ldr, n_tok, n, eps, sum, lds, y, ldy, q, d, None)


@pytest.mark.parametrize("change,code", [
    ({"x": None}, 1), ({"w": None}, 1), ({"dtype": 2}, 2), ({"dtype": -1}, 2), ({"n_tok": -1}, 3), ({"n_tok": 1 << 24}, 3),
    ({"n_tok": 1 << 23, "n": 2080, "ldx": 2080, "ldr": 2080, "lds": 2080}, 3),
    ({"n_tok": 1 << 22, "n": 8224, "ldx": 8224, "ldr": 8224, "lds": 8224}, 3), ({"n": 0}, 3), ({"n": 32769}, 3), ({"n": 48, "ldx": 48}, 3), ({"eps": -1.0}, 1), ({"eps": math.nan}, 1),
    ({"eps": math.inf}, 1), ({"q": None}, 1), ({"d": None}, 1), ({"q": None, "d": None}, 1), ({"ldx": 63}, 1), ({"ldr": 63}, 1),
    ({"lds": 63}, 1), ({"y": E, "ldy": 63}, 1), ({"x": C.c_void_p(4098)}, 4), ({"dtype": 1, "x": C.c_void_p(4097)}, 4),
    ({"q": C.c_void_p(8200)}, 4), ({"d": C.c_void_p(8194)}, 4), ({"w": C.c_void_p(4098)}, 4), ({"y": P}, 1), ({"y": A}, 1),
    ({"lds": 128}, 1), ({"sum": P, "lds": 128}, 1), ({"ldx": (1 << 32) + 1}, 1),
])
def test_norm_refusals(qh, change, code):
    assert norm(qh, **change) == code
    assert qh.lib().qh_last_error()


def test_norm_of_no_rows(qh):
    assert norm(qh, n_tok=0) == 0


def rows(qh, x=4096, out=8192, ld=512, ldo=512, heads=4):
    return qh.qh_rope_rows(x, out, ld, ldo, heads)


def rope(qh, turns=P, rot=64, inter=0, mag=1.0, hd=64, q=None, k="none", dtype=0, pos=P, n_tok=3):
    q = rows(qh) if q is None else q
    kk = None if k == "none" else C.byref(k)
    return qh.lib().qh_rope(turns, rot, inter, mag, hd, C.byref(q), kk, dtype, pos, n_tok, None)


@pytest.mark.parametrize("change,code", [
    ({"turns": None}, 1), ({"turns": C.c_void_p(4100)}, 4), ({"rot": 0}, 3), ({"rot": 63}, 3), ({"rot": 66}, 3),
    ({"rot": 258, "hd": 258}, 3), ({"hd": 512}, 3), ({"inter": 2}, 1), ({"mag": math.nan}, 1), ({"mag": math.inf}, 1),
    ({"dtype": 2}, 2), ({"pos": None}, 1), ({"pos": C.c_void_p(4098)}, 1), ({"n_tok": -1}, 3), ({"n_tok": 1 << 24}, 3),
])
def test_rope_refusals(qh, change, code):
    assert rope(qh, **change) == code
    assert qh.lib().qh_last_error()


@pytest.mark.parametrize("change,code", [
    ({"x": None}, 1), ({"out": None}, 1), ({"ld": 255}, 1), ({"ldo": 255}, 1), ({"heads": 0}, 3), ({"heads": 4097}, 3),
    ({"x": 4098}, 4), ({"out": 8194}, 4), ({"out": 4096, "ldo": 256}, 1),
])
def test_rope_row_refusals(qh, change, code):
    assert rope(qh, q=rows(qh, **change)) == code
    other = rows(qh, x=1 << 20, out=1 << 21)
    assert rope(qh, q=other, k=rows(qh, **change)) == code


def test_rope_of_shared_rows_and_no_rows(qh):
    a = rows(qh)
    assert rope(qh, q=a, k=rows(qh, x=1 << 20)) == 1          # both results in one place
    assert rope(qh, q=a, k=rows(qh, x=1 << 20, out=4096)) == 1  # k's result over q
    assert rope(qh, q=a, k=rows(qh, x=8192, out=1 << 20)) == 1  # q's result over k
    assert rope(qh, q=rows(qh, heads=2049, ld=1 << 18, ldo=1 << 18), k=rows(qh, x=1 << 20, out=1 << 21, heads=2048, ld=1 << 18, ldo=1 << 18)) == 3
    assert rope(qh, n_tok=0) == 0
    assert qh.lib().qh_rope(P, 64, 0, 1.0, 64, None, None, 0, P, 3, None) == 1


def turns(qh, **kw):
    a = dict(theta=1e4, rot_dim=64, scaling=0, factor=1.0, context=0.0, low=0.0, high=0.0)
    a.update(kw)
    out = np.full(max(a["rot_dim"], 2) // 2 + 1, -1.0)
    rc = qh.lib().qh_rope_turns(C.byref(qh.qh_rope_desc(*[a[n] for n, _ in qh.qh_rope_desc._fields_])), out.ctypes.data)
    assert out[-1] == -1.0 or a["rot_dim"] % 2
    return rc, out[:-1]


@pytest.mark.parametrize("rot", [2, 4, 64, 100, 256])
@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
def test_turns(qh, rot, scaling):
    rc, got = turns(qh, rot_dim=rot, scaling=scaling, factor=4.0, context=4096.0, low=1.0, high=32.0)
    assert rc == 0
    for i, g in enumerate(got):
        base = 1e4 if scaling != 2 or rot == 2 else 1e4 * 4.0 ** (rot / (rot - 2))
        f = base ** (-2 * i / rot) / math.tau
        if scaling == 1:
            f /= 4
        if scaling == 3:
            made = 4096 * f  # turns over the trained context
            keep = 1.0 if made >= 32 else 0.0 if made <= 1 else (made - 1) / 31
            f = keep * f + (1 - keep) * f / 4
        assert abs(g - f) <= 1e-14 * f  # a few roundings of 64 bits
    if scaling == 2 and rot > 2:  # the slowest pair is divided by factor, the first by nothing
        plain = turns(qh, rot_dim=rot)[1]
        assert got[0] == plain[0] and abs(got[-1] * 4 / plain[-1] - 1) < 1e-13


@pytest.mark.parametrize("change,code", [
    ({"rot_dim": 0}, 3), ({"rot_dim": 63}, 3), ({"rot_dim": 258}, 3), ({"scaling": 4}, 1), ({"scaling": -1}, 1), ({"theta": 0.0}, 1),
    ({"theta": math.nan}, 1), ({"theta": math.inf}, 1), ({"scaling": 1, "factor": 0.0}, 1), ({"scaling": 2, "factor": math.nan}, 1),
    ({"scaling": 3, "context": 0.0, "high": 1.0}, 1), ({"scaling": 3, "context": 9.0, "low": 2.0, "high": 2.0}, 1),
    ({"scaling": 3, "context": 9.0, "low": -1.0, "high": 2.0}, 1),
])
def test_turn_refusals(qh, change, code):
    assert turns(qh, **change)[0] == code


def test_null_turns(qh):
    assert qh.lib().qh_rope_turns(None, P) == 1
