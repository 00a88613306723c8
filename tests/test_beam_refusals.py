"""The beam entry points (qh_beam_select, qh_kv8_reorder) refuse bad arguments on the host; no kernel is launched."""
import ctypes as C

import pytest

from test_kv8_refusals import cache

P = C.c_void_p(4096)
A, B, D, W = (C.c_void_p(x) for x in (8192, 16384, 32768, 65536))


def select(qh, logits=P, dtype=0, ld=1000, scores=A, prompts=2, beams=3, n_valid=1000, k=6, parent=B, token=D,
           score=C.c_void_p(1 << 20), ws=W, ws_bytes=1 << 40):
    return qh.lib().qh_beam_select(logits, dtype, ld, scores, prompts, beams, n_valid, k, parent, token, score, ws, ws_bytes,
                                   None)


@pytest.mark.parametrize("change,code", [
    ({"logits": None}, 1), ({"dtype": 2}, 2), ({"ld": 999}, 1), ({"prompts": -1}, 3), ({"beams": 0}, 3), ({"beams": 257}, 3),
    ({"n_valid": 0}, 3), ({"n_valid": 262145, "ld": 262145}, 3), ({"prompts": 1 << 16}, 3), ({"prompts": 1 << 17, "beams": 1}, 3), ({"prompts": 1 << 30}, 3), ({"k": 0}, 7),
    ({"k": 257}, 7), ({"parent": None}, 1), ({"token": None}, 1), ({"score": None}, 1), ({"score": A}, 1), ({"ws": None}, 6),
    ({"ws_bytes": 0}, 6), ({"ws": C.c_void_p(65544)}, 4), ({"logits": C.c_void_p(4098)}, 4), ({"scores": C.c_void_p(8194)}, 4),
    ({"dtype": 1, "logits": C.c_void_p(4097)}, 4), ({"token": C.c_void_p(32770)}, 4),
])
def test_select_refusals(qh, change, code):
    assert select(qh, **change) == code
    assert qh.lib().qh_last_error()


def test_select_of_no_prompts(qh):
    assert select(qh, prompts=0, logits=None) == 0


def test_select_workspace(qh):
    f = qh.lib().qh_beam_workspace_bytes
    for dtype in (0, 1):
        need = f(dtype, 2, 3, 1000)
        assert 0 < need < 6 * 1000
        assert select(qh, dtype=dtype, ws_bytes=need - 1) == 6
        assert f(dtype, 24, 8, 151936) < 24 * 8 * 151936 // 16  # far below the logits
    assert f(0, 0, 3, 1000) == 0
    for bad in ((2, 2, 3, 1000), (0, -1, 3, 1000), (0, 2, 0, 1000), (0, 2, 257, 1000), (0, 2, 3, 0), (0, 2, 3, 262145)):
        assert f(*bad) == 0, bad


@pytest.mark.parametrize("change,code", [
    ({"pages": 0}, 1), ({"table": 0}, 1), ({"pages": 4104}, 4), ({"page_tokens": 24}, 3), ({"n_seqs": 0}, 3), ({"seq_pages": 0}, 3),
])
def test_reorder_refuses_bad_caches(qh, change, code):
    c = cache(qh, **change)
    assert qh.lib().qh_kv8_reorder(C.byref(c), P, P, 1, P, 1 << 40, None) == code
    assert qh.lib().qh_kv8_reorder_workspace_bytes(C.byref(c)) == 0


def test_reorder_lists_and_workspace(qh):
    L = qh.lib()
    small, large = cache(qh), cache(qh, n_seqs=100, seq_pages=100)
    assert L.qh_kv8_reorder(None, P, P, 1, P, 1 << 40, None) == 1
    assert L.qh_kv8_reorder_workspace_bytes(C.byref(small)) == 0
    need = L.qh_kv8_reorder_workspace_bytes(C.byref(large))
    assert need >= 4 * 100 * 100
    assert L.qh_kv8_reorder(C.byref(small), None, P, 1, None, 0, None) == 1
    assert L.qh_kv8_reorder(C.byref(small), P, P, -1, None, 0, None) == 1
    assert L.qh_kv8_reorder(C.byref(small), P, P, 5, None, 0, None) == 1
    assert L.qh_kv8_reorder(C.byref(small), P, P, 0, None, 0, None) == 0
    assert L.qh_kv8_reorder(C.byref(large), P, P, 1, None, 0, None) == 6
    assert L.qh_kv8_reorder(C.byref(large), P, P, 1, P, need - 1, None) == 6
    assert L.qh_kv8_reorder(C.byref(large), P, P, 1, C.c_void_p(4104), need, None) == 4
