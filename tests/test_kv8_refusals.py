"""The 8-bit paged cache's entry points refuse bad arguments on the host; no kernel is launched."""
import ctypes as C

import numpy as np
import pytest

from kv8_util import PlainKV8, nearest


def cache(qh, **kw):
    a = dict(pages=4096, table=4096, lens=4096, refs=4096, status=4096, n_layers=2, n_pages=8, page_tokens=32, n_kv_heads=2,
             head_dim=64, n_seqs=4, seq_pages=8)
    a.update(kw)
    return qh.qh_kv8_cache(*[a[n] for n, _ in qh.qh_kv8_cache._fields_])


P = C.c_void_p(4096)


def append(qh, c, layer=0, k=P, v=P, dtype=0, ldk=128, ldv=128, start=P, seqs=P, n=2, n_tok=5):
    return qh.lib().qh_kv8_append(C.byref(c), layer, k, v, dtype, ldk, ldv, start, seqs, n, n_tok, None)


def attend(qh, c, layer=0, q=P, out=C.c_void_p(8192), dtype=0, heads=4, ldq=256, ldo=256, start=P, seqs=P, n=2, n_tok=5,
           causal=1, scale=0.1, ws=P, ws_bytes=1 << 40):
    return qh.lib().qh_kv8_attention(C.byref(c), layer, q, out, dtype, heads, ldq, ldo, start, seqs, n, n_tok, causal,
                                     scale, ws, ws_bytes, None)


def test_page_bytes(qh):
    f = qh.lib().qh_kv8_page_bytes
    assert f(64, 2, 64) == 2 * 2 * 64 * 64 + 128  # codes, and 16 scales padded to a line
    assert f(256, 8, 128) == 2 * 8 * 256 * 128 + 2 * 8 * 16 * 4
    for bad in ((8, 2, 64), (48, 2, 64), (512, 2, 64), (64, 0, 64), (64, 2, 96), (64, 2, 256), (64, 257, 64)):
        assert f(*bad) == 0, bad


@pytest.mark.parametrize("change,code", [
    ({"pages": 0}, 1), ({"table": 0}, 1), ({"lens": 0}, 1), ({"refs": 0}, 1), ({"status": 0}, 1), ({"pages": 4104}, 4),
    ({"page_tokens": 24}, 3), ({"head_dim": 80}, 3), ({"n_kv_heads": 0}, 3), ({"n_layers": 0}, 3), ({"n_pages": 0}, 3),
    ({"n_pages": (1 << 20) + 1}, 3), ({"n_seqs": 0}, 3), ({"n_seqs": 32769}, 3), ({"seq_pages": 0}, 3),
    ({"seq_pages": 1 << 26}, 3),
])
def test_bad_caches_are_refused_by_every_call(qh, change, code):
    L, c = qh.lib(), cache(qh, **change)
    r = C.byref(c)
    assert L.qh_kv8_reset(r, None) == code
    assert L.qh_kv8_resize(r, P, P, 1, P, 1 << 40, None) == code
    assert L.qh_kv8_fork(r, P, P, 1, 0, P, 1 << 40, None) == code
    assert L.qh_kv8_compact(r, None, P, 1 << 40, None) == code
    assert append(qh, c) == code and attend(qh, c) == code
    assert L.qh_kv8_read(r, 0, P, P, 0, 128, 128, P, P, 2, 5, None) == code
    assert L.qh_kv8_pages_workspace_bytes(r) == 0 and L.qh_kv8_attention_workspace_bytes(r, 4, 2, 5) == 0


def test_null_cache(qh):
    L = qh.lib()
    assert L.qh_kv8_reset(None, None) == 1 and L.qh_kv8_compact(None, None, P, 1 << 40, None) == 1
    assert L.qh_kv8_attention_workspace_bytes(None, 4, 2, 5) == 0


@pytest.mark.parametrize("change,code", [
    ({"layer": -1}, 1), ({"layer": 2}, 1), ({"n": -1}, 1), ({"n_tok": -1}, 1), ({"start": None}, 1), ({"dtype": 2}, 2),
    ({"k": None}, 1), ({"v": None}, 1), ({"ldk": 127}, 1), ({"ldv": 64}, 1), ({"ldk": 130}, 4), ({"k": C.c_void_p(4100)}, 4),
    ({"dtype": 1, "ldk": 132}, 4), ({"n": 1 << 23}, 3), ({"n_tok": 1 << 29}, 3),
])
def test_append_refusals(qh, change, code):
    assert append(qh, cache(qh), **change) == code
    assert qh.lib().qh_last_error()


@pytest.mark.parametrize("change,code", [
    ({"layer": 2}, 1), ({"heads": 3}, 3), ({"heads": 0}, 3), ({"start": None}, 1), ({"causal": 2}, 1),
    ({"scale": float("nan")}, 1), ({"scale": float("inf")}, 1), ({"scale": -3e38}, 1), ({"dtype": 3}, 2), ({"q": None}, 1), ({"out": None}, 1),
    ({"ldq": 255}, 1), ({"ldo": 258}, 4), ({"out": C.c_void_p(4104)}, 4), ({"ws": C.c_void_p(4104)}, 4),
    ({"n_tok": 1 << 30}, 3), ({"n": 1 << 24}, 3), ({"n_tok": 1 << 29, "n": 1}, 3), ({"out": P, "q": P}, 1),
])
def test_attention_refusals(qh, change, code):
    assert attend(qh, cache(qh), **change) == code


def test_attention_workspace_is_checked(qh, monkeypatch):
    c = cache(qh, seq_pages=128)
    need = qh.lib().qh_kv8_attention_workspace_bytes(C.byref(c), 4, 2, 5)
    assert need > 0 and attend(qh, c, ws_bytes=need - 1) == 6 and attend(qh, c, ws=None) == 6
    assert qh.lib().qh_kv8_attention_workspace_bytes(C.byref(c), 4, 0, 0) == 0


def test_page_call_refusals(qh):
    L, c = qh.lib(), cache(qh)
    r, need = C.byref(c), qh.lib().qh_kv8_pages_workspace_bytes(C.byref(c))
    assert need > 0
    for f in (lambda *a: L.qh_kv8_resize(r, *a, None),
              lambda s, l, n, ws, b: L.qh_kv8_fork(r, s, l, n, 1, ws, b, None)):
        assert f(P, P, 5, P, need) == 1 and f(P, P, -1, P, need) == 1  # more entries than sequences
        assert f(None, P, 1, P, need) == 1 and f(P, None, 1, P, need) == 1
        assert f(P, P, 1, P, need - 1) == 6 and f(P, P, 1, None, need) == 6
        assert f(P, P, 1, C.c_void_p(4104), need) == 4
        assert f(P, P, 0, None, 0) == 0  # nothing to do
    assert L.qh_kv8_fork(r, P, P, 1, 2, P, need, None) == 1
    assert L.qh_kv8_compact(r, None, P, need - 1, None) == 6


def test_empty_batches_do_nothing(qh):
    c = cache(qh)
    assert append(qh, c, n=0, n_tok=0, k=None, v=None) == 0 and attend(qh, c, n_tok=0, q=None, ws=None) == 0
    assert append(qh, c, n=0, n_tok=5) == 0


def test_plain_model_rounds_as_the_definition_says():
    assert nearest(np.array([0.5, -0.5, 1.4999999, -2.5])).tolist() == [1.0, -1.0, 1.0, -3.0]
    m = PlainKV8(1, 2, 16, 1, 64, 1, 2)
    m.resize([0], [2])
    x = np.zeros((2, 1, 64), np.float32)
    x[0, 0, 0], x[1, 0, 0] = 127.0, 63.5
    m.append(0, [0], [2], x, x)
    assert m.values(0, 0)[0][:, 0, 0].tolist() == [127.0, 64.0]
    m.resize([0], [3])
    m.append(0, [0], [1], 2 * x[:1], x[:1])  # the scale doubles: 64 -> 32
    assert m.values(0, 0)[0][:, 0, 0].tolist() == [128.0, 64.0, 254.0]


def test_decoder_refuses_a_cache_of_another_device(qh):
    from types import SimpleNamespace as N
    with pytest.raises(qh.QHError, match="decoder on cuda:0"):
        qh.Decoder.bind_kv8(N(buf=N(device="cuda:0"), h=None), N(device="cuda:1"))
