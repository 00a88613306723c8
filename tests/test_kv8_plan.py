"""qh_kv8_attention_plan on the host: its refusals, and the limits of one launch."""
import ctypes as C

import pytest

from test_kv8_refusals import cache


def plan(qh, c, heads=4, n=2, n_tok=5, single=0):
    p = qh.qh_kv8_plan()
    return qh.lib().qh_kv8_attention_plan(C.byref(c), heads, n, n_tok, single, C.byref(p)), p


def test_refusals(qh):
    c = cache(qh)
    assert plan(qh, c)[0] == 0
    for kw, code in (({"heads": 3}, 3), ({"heads": 0}, 3), ({"n": 0}, 1), ({"n_tok": 0}, 1), ({"single": 1}, 1), ({"n": -1}, 1),
                     ({"n_tok": 1 << 30}, 3)):
        assert plan(qh, c, **kw)[0] == code, kw
    assert plan(qh, cache(qh, head_dim=80))[0] == 3
    assert qh.lib().qh_kv8_attention_plan(C.byref(c), 4, 2, 5, 0, None) == 1


@pytest.mark.parametrize("seq_pages,entries,launches", [(1 << 22, 64, 1), (1 << 22, 65, 2), (1 << 22, 1000, 16), (1 << 18, 1024, 1),
                                                        (1 << 18, 1025, 2)])
def test_a_launch_counts_its_tiles_in_an_int(qh, seq_pages, entries, launches):
    """2^30 tiles of 64 positions at most."""
    c = cache(qh, page_tokens=256, seq_pages=seq_pages, n_kv_heads=1)
    rc, p = plan(qh, c, heads=2, n=entries, n_tok=entries, single=1)
    assert rc == 0 and p.kernel == qh.KV8_SHARES and p.launches == launches
    # with starts, as many entries go to the kernel of many rows, which counts each entry's tiles alone
    rc, p = plan(qh, c, heads=2, n=entries, n_tok=entries)
    assert rc == 0 and p.kernel == (qh.KV8_SHARES if entries + entries // 8 <= min(1024, (1 << 30) // (4 * seq_pages)) else
                                    qh.KV8_TILES)


def test_workspaces_of_the_alignment_the_header_names(qh):
    """16 bytes, for the page calls and for attention: every other address is refused, none of those with it is for that."""
    import os
    import re
    from conftest import ROOT
    from test_kv8_refusals import P, attend
    text = open(os.path.join(ROOT, "include", "quanta_hip.h")).read()
    names = re.findall(r"/\* Workspace bytes of (?:a )?(qh_kv8_\w+)[^*]*?\((\d+)-byte aligned", text.replace("\n *", ""))
    assert names == [("qh_kv8_resize", "16"), ("qh_kv8_attention", "16")]
    c = cache(qh, seq_pages=128)
    L, r, need = qh.lib(), C.byref(c), qh.lib().qh_kv8_pages_workspace_bytes(C.byref(c))
    for off in (4, 8, 12):
        ws = C.c_void_p(4096 + off)
        assert L.qh_kv8_resize(r, P, P, 1, ws, need, None) == 4 and L.qh_kv8_fork(r, P, P, 1, 0, ws, need, None) == 4
        assert L.qh_kv8_compact(r, None, ws, need, None) == 4 and attend(qh, c, ws=ws) == 4
