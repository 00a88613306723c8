"""Beam search's selection (qh_beam_select) against its definition in 64 bits: sizes, ties, masks, rows without candidates,
logits that lie next to each other, and the reordering of the cache's sequences (qh_kv8_reorder) against a plain model.

Parents and tokens are equal. A score is the 64-bit one, whose exponentials are off by 2^-38 and whose sums by less, rounded to
f32 once: 2^-24 of it and 1e-11."""
import math

import numpy as np
import pytest
import torch

from kv8_util import PlainKV8

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16}


def plain_select(logits, scores, beams, k, n_valid):
    x = logits.float().cpu().numpy().astype(np.float64)[:, :n_valid]
    rows = x.shape[0]
    s = np.zeros(rows) if scores is None else scores.cpu().numpy().astype(np.float64)
    parent, token = np.full((rows // beams, k), -1, np.int32), np.full((rows // beams, k), -1, np.int32)
    score = np.full((rows // beams, k), -np.inf)
    for p in range(rows // beams):
        flat, val = [], []
        for b in range(p * beams, (p + 1) * beams):
            r = x[b]
            if np.isnan(r).any() or (r == np.inf).any() or not (r > -np.inf).any() or not np.isfinite(s[b]):
                continue
            m = r.max()
            e = np.exp(r - m)
            there = np.flatnonzero(r > -np.inf)
            flat.append(b * n_valid + there)
            val.append((r[there] - m) + (s[b] - math.log(math.fsum(e))))
        if not flat:
            continue
        flat, val = np.concatenate(flat), np.concatenate(val)
        best = np.lexsort((flat, -val))[:k]
        n = len(best)
        parent[p, :n], token[p, :n], score[p, :n] = flat[best] // n_valid, flat[best] % n_valid, val[best]
    return parent, token, score


def check(qh, logits, scores, beams, k, n_valid=None):
    parent, token, score = qh.beam_select(logits, scores, beams, k, n_valid)
    want = plain_select(logits, scores, beams, k, logits.shape[1] if n_valid is None else n_valid)
    assert np.array_equal(parent.cpu().numpy(), want[0])
    assert np.array_equal(token.cpu().numpy(), want[1])
    # past f32's largest value plus half its step (2^128 - 2^103), rounding to f32 gives infinity
    got, ref = score.cpu().numpy().astype(np.float64), np.where(want[2] <= -(2.0 ** 128 - 2.0 ** 103), -np.inf, want[2])
    there = np.isfinite(ref)
    assert np.array_equal(got[~there], ref[~there])
    assert (np.abs(got[there] - ref[there]) <= 2.0 ** -24 * np.abs(ref[there]) + 1e-11).all()
    return parent, token, score


def make(gpu, rows, vocab, dtype, seed=0, spread=2.0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    logits = (spread * torch.randn(rows, vocab, generator=gen, device=gpu)).to(TYPES[dtype])
    return logits, -20 * torch.rand(rows, generator=gen, device=gpu)


SHAPES = [(1, 1, 1, 1), (1, 1, 1, 5), (3, 2, 1, 4), (1, 4, 3, 8), (2, 1, 255, 1), (2, 3, 256, 7), (2, 3, 257, 7), (1, 2, 511, 40),
          (1, 2, 513, 40), (5, 4, 1000, 8), (1, 1, 1000, 256), (3, 2, 4096, 256), (2, 8, 5003, 16), (1, 5, 32000, 10),
          (2, 4, 50257, 8), (1, 4, 151936, 8), (3, 8, 151936, 16), (1, 32, 50257, 64), (64, 4, 300, 8), (1, 40, 200000, 80),
          (2, 12, 100, 24), (300, 1, 77, 3), (2, 8, 50257, 40), (1, 1, 262144, 8)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("prompts,beams,vocab,k", SHAPES)
def test_select(qh, gpu, dtype, prompts, beams, vocab, k):
    logits, scores = make(gpu, prompts * beams, vocab, dtype, seed=vocab + k)
    check(qh, logits, scores, beams, k)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_select_most_beams(qh, gpu, dtype):
    """256 beams over a large vocabulary: the largest groups, and the picking kernel with the most keys to a thread."""
    logits, scores = make(gpu, 256, 140001, dtype)
    check(qh, logits, scores, 256, 256)


def test_select_largest_vocabulary(qh, gpu):
    logits, scores = make(gpu, 6, 262144, "f32")
    check(qh, logits, scores, 3, 12)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [7, 300, 5000, 151936])
@pytest.mark.parametrize("k", [1, 8, 256])
def test_select_equal_logits(qh, gpu, dtype, vocab, k):
    """Every logit the same: the lowest ids of the first beam; with two beams equal and one above them, that one first."""
    logits = torch.full((6, vocab), 3.25, dtype=TYPES[dtype], device=gpu)
    check(qh, logits, None, 3, k)
    check(qh, logits, torch.tensor([-1.0, -1.0, -0.5, -2.0, -2.0, -2.0], device=gpu), 3, k)


@pytest.mark.parametrize("k", [1, 10, 256])
def test_select_few_values(qh, gpu, k):
    """Logits of a handful of values, so that thousands of candidates share the one at the border."""
    gen = torch.Generator(device=gpu).manual_seed(k)
    logits = torch.randint(0, 5, (8, 30011), generator=gen, device=gpu).float()
    check(qh, logits, -torch.arange(8, device=gpu, dtype=torch.float32) / 3, 4, k)
    check(qh, logits, None, 8, k)


@pytest.mark.parametrize("vocab", [3000, 151936])
@pytest.mark.parametrize("k", [8, 256])
def test_select_neighbouring_logits(qh, gpu, vocab, k):
    """Sorted logits: the best ones lie in one group, or at the end of one."""
    up = torch.linspace(-8, 8, vocab, device=gpu)
    logits = torch.stack([up, up.flip(0), up * 0.5, up.flip(0) * 0.9])
    check(qh, logits, torch.tensor([-1.0, -2.0, -1.5, -1.1], device=gpu), 4, k)
    check(qh, logits, torch.tensor([-1.0, -2.0, -1.5, -1.1], device=gpu), 2, k)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("beams,k", [(8, 2), (8, 16), (40, 1), (40, 8), (40, 32), (40, 33)])
def test_select_groups_far_apart(qh, gpu, dtype, beams, k):
    """The best candidates in every 64th group of 1,024 ids, and every other row without any of them."""
    logits, scores = make(gpu, beams, 151936, dtype, seed=k)
    groups = torch.arange(beams, device=gpu)[:, None] * 149 + torch.arange(151936, device=gpu)[None] // 1024
    best = (groups % 64 == 0) & (torch.arange(151936, device=gpu) % 1024 == 7)
    check(qh, torch.where(best, logits + 30, logits), None, beams, k)
    rows = torch.arange(beams, device=gpu)[:, None] % 2 == 0
    check(qh, torch.where(best & rows, logits + 30, logits), scores, beams, k)


def test_select_close_scores(qh, gpu):
    """Beams whose candidates interleave at distances far below f32's: 64-bit scores tell them apart."""
    logits = torch.zeros(4, 2000, device=gpu)
    logits[:, :50] = 10 + torch.arange(50, device=gpu) * 1e-6
    logits[1, 100] = 1e-4  # moves the row's sum by 2^-40 or so of it
    logits[2, 200] = 2e-3
    check(qh, logits, torch.full((4,), -31.0, device=gpu), 4, 120)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_select_masks(qh, gpu, dtype):
    """Forbidden ids as -infinity and as the type's lowest value; whole rows of both; fewer candidates than k."""
    low = torch.finfo(TYPES[dtype]).min
    logits, scores = make(gpu, 12, 3001, dtype)
    logits[0, 5:] = -math.inf          # five candidates
    logits[1] = -math.inf              # none
    logits[2] = low                    # all, and all alike
    logits[3, ::2] = low
    logits[4, 100:] = -math.inf
    logits[5, :3000] = -math.inf       # the last id alone
    logits[6:9] = -math.inf            # a prompt without candidates
    logits[9, 1:] = -math.inf
    logits[10] = -math.inf
    logits[11, :] = -math.inf
    logits[11, 7] = low                # a single candidate of the lowest value: its probability is 1
    for k in (1, 4, 256):
        check(qh, logits, scores, 3, k)


def test_select_rows_without_candidates(qh, gpu):
    logits, scores = make(gpu, 8, 4000, "f32")
    logits[0, 3999] = math.nan
    logits[1, 17] = math.inf
    logits[2, 0], logits[2, 1] = math.inf, math.nan
    scores[3] = -math.inf
    scores[4] = math.nan
    scores[5] = math.inf
    for beams in (1, 2, 4, 8):
        check(qh, logits, scores, beams, 8)


def test_select_large_values(qh, gpu):
    """Logits to f32's ends: differences count, not sizes."""
    logits = torch.zeros(6, 1000, device=gpu)
    logits[0] = 1e30
    logits[1, :3] = 3.4e38
    logits[1, 3:] = -3.4e38
    logits[2] = -3.4028234e38
    logits[3] = 2.0 ** 23 + torch.arange(1000, device=gpu) % 7
    logits[4, 5] = 800.0
    logits[5] = torch.arange(1000, device=gpu) * -1e4
    check(qh, logits, None, 1, 12)
    check(qh, logits, None, 6, 20)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("off,ld", [(0, 1000), (1, 1001), (3, 1007), (5, 1024)])
def test_select_strides_and_ids_behind(qh, gpu, dtype, off, ld):
    """Rows that begin anywhere, and NaN and large values behind n_valid and between the rows, which do not count."""
    buf = torch.full((off + 6 * ld + 64,), math.nan, dtype=TYPES[dtype], device=gpu)
    rows = buf[off:off + 6 * ld].view(6, ld)
    logits, scores = make(gpu, 6, 900, dtype)
    rows[:, :900] = logits
    rows[:, 900:950] = 60000.0
    view = rows[:, :1000]
    got = check(qh, view, scores, 3, 9, n_valid=900)
    for a, b in zip(got, qh.beam_select(logits.contiguous(), scores, 3, 9)):
        assert torch.equal(a, b)


def test_select_far_rows(qh, gpu):
    """Rows past 4 GiB of the first one."""
    ld = (1 << 30) + 4
    buf = torch.empty(2 * ld, device=gpu)
    view = buf.view(2, ld)[:, :5000]
    logits, scores = make(gpu, 2, 5000, "f32")
    view.copy_(logits)
    for a, b in zip(qh.beam_select(view, scores, 2, 8), qh.beam_select(logits, scores, 2, 8)):
        assert torch.equal(a, b)


def test_select_captured_and_on_another_stream(qh, gpu):
    logits, scores = make(gpu, 8, 50000, "f32")
    eager = lambda: qh.beam_select(logits, scores, 4, 8)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = eager()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, eager()))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = eager()
        graphs.append((g, out))
    for i in range(4):
        logits.copy_(torch.randn_like(logits) * 3)
        scores.sub_(0.25 * i)
        want = eager()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_select_refuses(qh, gpu):
    logits, scores = make(gpu, 6, 100, "f32")
    for call in (lambda: qh.beam_select(logits.double(), scores, 3, 4), lambda: qh.beam_select(logits, scores[:5], 3, 4),
                 lambda: qh.beam_select(logits, scores, 4, 4), lambda: qh.beam_select(logits, scores, 3, 0),
                 lambda: qh.beam_select(logits, scores, 3, 257), lambda: qh.beam_select(logits, scores, 3, 4, n_valid=101),
                 lambda: qh.beam_select(logits.t(), None, 2, 4), lambda: qh.beam_select(logits, scores.double(), 3, 4),
                 lambda: qh.beam_select(logits, scores.cpu(), 3, 4), lambda: qh.beam_select(logits.cpu(), scores.cpu(), 3, 4),
                 lambda: qh.beam_select(logits, scores, 0, 4)):
        with pytest.raises(qh.QHError):
            call()


# ------------------------------------------------------------------------------------------------- reordered sequences

def plain_reorder(m, src, dst):
    n = len(m.lens)
    if len(set(dst)) < len(dst) or any(not 0 <= d < n for d in dst) or any(not -1 <= s < n for s in src):
        m.status |= 2
        return
    rows = [(list(m.table[s, :m.need(m.lens[s])]), int(m.lens[s])) if s >= 0 else ([], 0) for s in src]
    for d in dst:
        m._drop(d, 0)
        m.lens[d] = 0
    for (row, length), d in zip(rows, dst):
        for j, page in enumerate(row):
            m.table[d, j] = page
            m.refs[page] += 1
        m.lens[d] = length


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def same_state(cache, m):
    assert np.array_equal(cache.lens.cpu().numpy(), m.lens)
    assert np.array_equal(cache.refs.cpu().numpy(), m.refs)
    assert np.array_equal(cache.table.cpu().numpy(), m.table)
    assert int(cache.status) == m.status
    held = np.zeros(m.n_pages, np.int64)
    for row in m.table:
        np.add.at(held, row[row >= 0], 1)
    assert np.array_equal(held, m.refs)


def both(qh, gpu, n_seqs, seq_pages, n_pages, page=16):
    return (qh.KV8Cache(1, n_pages, page, 1, 64, n_seqs, seq_pages, device=gpu),
            PlainKV8(1, n_pages, page, 1, 64, n_seqs, seq_pages))


@pytest.mark.parametrize("n_seqs,seq_pages,seed", [(1, 3, 0), (4, 5, 1), (4, 5, 2), (17, 9, 3), (64, 128, 4), (65, 128, 5),
                                                  (300, 40, 6), (1000, 9, 7), (2500, 3, 8), (8192, 1, 9), (9000, 1, 10), (3, 4000, 11)])
def test_reorder(qh, gpu, n_seqs, seq_pages, seed):
    """Random parents, some repeated, some -1, over rows of every length, then room for one more token: in one workgroup up to
    8,192 table entries and over the whole GPU above."""
    rng = np.random.default_rng(seed)
    cache, m = both(qh, gpu, n_seqs, seq_pages, 2 * n_seqs * seq_pages + 8)
    everyone = list(range(n_seqs))
    lens = rng.integers(0, 16 * seq_pages, n_seqs).tolist()
    cache.resize(ints(everyone, gpu), ints(lens, gpu))
    m.resize(everyone, lens)
    same_state(cache, m)
    for turn in range(4):
        if turn == 2:
            dst = rng.permutation(n_seqs)[:max(1, n_seqs // 2)].tolist()
            src = rng.integers(-1, n_seqs, len(dst)).tolist()
            cache.reorder(ints(src, gpu), ints(dst, gpu))
        else:
            dst, src = everyone, rng.integers(-1 if turn else 0, n_seqs, n_seqs).tolist()
            cache.reorder(ints(src, gpu))
        plain_reorder(m, src, dst)
        same_state(cache, m)
        grown = [min(int(l) + 1, 16 * seq_pages) for l in m.lens]
        cache.resize(ints(everyone, gpu), ints(grown, gpu))
        m.resize(everyone, grown)
        same_state(cache, m)


@pytest.mark.parametrize("n_seqs,seq_pages", [(6, 4), (100, 100)])
@pytest.mark.parametrize("what", ["twice", "dst", "src", "negative"])
def test_reorder_bad_lists_do_nothing(qh, gpu, n_seqs, seq_pages, what):
    cache, m = both(qh, gpu, n_seqs, seq_pages, n_seqs * seq_pages)
    lens = [7 * (i + 1) % (16 * seq_pages) for i in range(n_seqs)]
    everyone = list(range(n_seqs))
    cache.resize(ints(everyone, gpu), ints(lens, gpu))
    m.resize(everyone, lens)
    src, dst = everyone[::-1], list(everyone)
    if what == "twice":
        dst[3] = dst[1]
    elif what == "dst":
        dst[2] = n_seqs
    elif what == "src":
        src[2] = n_seqs
    else:
        src[0] = -2
    cache.reorder(ints(src, gpu), ints(dst, gpu))
    plain_reorder(m, src, dst)
    assert m.status == 2
    same_state(cache, m)


@pytest.mark.parametrize("n_seqs,seq_pages", [(6, 4), (100, 100)])
def test_reorder_swaps_and_rotates(qh, gpu, n_seqs, seq_pages):
    """Cycles through all sequences: no row is read after it was written; n turns of one place are where it began."""
    cache, m = both(qh, gpu, n_seqs, seq_pages, n_seqs * seq_pages)
    everyone = list(range(n_seqs))
    lens = [(5 + 11 * i) % (16 * seq_pages) for i in everyone]
    cache.resize(ints(everyone, gpu), ints(lens, gpu))
    before = cache.table.clone()
    turn = ints(everyone[1:] + [0], gpu)
    for _ in range(n_seqs):
        cache.reorder(turn)
    assert torch.equal(cache.table, before) and cache.lens.tolist() == lens and int(cache.status) == 0


def test_reorder_captured(qh, gpu):
    cache, m = both(qh, gpu, 8, 6, 96)
    everyone = list(range(8))
    lens = [10 * i for i in everyone]
    cache.resize(ints(everyone, gpu), ints(lens, gpu))
    m.resize(everyone, lens)
    src = ints(everyone, gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.reorder(src)
    rng = np.random.default_rng(0)
    for _ in range(5):
        new = rng.integers(-1, 8, 8).tolist()
        src.copy_(ints(new, gpu))
        g.replay()
        torch.cuda.synchronize()
        plain_reorder(m, new, everyone)
        same_state(cache, m)
        everyone2 = [0, 3]
        cache.resize(ints(everyone2, gpu), ints([33, 50], gpu))
        m.resize(everyone2, [33, 50])
        same_state(cache, m)


def test_reorder_refuses(qh, gpu):
    cache, _ = both(qh, gpu, 4, 3, 16)
    for call in (lambda: cache.reorder(torch.zeros(5, dtype=torch.int32, device=gpu)),
                 lambda: cache.reorder(torch.zeros(4, dtype=torch.int64, device=gpu)),
                 lambda: cache.reorder(torch.zeros(4, dtype=torch.int32)),
                 lambda: cache.reorder(ints([0, 1], gpu), ints([0], gpu))):
        with pytest.raises(qh.QHError):
            call()
