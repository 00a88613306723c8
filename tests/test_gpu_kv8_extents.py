"""8-bit cache attention at the largest lengths that a cache may have: counts of tiles past what an int holds.

The sequences have a length and, but for their first and last page, no pages: tokens without a page are left out, so the result
is that of a short sequence of the two pages."""
import pytest

from kv8_bound import exact_attention, filled, ints, randn, worst

pytestmark = pytest.mark.gpu


def holes(qh, kv, seq_pages):
    """A cache of two sequences: 0 as long as the table, with two pages, 1 of those two pages."""
    page = 256
    c = qh.KV8Cache(1, 2, page, kv, 64, 3, seq_pages)
    c.resize(ints([1]), ints([2 * page]))
    c.append(0, randn(1, 2 * page, kv, 64), randn(2, 2 * page, kv, 64), start=ints([0, 2 * page]), seqs=ints([1]))
    c.lens[0] = seq_pages * page
    c.table[0, 0], c.table[0, -1] = c.table[1, 0], c.table[1, 1]
    return c


def check(c, q, seqs):
    import torch
    got = c.attention(0, q, seqs=ints(seqs))
    torch.cuda.synchronize()
    rows = [i for i, s in enumerate(seqs) if s == 0]
    want, bound = exact_attention(c, 0, q[rows], [1] * len(rows), [1] * len(rows))
    ratio, at = worst(got[rows], want, bound)
    assert ratio <= 1, (ratio, at)
    rest = [i for i, s in enumerate(seqs) if s != 0]
    assert not got[rest].any()


def test_many_short_sequences_beside_a_long_one(qh, gpu):
    """Two shares to a KV head and 1,024 sequences: every item on shares of its own would be 2^32 tiles."""
    c = holes(qh, 256, 1 << 21)
    check(c, randn(3, 1024, 256, 64), [2] * 500 + [0] + [2] * 523)


def test_long_sequences_together(qh, gpu):
    """66 times 2^30 positions, 2^24 tiles each: in two launches."""
    c = holes(qh, 1, 1 << 22)
    check(c, randn(3, 66, 2, 64), [0] * 66)
