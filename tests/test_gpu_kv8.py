"""The 8-bit paged cache on the GPU against a plain 64-bit model (kv8_util): stored values bit for bit, page tables and
page contents exactly, attention within bounds derived from the number formats."""
import numpy as np
import pytest

from kv8_util import PlainKV8, attention_bound

pytestmark = pytest.mark.gpu

SEED = 11


@pytest.fixture(autouse=True)
def _gpu(gpu):
    return gpu


def ints(x):
    import torch
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def starts(counts):
    return ints(np.concatenate([[0], np.cumsum(counts)]))


class Pair:
    """The GPU cache and the plain model, driven alike."""

    def __init__(self, qh, layers, pages, page_tokens, kv, hd, seqs, seq_pages):
        import torch
        self.torch = torch
        self.gpu = qh.KV8Cache(layers, pages, page_tokens, kv, hd, seqs, seq_pages)
        self.gpu.pages.fill_(0x7f)  # stale contents: codes of 127 and NaN scales
        self.plain = PlainKV8(layers, pages, page_tokens, kv, hd, seqs, seq_pages)

    def resize(self, seqs, lens):
        self.gpu.resize(ints(seqs), ints(lens))
        self.plain.resize(list(seqs), list(lens))

    def fork(self, src, dst, copy=False):
        self.gpu.fork(ints(src), ints(dst), copy)
        self.plain.fork(list(src), list(dst), copy)

    def rows(self, rng, n, dtype, width=None):
        """k, v of n tokens as views of one wider row, and as float64 arrays."""
        p = self.plain
        x = rng.standard_normal((n, 2 * p.kv + 1, p.hd)).astype(np.float32) * np.float32(2.0) ** rng.integers(-3, 4, (n, 1, 1))
        t = self.torch.from_numpy(x.astype(np.float32)).to("cuda").to(getattr(self.torch, dtype))
        a = t.cpu().float().numpy()
        return t[:, :p.kv], t[:, p.kv:2 * p.kv], a[:, :p.kv], a[:, p.kv:2 * p.kv]

    def append(self, rng, layer, seqs, counts, dtype="float32", single=False, edit=None):
        n = sum(counts)
        k, v, ka, va = self.rows(rng, n, dtype)
        if edit:
            edit(k, v)
            ka, va = k.cpu().float().numpy(), v.cpu().float().numpy()
        self.gpu.append(layer, k, v, start=None if single else starts(counts), seqs=ints(seqs))
        self.plain.append(layer, list(seqs), list(counts), ka, va)

    def check_state(self):
        g, p = self.gpu, self.plain
        assert np.array_equal(g.lens.cpu().numpy(), p.lens)
        assert np.array_equal(g.refs.cpu().numpy(), p.refs)
        assert np.array_equal(g.table.cpu().numpy(), p.table)
        assert int(g.status.cpu()) == p.status

    def check_values(self, layer):
        p = self.plain
        live = [s for s in range(len(p.lens)) if p.lens[s] > 0]
        counts = [int(p.lens[s]) for s in live]
        k, v = (t.cpu().numpy() for t in self.gpu.read(layer, sum(counts), start=starts(counts), seqs=ints(live)))
        at = 0
        for s, m in zip(live, counts):
            for got, want, what in zip((k, v), p.values(layer, s), "kv"):
                bad = np.argwhere(~((got[at:at + m] == want) | (np.isnan(got[at:at + m]) & np.isnan(want))))
                assert bad.size == 0, (what, s, bad[:5], got[at:at + m][tuple(bad[0])], want[tuple(bad[0])])
            at += m


# ------------------------------------------------------------------------------------------------ append and read

@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("kv,hd,page", [(2, 64, 64), (1, 128, 16), (3, 128, 32), (8, 64, 256)])
def test_append_in_steps(qh, dtype, kv, hd, page):
    """Stretches that begin and end inside blocks and pages, with scales that grow and do not, read back bit for bit."""
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 2, 40, page, kv, hd, 5, -(-300 // page) + 1)
    lens = [0, 0, 0, 0, 0]
    for seqs, counts in (([0, 1, 2], [5, 16, 33]), ([3, 0], [1, 11]), ([2, 4, 1, 0], [100, 17, 1, 1]), ([4], [15]),
                         ([1, 3], [2, 47])):
        for s, m in zip(seqs, counts):
            lens[s] += m
        c.resize(seqs, [lens[s] for s in seqs])
        for layer in (1, 0):
            c.append(rng, layer, seqs, counts, dtype)
        c.check_state()
        c.check_values(0)
        c.check_values(1)
    assert c.plain.status == 0


def test_append_single_tokens(qh):
    rng = np.random.default_rng(SEED + 1)
    c = Pair(qh, 1, 30, 16, 2, 64, 6, 6)
    for step in range(1, 36):
        seqs = [5, 0, 3] if step % 2 else [0, 5, 3]
        c.resize(seqs, [step] * 3)
        c.append(rng, 0, seqs, [1, 1, 1], single=True)
    c.check_state()
    c.check_values(0)


@pytest.mark.parametrize("n_entries", [1, 63, 64, 65, 200])
def test_append_many_entries(qh, n_entries):
    """Entry lookup past 64 entries, some of them without rows."""
    rng = np.random.default_rng(SEED + n_entries)
    c = Pair(qh, 1, 900, 16, 1, 64, 210, 4)
    counts = [int(x) for x in rng.integers(0, 40, n_entries)]
    seqs = [int(x) for x in rng.permutation(210)[:n_entries]]
    c.resize(seqs, counts)
    c.append(rng, 0, seqs, counts)
    c.check_state()
    c.check_values(0)


def test_thousands_of_entries(qh):
    """Entry lookup past 64 x 64 entries, some without rows, by append, read and attention."""
    rng = np.random.default_rng(SEED)
    n = 4200
    counts = [int(x) for x in rng.choice([0, 1, 2, 17], n, p=[.3, .4, .29, .01])]
    c = Pair(qh, 1, n + 60, 16, 1, 64, n, 2)
    seqs = [int(x) for x in rng.permutation(n)]
    c.resize(seqs, counts)
    c.append(rng, 0, seqs, counts, "float32")
    check_attention(c, rng, seqs, counts, 2, "float32")
    c.check_values(0)
    # few entries with rows among many without
    check_attention(c, rng, seqs, [0] * (n - 3) + [100, 0, 40], 2, "float32", causal=False)


def test_append_extreme_values(qh):
    """Zeros, the largest and the smallest numbers, halves between codes, infinities and NaN: the block of the head reads
    as NaN, the others are untouched by it."""
    import torch
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 1, 8, 32, 2, 64, 2, 4)
    c.resize([0], [100])

    def edit(k, v):
        k[0:16] = 0                      # a block of zeros
        k[16:32, 0] *= 1e38 / 60         # near the end of the range
        v[0:16, 0] *= 1e-38              # subnormal scales
        v[16:32, 1] *= 1e-42             # scales that round to 0 or a few bits
        k[32:48, 1] = torch.arange(64, device="cuda") - 31.5  # halves
        k[32, 1, 0] = 127.0
        k[50, 0, 3] = float("inf")
        v[70, 1, 5] = float("nan")
        k[85, 1, 1] = -float("inf")
    c.append(rng, 0, [0], [100], edit=edit)
    c.check_values(0)
    k, v = c.gpu.read(0, 100, start=starts([100]))
    assert torch.isnan(k[48:64, 0]).all() and not torch.isnan(k[48:64, 1]).any() and not torch.isnan(v[48:64]).any()
    assert torch.isnan(v[64:80, 1]).all() and torch.isnan(k[80:96, 1]).all() and not torch.isnan(k[96:]).any()
    c.resize([0], [102])  # a poisoned block's successor begins anew
    c.append(rng, 0, [0], [2])
    c.check_values(0)


def test_append_leaves_other_pages_and_rows_alone(qh):
    """Shared pages, entries without a sequence, rows behind the last entry: nothing else is written."""
    import torch
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 1, 12, 16, 2, 64, 4, 5)
    c.resize([0, 1], [20, 7])
    c.append(rng, 0, [0, 1], [20, 7])
    c.fork([0], [2])
    before = c.gpu.pages.clone()
    c.append(rng, 0, [2, -1, 9], [3, 2, 4])  # tokens 17 .. 19 lie in a page that 0 and 2 share
    assert torch.equal(before, c.gpu.pages) and c.plain.status == 4
    c.check_state()
    c.resize([2], [22])
    c.append(rng, 0, [2], [2])
    c.check_state()
    c.check_values(0)
    # rows that no entry owns are neither read nor written
    out = torch.full((2, 9, 2, 64), 5.0, device="cuda")
    r = qh.lib()
    import ctypes as C
    assert r.qh_kv8_read(C.byref(c.gpu.view), 0, out[0].data_ptr(), out[1].data_ptr(), 0, 128, 128,
                         starts([3, 2]).data_ptr(), ints([1, -1]).data_ptr(), 2, 9, None) == 0
    torch.cuda.synchronize()
    assert (out[:, 3:] == 5).all() and not (out[:, :3] == 5).any()
    # a longer entry than its sequence: rows before the first position have no place
    c.append(rng, 0, [1], [9])
    c.check_values(0)


def test_append_into_a_missing_page(qh):
    import torch
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 1, 6, 16, 1, 64, 1, 4)
    c.resize([0], [40])
    c.gpu.table[0, 1] = -1
    c.plain.table[0, 1] = -1
    before = c.gpu.pages[0, c.plain.n_pages - 1].clone()
    c.append(rng, 0, [0], [40])
    c.check_values(0)
    c.gpu.table[0, 1] = 1 << 20  # and one past the pool
    c.append(rng, 0, [0], [40])
    c.gpu.attention(0, torch.ones(40, 2, 64, device="cuda"), start=starts([40]))
    torch.cuda.synchronize()
    assert torch.equal(before, c.gpu.pages[0, c.plain.n_pages - 1])


# ------------------------------------------------------------------------------------------------ attention

def filled(qh, rng, lens, kv, hd, page, dtype, room=0):
    """A cache with sequences of these lengths and room for `room` more tokens in each."""
    need = [-(-(n + room) // page) for n in lens]
    c = Pair(qh, 1, sum(need) + 2, page, kv, hd, len(lens), max(1, max(need)))
    # pages in a mixed order: sequences grow in turns
    at = [0] * len(lens)
    while at != list(lens):
        grow = [s for s in range(len(lens)) if at[s] < lens[s]]
        new = [min(lens[s], at[s] + page + 3) for s in grow]
        c.resize(grow, new)
        c.append(rng, 0, grow, [b - at[s] for s, b in zip(grow, new)], dtype)
        for s, b in zip(grow, new):
            at[s] = b
    return c


def check_attention(c, rng, seqs, counts, heads, dtype, causal=True, scale=None, single=False, extra_rows=0, q_scale=1.0):
    import torch
    hd, n = c.plain.hd, sum(counts)
    wide = torch.from_numpy(rng.standard_normal((n + extra_rows, heads + 1, hd)).astype(np.float32) * q_scale)
    wide = wide.to("cuda").to(getattr(torch, dtype))
    q = wide[:, :heads]  # rows further apart than they are wide
    room = torch.full((n + extra_rows, heads + 2, hd), 3.0, dtype=q.dtype, device="cuda")
    out = room[:, :heads]
    got = c.gpu.attention(0, q, start=None if single else starts(counts), seqs=ints(seqs), causal=causal, scale=scale,
                          out=out)
    assert got is out
    got = out.cpu().double().numpy()
    assert (room[:, heads:] == 3).all() and (got[n:] == 3).all()
    used = hd ** -0.5 if scale is None else scale
    want, *sizes = c.plain.attention(0, seqs, counts, q.cpu().float().numpy(), causal, used)
    most = max([int(c.plain.lens[s]) for s in seqs if 0 <= s < len(c.plain.lens)] + [0])
    bound = attention_bound("f32" if dtype == "float32" else "f16", want, *sizes, most, hd)
    off = np.abs(got[:n] - want[:n]) - bound[:n]
    assert np.isfinite(got[:n]).all()
    assert (off <= 0).all(), (np.argwhere(off > 0)[:5], off.max(), np.abs(got[:n] - want[:n]).max())


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 257, 500]


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("heads,kv,hd,page", [(14, 2, 64, 64), (6, 2, 128, 16), (1, 1, 64, 256), (8, 8, 128, 32),
                                              (40, 2, 64, 16), (17, 1, 128, 64)])
def test_single_tokens(qh, dtype, heads, kv, hd, page):
    """One token for each of sequences of many lengths, an empty one and two without a sequence among them."""
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, LENGTHS + [0], kv, hd, page, dtype)
    seqs = [int(s) for s in rng.permutation(len(LENGTHS) + 1)] + [-1, 99]
    check_attention(c, rng, seqs, [1] * len(seqs), heads, dtype, single=True)
    check_attention(c, rng, seqs, [1] * len(seqs), heads, dtype, extra_rows=3)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("n,page", [(1, 64), (4000, 16), (9001, 256)])
def test_one_long_sequence(qh, dtype, n, page):
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [n], 2, 64, page, dtype)
    check_attention(c, rng, [0], [1], 14, dtype, single=True)
    check_attention(c, rng, [0], [min(n, 3)], 14, dtype)


def test_scores_far_apart(qh):
    """Queries so large that one position takes all the weight, and so small that all share it."""
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [700, 90], 2, 128, 32, "float32")
    for s in (1e-30, 1e-3, 60.0):
        check_attention(c, rng, [0, 1], [1, 1], 4, "float32", single=True, q_scale=s)
        check_attention(c, rng, [0, 1], [40, 90], 4, "float32", q_scale=s)
    check_attention(c, rng, [0, 1], [1, 1], 4, "float32", single=True, scale=0.0)
    check_attention(c, rng, [0, 1], [1, 1], 4, "float32", single=True, scale=-0.3)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_and_values_that_grow(qh, dtype, hd):
    """Keys and values that grow along the sequence: the largest score and the values' unit move again and again."""
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 1, 60, 16, 2, hd, 2, 48)
    c.resize([0, 1], [700, 90])

    def grow(k, v):
        import torch
        at = torch.cat([torch.arange(700), torch.arange(90)]).to("cuda").view(-1, 1, 1)
        k.mul_((at / 40 + 0.05).to(k.dtype))
        v.mul_(torch.exp2(at / 100 - 6).to(v.dtype))

    c.append(rng, 0, [0, 1], [700, 90], dtype, edit=grow)
    for q_scale in (0.1, 2.0):
        check_attention(c, rng, [0, 1], [90, 90], 6, dtype, q_scale=q_scale)
        check_attention(c, rng, [0, 1], [1, 1], 6, dtype, q_scale=q_scale)
        check_attention(c, rng, [0, 1], [300, 5], 6, dtype, q_scale=q_scale, causal=False)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("heads,kv,hd,page", [(14, 2, 64, 64), (4, 2, 128, 16), (5, 5, 64, 32), (33, 1, 128, 128)])
def test_ragged_prompts(qh, dtype, heads, kv, hd, page):
    """Entries of one row to hundreds, at the front of their sequences and far behind it, and one without rows."""
    rng = np.random.default_rng(SEED)
    lens = [300, 1, 64, 129, 400, 16, 70]
    c = filled(qh, rng, lens, kv, hd, page, dtype)
    check_attention(c, rng, [0, 1, 2, 3, 4, 5, 6], [300, 1, 30, 129, 65, 0, 70], heads, dtype, extra_rows=2)
    check_attention(c, rng, [4, 0], [33, 5], heads, dtype)
    check_attention(c, rng, [4, 4, 0], [4, 2, 1], heads, dtype)  # one sequence read twice


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_whole_sequences(qh, dtype):
    """Without the causal limit: rows of another length than the sequence, an empty sequence among them."""
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [130, 17, 0, 900], 2, 64, 32, dtype)
    check_attention(c, rng, [0, 1, 2, 3], [1, 1, 1, 1], 6, dtype, causal=False, single=True)
    check_attention(c, rng, [0, 1, 2, 3], [10, 200, 3, 77], 6, dtype, causal=False)
    # causal rows before the first position see nothing
    check_attention(c, rng, [1, 2], [60, 5], 6, dtype)


def test_rows_that_see_no_poison_are_clean(qh):
    """NaN blocks (from an infinite value) behind what a row sees leave it finite and right; rows that see one are NaN."""
    import torch
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [100], 1, 64, 16, "float32", room=60)
    c.resize([0], [160])

    def edit(k, v):
        v[20, 0, 3] = float("inf")  # position 120: block 112 .. 127
        k[40, 0, 1] = float("nan")  # position 140: block 128 .. 143
    c.append(rng, 0, [0], [60], edit=edit)
    c.check_state()
    q = torch.from_numpy(rng.standard_normal((160, 4, 64)).astype(np.float32)).to("cuda")
    out = c.gpu.attention(0, q, start=starts([160]))
    clean = torch.isfinite(out).all(-1).all(-1).cpu().numpy()
    assert clean[:112].all() and torch.isnan(out[112:]).all()
    few = c.gpu.attention(0, q[:2], start=starts([2]))
    assert torch.isnan(few).all()
    want, *sizes = c.plain.attention(0, [0], [160], q.cpu().numpy(), True, 0.125)
    got = out.cpu().double().numpy()[:112]
    assert (np.abs(got - want[:112]) <= attention_bound("f32", want, *sizes, 160, 64)[:112]).all()


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_a_query_that_is_not_finite_is_its_own_row(qh, dtype):
    import torch
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [160], 2, 128, 16, dtype)
    q = torch.from_numpy(rng.standard_normal((160, 4, 128)).astype(np.float32)).to("cuda").to(getattr(torch, dtype))
    for rows in (160, 3):  # both kernels
        x = q[-rows:].clone()
        want = c.gpu.attention(0, x, start=starts([rows]))
        x[0, 1, 0], x[1, 2, 100], x[2, 3, 7] = float("nan"), float("inf"), -float("inf")
        got = c.gpu.attention(0, x, start=starts([rows]))
        bad = torch.zeros(rows, 4, dtype=torch.bool, device="cuda")
        bad[0, 1] = bad[1, 2] = bad[2, 3] = True
        assert torch.isnan(got[bad]).all() and torch.isfinite(want).all()
        assert torch.equal(got[~bad], want[~bad])


def test_split_prompts_join(qh):
    """A few rows behind a long cache: the positions are split over workgroups and joined."""
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [3000], 1, 64, 64, "float16")
    for m in (1, 9, 40, 130):
        check_attention(c, rng, [0], [m], 8, "float16")


@pytest.mark.parametrize("dtype,kv,hd", [("float32", 2, 64), ("float16", 1, 128)])
def test_prompts_on_part_of_the_gpu(qh, dtype, kv, hd):
    """Few row tiles: halves of a workgroup share the positions, an odd and an even number of tiles, one and none."""
    rng = np.random.default_rng(SEED)
    lens = [470, 64, 65, 120, 300, 0, 129]
    c = filled(qh, rng, lens, kv, hd, 16, dtype)
    for counts in ([470, 64, 65, 120, 300, 0, 129], [40, 64, 1, 33, 200, 0, 100], [0, 0, 0, 0, 0, 40, 0]):
        for causal in (True, False):
            check_attention(c, rng, list(range(7)), counts, 6 * kv, dtype, causal=causal)


def test_pools_and_rows_past_32_bit_offsets(qh):
    """Pages behind more than 4 GiB of pool, rows more than 2^32 bytes apart: as in a small pool."""
    import torch
    rng = np.random.default_rng(SEED)
    small = filled(qh, rng, [700, 300], 8, 128, 256, "float16").gpu
    big = qh.KV8Cache(1, 12000, 256, 8, 128, 2, 3)  # 6.3 GB
    big.refs[:11990] = 1  # in use by somebody: the sequences get the last pages
    big.resize(ints([0, 1]), ints([700, 300]))
    assert big.table[big.table >= 0].min() >= 11990
    kv = small.read(0, 1000, start=starts([700, 300]), dtype=torch.float16)
    big.append(0, kv[0], kv[1], start=starts([700, 300]))
    small.resize(ints([0, 1]), ints([0, 0]))
    small.resize(ints([0, 1]), ints([700, 300]))
    small.append(0, kv[0], kv[1], start=starts([700, 300]))  # the values rounded twice, in both alike
    for a, b in zip(*(c.read(0, 1000, start=starts([700, 300])) for c in (small, big))):
        assert torch.equal(a, b)
    q = torch.from_numpy(rng.standard_normal((9, 32, 128)).astype(np.float32)).to("cuda").half()
    far = torch.empty((9, 1 << 28), dtype=torch.float16, device="cuda")
    far[:, :32 * 128] = q.view(9, -1)
    for counts in ([4, 5], [1, 8]):
        want = small.attention(0, q, start=starts(counts)).view(9, -1)
        assert torch.equal(want, big.attention(0, far[:, :32 * 128], start=starts(counts), out=far[:, 4096 * 2:4096 * 3]))
    assert torch.equal(small.attention(0, q[7:]).view(2, -1), big.attention(0, far[7:, :4096]).view(2, -1))
    far[:, :1024], far[:, 1024:2048] = kv[0][:9].view(9, -1), kv[1][:9].view(9, -1)
    for c in (small, big):
        c.resize(ints([1]), ints([0]))
        c.resize(ints([1]), ints([9]))
    small.append(0, kv[0][:9], kv[1][:9], start=starts([9]), seqs=ints([1]))
    big.append(0, far[:, :1024], far[:, 1024:2048], start=starts([9]), seqs=ints([1]))
    for a, b in zip(*(c.read(0, 9, start=starts([9]), seqs=ints([1])) for c in (small, big))):
        assert torch.equal(a, b)


def test_many_sequences(qh):
    """More entries than one launch of the few-row kernel takes."""
    rng = np.random.default_rng(SEED)
    lens = [int(x) for x in rng.integers(0, 20, 1100)]
    c = filled(qh, rng, lens, 1, 64, 16, "float32")
    check_attention(c, rng, list(range(1100)), [1] * 1100, 2, "float32", single=True)
    check_attention(c, rng, list(range(1000)), [1] * 1000, 2, "float32", single=True)
    check_attention(c, rng, list(range(1000)), [1] * 1000, 2, "float32")


@pytest.mark.parametrize("longest", [1100, 2100])
def test_many_sequences_of_unlike_lengths(qh, longest):
    """The same for long sequences, whole and in shares that are joined, with two row tiles to an entry, in and out of
    order."""
    import torch
    rng = np.random.default_rng(SEED)
    lens = [int(x) for x in rng.integers(0, 20, 530)]
    lens[3], lens[511], lens[512], lens[529] = longest, 700, 1030, 65
    c = filled(qh, rng, lens, 1, 64, 16, "float32")
    check_attention(c, rng, [int(x) for x in rng.permutation(530)], [1] * 530, 17, "float32", single=True)
    q = torch.from_numpy(rng.standard_normal((530, 17, 64)).astype(np.float32)).to("cuda")
    assert torch.equal(c.gpu.attention(0, q), c.gpu.attention(0, q, seqs=ints(range(530))))


# ------------------------------------------------------------------------------------------------ pages

def test_pages_follow_the_plain_model(qh):
    """Random growth, release, forks (shared and copied), compaction, refused calls: tables, counts and values."""
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 2, 48, 32, 1, 64, 9, 8)
    for step in range(60):
        what = rng.integers(0, 6)
        if what <= 2:
            k = int(rng.integers(1, 6))
            seqs = [int(s) for s in rng.permutation(9)[:k]]
            lens = [int(x) for x in rng.choice([0, 1, 31, 32, 33, 64, 100, 170, 256], k)]
            before = c.plain.lens.copy()
            c.resize(seqs, lens)
            grown = [(s, int(c.plain.lens[s] - before[s])) for s in seqs if c.plain.lens[s] > before[s]]
            if grown:
                for layer in (0, 1):
                    c.append(rng, layer, [s for s, _ in grown], [m for _, m in grown])
        elif what <= 4:
            order = [int(s) for s in rng.permutation(9)]
            src = [order[0], order[1], order[0]][:int(rng.integers(1, 4))]
            c.fork(src, order[2:2 + len(src)], copy=bool(rng.integers(0, 2)))
        else:
            live = c.gpu.compact()
            assert int(live.cpu()) == c.plain.compact()
        c.check_state()
        if step % 6 == 5:
            c.check_values(0)
            c.check_values(1)
    assert c.plain.status in (0, 1) and len(c.plain.copied) > 10
    c.gpu.reset()
    assert int(c.gpu.refs.sum()) == 0 and int(c.gpu.lens.sum()) == 0 and int(c.gpu.status) == 0
    assert (c.gpu.table == -1).all()


def test_bad_lists_change_nothing(qh):
    c = Pair(qh, 1, 20, 16, 1, 64, 4, 6)
    c.resize([0, 1], [40, 10])
    for seqs, lens in (([0, 0], [1, 2]), ([4], [1]), ([-1], [1]), ([1], [97]), ([1], [-1]), ([2, 0, 3, 2], [1, 1, 1, 1])):
        c.resize(seqs, lens)
        c.check_state()
        assert c.plain.status == 2
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [4]), ([-3], [2])):
        for copy in (False, True):
            c.fork(src, dst, copy)
            c.check_state()


def test_too_few_pages(qh):
    c = Pair(qh, 1, 5, 16, 1, 64, 4, 6)
    c.resize([0, 1], [33, 16])
    c.resize([1, 2, 3], [0, 40, 16])  # 1's page comes back, four are wanted, two are free: neither grows
    c.check_state()
    assert c.plain.status == 1 and c.plain.lens.tolist() == [33, 0, 0, 0]
    c.resize([2], [32])
    c.check_state()
    c.fork([0], [2], copy=True)  # 2 gives its pages back first: two of three
    c.check_state()
    assert c.plain.lens.tolist() == [33, 0, 0, 0]


@pytest.mark.parametrize("n_pages", [1, 1023, 1025, 5000, 9000])
def test_large_pools(qh, n_pages):
    """Free lists and compaction over pools of more than one round of the planning workgroup, page bytes included."""
    import torch
    rng = np.random.default_rng(n_pages)
    n_seqs = min(n_pages, 1500)
    c = Pair(qh, 2, n_pages, 16, 1, 64, n_seqs, 12)
    c.gpu.pages.copy_(torch.from_numpy(rng.integers(0, 256, tuple(c.gpu.pages.shape), np.uint8)))
    lens = rng.integers(0, 16 * 12 + 1, n_seqs)
    while sum(-(-lens // 16)) > n_pages:
        lens = lens // 2
    c.resize(range(n_seqs), lens.tolist())
    c.check_state()
    gone = [int(s) for s in rng.permutation(n_seqs)[:n_seqs // 2]]
    c.resize(gone, [0] * len(gone))
    pages = c.gpu.pages.cpu().numpy()
    assert int(c.gpu.compact().cpu()) == c.plain.compact()
    c.check_state()
    for a, b in c.plain.copied:
        pages[:, b] = pages[:, a]
    assert np.array_equal(pages, c.gpu.pages.cpu().numpy())


def test_growth_of_many_pages_at_once(qh):
    c = Pair(qh, 1, 9000, 16, 1, 64, 5, 8000)
    c.resize([3, 0, 4], [16 * 4000 + 1, 5, 16 * 3000])
    c.check_state()
    c.fork([3], [1], copy=False)
    c.check_state()
    c.resize([1, 3], [16 * 4000 + 2, 16 * 4000 + 3])  # the shared last page: both take copies
    c.check_state()


# ------------------------------------------------------------------------------------------------ together

def step_of(c, k, v, q, layers, seqs, lens):
    c.resize(seqs, lens)
    return [c.append(l, k[l], v[l], seqs=seqs) or c.attention(l, q[l], seqs=seqs) for l in range(layers)]


def test_a_served_batch(qh):
    """A prompt, replies forked from it, steps of all of them, one ending, compaction, more steps: against the plain
    model at every step."""
    rng = np.random.default_rng(SEED)
    c = Pair(qh, 2, 64, 16, 2, 64, 6, 12)
    c.resize([0], [75])
    for layer in (0, 1):
        c.append(rng, layer, [0], [75], "float16")
    check_attention(c, rng, [0], [75], 4, "float16")
    c.fork([0, 0, 0], [1, 2, 3])
    c.fork([0], [4], copy=True)
    live = [0, 1, 2, 3, 4]
    for step in range(8):
        if step == 4:
            c.resize([2], [0])
            live.remove(2)
            assert int(c.gpu.compact().cpu()) == c.plain.compact()
        c.resize(live, [int(c.plain.lens[s]) + 1 for s in live])
        for layer in (0, 1):
            c.append(rng, layer, live, [1] * len(live), "float16", single=True)
        c.check_state()
        check_attention(c, rng, live, [1] * len(live), 4, "float16", single=True)
    c.check_values(0)
    c.check_values(1)
    assert c.plain.status == 0


def test_captured_steps(qh):
    """A decode step captured once and replayed with new inputs and lengths equals eager steps, replay for replay; a second
    captured graph on the same cache keeps apart from it."""
    import torch
    rng = np.random.default_rng(SEED)
    dev = "cuda"

    def fresh():
        c = qh.KV8Cache(2, 40, 16, 2, 64, 4, 10)
        c.pages.zero_()
        return c

    seqs, k, v, q = ints([0, 1, 2]), [torch.zeros(3, 2, 64, device=dev) for _ in range(2)], \
        [torch.zeros(3, 2, 64, device=dev) for _ in range(2)], [torch.zeros(3, 8, 64, device=dev) for _ in range(2)]
    lens = ints([0, 0, 0])
    data = [[torch.from_numpy(rng.standard_normal((2, 3, h, 64)).astype(np.float32)).to(dev) for h in (2, 2, 8)]
            for _ in range(40)]

    def feed(i):
        for buf, x in zip((k, v, q), data[i]):
            for l in range(2):
                buf[l].copy_(x[l])
        lens.copy_(ints([i + 1, i // 2 + 1, 3 * (i + 1) if i < 20 else 60]))

    eager_c, want = fresh(), []
    for i in range(40):
        feed(i)
        want.append([o.clone() for o in step_of(eager_c, k, v, q, 2, seqs, lens)])
    c = fresh()
    stream = torch.cuda.Stream()
    feed(0)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step_of(c, k, v, q, 2, seqs, lens)  # a first step outside the graph
    torch.cuda.current_stream().wait_stream(stream)
    c.reset()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step_of(c, k, v, q, 2, seqs, lens)
    with torch.cuda.graph(g2):
        again = [c.attention(l, q[l], seqs=seqs) for l in range(2)]
    for i in range(40):
        feed(i)
        g.replay()
        g2.replay()
        for l in range(2):
            assert torch.equal(outs[l], want[i][l]), (i, l)
            assert torch.equal(again[l], want[i][l]), (i, l)
        torch.ones(1000, device=dev).sum().item()  # the program's own work between replays
    assert torch.equal(c.lens, eager_c.lens) and torch.equal(c.table, eager_c.table) and int(c.status) == 0


def test_two_streams_at_once(qh):
    """Attention of two batches on two streams over one cache, each with its own workspace."""
    import torch
    rng = np.random.default_rng(SEED)
    c = filled(qh, rng, [2000, 1500], 2, 64, 32, "float32")
    q = torch.from_numpy(rng.standard_normal((2, 14, 64)).astype(np.float32)).to("cuda")
    want = c.gpu.attention(0, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(c.gpu.attention(0, q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_python_refusals(qh):
    import torch
    with pytest.raises(qh.QHError):
        qh.KV8Cache(1, 4, 24, 2, 64, 1, 4)
    with pytest.raises(qh.QHError):
        qh.KV8Cache(1, 0, 16, 2, 64, 1, 4)
    c = qh.KV8Cache(1, 4, 16, 2, 64, 3, 4)
    k = torch.zeros(3, 2, 64, device="cuda")
    for bad in (lambda: c.append(0, k, k[:2]), lambda: c.append(0, k, k.half()), lambda: c.append(0, k.double(), k.double()),
                lambda: c.append(0, k.cpu(), k.cpu()), lambda: c.append(0, k.transpose(1, 2), k),
                lambda: c.append(0, k, k, seqs=ints([0, 1])), lambda: c.append(1, k, k),
                lambda: c.append(0, k, k, seqs=ints([0, 1, 2]).long()), lambda: c.append(0, k, k, start=ints([0, 3]).cpu()),
                lambda: c.append(0, torch.zeros(5, 2, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda")),
                lambda: c.attention(0, torch.zeros(3, 5, 64, device="cuda")),
                lambda: c.attention(0, k, out=torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)),
                lambda: c.attention(0, torch.zeros(3, 2, 65, device="cuda")[:, :, 1:]),
                lambda: c.attention(0, k, scale=float("nan")), lambda: c.resize(ints([0, 1]), ints([1])),
                lambda: c.fork(ints([0]), ints([1, 2])), lambda: c.resize(ints([0, 1, 2, 0]), ints([1, 1, 1, 1]))):
        with pytest.raises(qh.QHError):
            bad()
    # nothing to do
    c.append(0, k[:0], k[:0], start=ints([0]))
    assert c.attention(0, k[:0], start=ints([0])).shape == (0, 2, 64)
    c.resize(ints([]), ints([]))
