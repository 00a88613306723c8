"""A plain model of the 8-bit paged cache (quanta_hip.h, qh_kv8_*): numpy, 64 bits, one token or page at a time."""
import numpy as np

BLOCK = 16


def nearest(x):
    """Nearest integer, halves away from zero."""
    return np.sign(x) * np.floor(np.abs(x) + 0.5)


def block_scale(amax):
    return np.float32(np.float64(amax) / 127.0)


class PlainKV8:
    def __init__(self, n_layers, n_pages, page_tokens, kv, hd, n_seqs, seq_pages):
        self.layers, self.n_pages, self.page, self.kv, self.hd = n_layers, n_pages, page_tokens, kv, hd
        self.table = np.full((n_seqs, seq_pages), -1, np.int64)
        self.lens = np.zeros(n_seqs, np.int64)
        self.refs = np.zeros(n_pages, np.int64)
        self.status = 0
        blocks = page_tokens // BLOCK
        self.codes = np.zeros((n_layers, n_pages, blocks, 2, kv, BLOCK, hd))
        self.scale = np.zeros((n_layers, n_pages, blocks, 2, kv))
        self.copied = []  # (from, to) of every page copy, in order

    # ---- pages
    def need(self, tokens):
        return -(-tokens // self.page)

    def _drop(self, s, first):
        for j in range(first, self.need(self.lens[s])):
            self.refs[self.table[s, j]] -= 1
            self.table[s, j] = -1

    def _copy(self, a, b):
        self.codes[:, b] = self.codes[:, a]
        self.scale[:, b] = self.scale[:, a]
        self.copied.append((int(a), int(b)))

    def resize(self, seqs, lens):
        cap = self.table.shape[1] * self.page
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lens) for s in seqs) or any(
                not 0 <= n <= cap for n in lens):
            self.status |= 2
            return
        for s, n in zip(seqs, lens):
            if n <= self.lens[s]:
                self._drop(s, self.need(n))
                self.lens[s] = n
        growers = [(s, n) for s, n in zip(seqs, lens) if n > self.lens[s]]
        split = [bool(self.lens[s] % self.page) and self.refs[self.table[s, self.need(self.lens[s]) - 1]] > 1
                 for s, _ in growers]
        free = [int(p) for p in np.nonzero(self.refs == 0)[0]]
        if sum(self.need(n) - self.need(self.lens[s]) + sp for (s, n), sp in zip(growers, split)) > len(free):
            self.status |= 1
            return
        copies = []
        for (s, n), sp in zip(growers, split):
            have = self.need(self.lens[s])
            if sp:
                old, new = self.table[s, have - 1], free.pop(0)
                copies.append((old, new))
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[s, have - 1] = new
            for j in range(have, self.need(n)):
                p = free.pop(0)
                self.table[s, j], self.refs[p] = p, 1
            self.lens[s] = n
        for a, b in copies:
            self._copy(a, b)

    def fork(self, src, dst, copy):
        n = len(self.lens)
        if len(set(dst)) < len(dst) or set(src) & set(dst) or any(not 0 <= s < n for s in list(src) + list(dst)):
            self.status |= 2
            return
        for d in dst:
            self._drop(d, 0)
            self.lens[d] = 0
        if not copy:
            for s, d in zip(src, dst):
                for j in range(self.need(self.lens[s])):
                    self.table[d, j] = self.table[s, j]
                    self.refs[self.table[s, j]] += 1
                self.lens[d] = self.lens[s]
            return
        free = [int(p) for p in np.nonzero(self.refs == 0)[0]]
        if sum(self.need(self.lens[s]) for s in src) > len(free):
            self.status |= 1
            return
        for s, d in zip(src, dst):
            for j in range(self.need(self.lens[s])):
                p = free.pop(0)
                self._copy(self.table[s, j], p)
                self.table[d, j], self.refs[p] = p, 1
            self.lens[d] = self.lens[s]

    def compact(self):
        live = int((self.refs > 0).sum())
        high = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        holes = [p for p in range(live) if self.refs[p] == 0]
        for a, b in zip(high, holes):
            self._copy(a, b)
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b
        return live

    # ---- tokens
    def at(self, s, pos):
        return self.table[s, pos // self.page], pos % self.page // BLOCK, pos % BLOCK

    def append(self, layer, seqs, counts, k, v):
        """k, v: float arrays [rows][kv][hd]."""
        row = 0
        for s, m in zip(seqs, counts):
            if not 0 <= s < len(self.lens):
                row += m
                continue
            end = int(self.lens[s])
            p0 = end - m
            first = max(p0, 0)
            for b in range(first // BLOCK, -(-end // BLOCK)):
                lo, hi = max(first, b * BLOCK), min(end, (b + 1) * BLOCK)
                page, blk, _ = self.at(s, b * BLOCK)
                if page < 0:
                    continue
                if self.refs[page] > 1:
                    self.status |= 4
                    continue
                held = lo - b * BLOCK
                for w, x in enumerate((k, v)):
                    rows = x[row + lo - p0:row + hi - p0].astype(np.float64)
                    for h in range(self.kv):
                        top = np.abs(rows[:, h]).max()
                        before = self.scale[layer, page, blk, w, h] if held else 0.0
                        c = self.codes[layer, page, blk, w, h]
                        if not np.isfinite(top) or np.isnan(before):
                            d = np.nan
                        else:
                            d = max(np.float64(block_scale(top)), before)
                        if not d > 0:
                            c[:] = 0
                        else:
                            c[:held] = np.minimum(nearest(np.abs(c[:held]) * before / d), 127) * np.sign(c[:held])
                            c[held:] = 0
                            c[held:held + hi - lo] = np.clip(nearest(rows[:, h] / d), -127, 127)
                        self.scale[layer, page, blk, w, h] = d
            row += m

    def values(self, layer, s):
        """Stored values of a sequence, f32: (k, v) [len][kv][hd]."""
        n = int(self.lens[s])
        out = np.zeros((2, n, self.kv, self.hd), np.float32)
        for p in range(n):
            page, blk, t = self.at(s, p)
            if page >= 0:
                out[:, p] = (self.codes[layer, page, blk, :, :, t].astype(np.float32) *
                             self.scale[layer, page, blk].astype(np.float32)[..., None])
        return out[0], out[1]

    def attention(self, layer, seqs, counts, q, causal, scale):
        """(out, spread, score, small) of rows q [rows][heads][hd], 64 bits: the result, sum p |v|, the largest sum of
        |q k| * scale that a row's scores come from (what the errors of sums are measured by), and the sum of |code| times
        the largest value scale of the sequence's head."""
        heads = q.shape[1]
        group = heads // self.kv
        out = np.zeros(q.shape)
        spread = np.zeros(q.shape)
        small = np.zeros(q.shape)
        score = np.zeros(q.shape[:2])
        row = 0
        for s, m in zip(seqs, counts):
            known = 0 <= s < len(self.lens)
            k, v = (x.astype(np.float64) for x in self.values(layer, s)) if known else (np.zeros((0, self.kv, self.hd)),) * 2
            n = k.shape[0]
            top = np.zeros(self.kv)
            code = np.zeros(k.shape)
            for p in range(n):
                page, blk, t = self.at(s, p)
                if page >= 0:
                    d = self.scale[layer, page, blk, 1]
                    top = np.fmax(top, d)
                    code[p] = np.abs(self.codes[layer, page, blk, 1, :, t])
            for i in range(m):
                see = min(max(n - m + i + 1, 0), n) if causal else n
                if see == 0:
                    continue
                for h in range(heads):
                    g = h // group
                    qq = q[row + i, h].astype(np.float64)
                    x = k[:see, g] @ qq * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[row + i, h] = p @ v[:see, g]
                    spread[row + i, h] = p @ np.abs(v[:see, g])
                    small[row + i, h] = top[g] * code[:see, g].sum(0)
                    score[row + i, h] = (np.abs(k[:see, g]) @ np.abs(qq)).max() * abs(scale)
            row += m
        return out, spread, score, small


def attention_bound(dtype, out, spread, score, small, n, hd):
    """How far a result may be off, from the number formats alone (a rounding is half a step: f32 2^-24, f16 2^-11).
    A score: the query split keeps 2^-22 of each product (two f16 of 11 bits), hd products and their sum round at most
    hd + 4 times, scale, key scale, unit and maximum four times more: all relative to sum |q k| scale, and a weight's
    relative error is the score's absolute one; twice, for the sum below the fraction too. A weight: exp2 and its product
    with the value scale, five roundings, and its own format: two f16 (2^-22) or one (2^-11). The sums over n positions
    round n times, in both parts of the fraction; joining partial results adds sixteen. The smallest weights end in f16's
    subnormals: a weight (times its value scale, over a unit of at most twice the largest scale, times 2^6) is off by at
    most half their step of 2^-24, so a position by 2^-25 / 2^6 * 2 * largest scale * |code| = 2^-30 of them; the weights'
    sum is at least 1."""
    f32 = dtype == "f32"
    weight = 2 * score * (2.0 ** -22 + (hd + 8) * 2.0 ** -24)
    rel = weight + 10 * 2.0 ** -24 + (2.0 ** -22 if f32 else 2.0 ** -11) + 2 * (n + 16) * 2.0 ** -24
    bound = spread * rel[..., None] + small * 2.0 ** -30
    return bound + (np.abs(out) * 2.0 ** -24 + 1e-37 if f32 else np.abs(out) * 2.0 ** -11 + 2.0 ** -25)
