"""Attention over an 8-bit cache in 64 bits from what the cache holds (its values read back, its scales from the page bytes),
and how far a result may be off: from the roundings of each step, of positions that the row sees and nothing else.

The values read back are checked against the plain model (kv8_util) bit for bit elsewhere."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}  # half a step of the format, relative to a value


def value_scales(cache, layer, seq):
    """Scales of a sequence's value blocks, [blocks][kv], 64 bits (pages: codes of keys and values, then the scales f32
    [keys, values][kv][blocks of a page]; the sign is a mark of its own)."""
    per, kv = cache.page_tokens // 16, cache.n_kv_heads
    at, n = 2 * kv * cache.page_tokens * cache.head_dim, 2 * kv * per
    length = int(cache.lens[seq])
    pages = cache.table[seq, :-(-length // cache.page_tokens)].long()
    raw = cache.pages[layer, pages, at:at + 4 * n].contiguous().view(torch.float32)
    return raw.view(-1, 2, kv, per)[:, 1].transpose(1, 2).reshape(-1, kv).abs().double()


def exact_attention(cache, layer, q, seqs, counts, causal=True, scale=None, two=None):
    """(out, bound) of rows q [rows][heads][hd] in 64 bits; two: weights as two f16 each (None: in f32 calls). A row that
    sees nothing is 0.

    A score is off by dx: the f32 query in two f16 (2^-22 of each value and, in f16's subnormals, 2^-38 of the row's largest;
    an f16 query is exact), 2 hd products summed (hd for f16 queries), and 8 roundings of unit, scales and products. The
    weight's relative error is dx, once above and once below the fraction. A weight itself: its exponential and products, 10
    roundings; its format, two f16 (2^-22) or one (2^-11); and in f16's subnormals half of 2^-24, where the row's largest
    weight times value scale stands at 2^6 at least, so 2^-31 of that for each code (the largest of tokens whose values are
    not all zero: the others count in the sum of weights alone). Sums over the n positions that the
    row sees: n roundings above and below, and 32 of joins."""
    hd, heads = cache.head_dim, q.shape[1]
    group = heads // cache.n_kv_heads
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    row, f32 = 0, q.dtype == torch.float32
    two = f32 if two is None else two
    start = lambda n: torch.tensor([0, n], dtype=torch.int32, device=q.device)
    for s, m in zip(seqs, counts):
        n = int(cache.lens[s]) if 0 <= s < cache.n_seqs else 0
        if n == 0 or m == 0:
            row += m
            continue
        k, v = (t.double() for t in cache.read(layer, n, start=start(n), seqs=torch.tensor([s], dtype=torch.int32, device=q.device)))
        d = value_scales(cache, layer, s)
        d = d.repeat_interleave(16, 0)[:n]
        pos = torch.arange(n, device=q.device)
        see = torch.arange(n - m, n, device=q.device).clamp(max=n - 1) if causal else torch.full((m,), n - 1, device=q.device)
        for h in range(heads):
            g = h // group
            x = q[row:row + m, h].double()
            kt = k[:, g].t().contiguous()
            hidden = pos[None] > see[:, None]
            sc = (x @ kt * scale).masked_fill(hidden, float("-inf"))
            top = sc.amax(1, keepdim=True)
            p = torch.exp(sc - top.clamp(min=-1e300))
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total.clamp(min=1e-300), torch.zeros_like(p))
            o = p @ v[:, g]
            av = v[:, g].abs()
            size = (x.abs() @ kt.abs() * abs(scale)).masked_fill(hidden, 0).amax(1)
            seen = (see + 1).clamp(min=0).double()
            if f32:
                dx = size * (2.0 ** -22 + (2 * hd + 8) * 2.0 ** -24)
                far = kt.abs().sum(0)[None].expand(m, n).masked_fill(hidden, 0).amax(1)
                dx = dx + 2.0 ** -38 * x.abs().amax(1) * far * abs(scale)
            else:
                dx = size * (hd + 8) * 2.0 ** -24
            rel = 2 * dx + 10 * 2.0 ** -24 + (2.0 ** -22 if two else 2.0 ** -11) + 2 * (seen + 32) * 2.0 ** -24
            largest = (p * (d[:, g] * (av.amax(1) > 0))[None]).amax(1)
            codes = (av / d[:, g, None].clamp(min=1e-300))
            codes = (~hidden).double() @ codes
            off = rel[:, None] * (p @ av) + 2.0 ** -31 * largest[:, None] * codes
            out[row:row + m, h] = o
            bound[row:row + m, h] = off + o.abs() * HALF[q.dtype] + (1e-37 if f32 else 2.0 ** -25)
        row += m
    return out, bound


def worst(got, want, bound):
    """Where got is furthest past its bound: (error / bound, index), for the message of an assertion."""
    ratio = (got.double() - want).abs() / bound
    ratio = torch.where(bound == 0, (got.double() != want).double() * 1e9, ratio)
    ratio = torch.where(torch.isnan(ratio), torch.full_like(ratio, 1e12), ratio)
    i = int(ratio.argmax())
    return float(ratio.flatten()[i]), tuple(int(t) for t in torch.unravel_index(torch.tensor(i), ratio.shape))


# ---- caches and inputs of the tests

def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def starts(counts):
    return ints(np.concatenate([[0], np.cumsum(counts)]))


def filled(qh, k, v, lens, page=32, seq_pages=None):
    """A cache that holds the rows k and v of sequences of these lengths."""
    need = [-(-n // page) for n in lens]
    c = qh.KV8Cache(1, sum(need) + 1, page, k.shape[1], k.shape[2], len(lens), seq_pages or max(need))
    c.pages.fill_(0x7f)
    c.resize(ints(range(len(lens))), ints(lens))
    c.append(0, k, v, start=starts(lens))
    return c


def randn(seed, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen)
