"""The 8-bit paged key / value cache (``KV8Cache``): what its operators cost over the range they are used in.

Four kinds of pass:

* append: new key / value rows of a batch of sequences quantized into their pages, and the touched blocks read back;
* attend: attention of a batch's query rows over the cache, single tokens and prompts;
* fork: a sequence's pages handed to others (shared, or copied), and room for what those write next;
* compact: sequences that ended give their pages back, and the live pages move to the front of the pool.

A block is 16 tokens of one KV head, keys and values apart, with one f32 scale d = max|x| / 127 (rounded to f32) and
the codes nearest to x / d, halves away from zero. A block that gains tokens takes the larger of its scale and theirs,
and its earlier codes are rounded to the new one. Keys have a few channels several times as wide as the others, as
rotated keys of trained models do; lengths, head layouts and page sizes follow the repository's benchmark (14 query
heads over 2 KV heads of 64, 24 layers, a 512-token prompt) or are generic.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

BLOCK = 16
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def _package():
    """The framework's package: quanta.cpp_amd/ is not an importable name, so it is loaded by path."""
    if "quanta_cpp_amd" not in sys.modules:
        where = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quanta.cpp_amd")
        spec = importlib.util.spec_from_file_location("quanta_cpp_amd", os.path.join(where, "__init__.py"),
                                                      submodule_search_locations=[where])
        module = importlib.util.module_from_spec(spec)
        sys.modules["quanta_cpp_amd"] = module
        spec.loader.exec_module(module)
        module.init(0)
    return sys.modules["quanta_cpp_amd"]


# ------------------------------------------------------------------------------------------------ the cases

def _append(name, seqs, new, old, kv, hd, page, dtype):
    return {"name": name, "kind": "append", "seqs": seqs, "new": new, "old": old, "kv": kv, "hd": hd, "page": page,
            "dtype": dtype}


def _attend(name, seqs, new, old, heads, kv, hd, page, dtype, causal=True):
    return {"name": name, "kind": "attend", "seqs": seqs, "new": new, "old": old, "heads": heads, "kv": kv, "hd": hd,
            "page": page, "dtype": dtype, "causal": causal}


def _fork(name, parents, children, tokens, grow, copy, layers, kv, hd, page):
    return {"name": name, "kind": "fork", "parents": parents, "children": children, "tokens": tokens, "grow": grow,
            "copy": copy, "layers": layers, "kv": kv, "hd": hd, "page": page}


def _compact(name, seqs, tokens, ended, layers, kv, hd, page):
    return {"name": name, "kind": "compact", "seqs": seqs, "tokens": tokens, "ended": ended, "layers": layers, "kv": kv,
            "hd": hd, "page": page}


def listed():
    return [
        # One decode step of a few conversations on the benchmark's heads: one token each. The smallest store.
        _append("append_step", 8, 1, 700, 2, 64, 64, "f32"),
        # Prompts of mixed lengths admitted together, some behind a kept context that ends inside a block.
        _append("append_prompts", 12, 700, 90, 8, 128, 32, "f16"),
        # A long document stored in one call.
        _append("append_document", 1, 24001, 0, 8, 128, 256, "f32"),
        # The benchmark's conversation: one token after 600, where only latency counts.
        _attend("attend_step", 1, 1, 600, 14, 2, 64, 64, "f32"),
        # A server's decode step: conversations of mixed lengths, pages smaller than a tile of keys.
        _attend("attend_step_batch", 48, 1, 5000, 32, 8, 128, 16, "f16"),
        # Two very long contexts: few rows, the length split over the whole card.
        _attend("attend_step_long", 2, 1, 131000, 12, 2, 128, 256, "f32"),
        # Four drafted tokens each, checked at once.
        _attend("attend_draft", 16, 4, 3000, 14, 2, 64, 32, "f16"),
        # The benchmark's 512-token prompt.
        _attend("attend_prompt", 1, 512, 0, 14, 2, 64, 64, "f32"),
        # Long prompts in chunks behind what is cached already, one query head layout of larger models.
        _attend("attend_prompt_long", 4, 2000, 6000, 32, 8, 128, 64, "f16"),
        # Several replies to one prompt: its pages shared, the partly filled one copied as the replies grow.
        _fork("fork_replies", 1, 4, 530, 1, False, 24, 2, 64, 64),
        # Conversations copied whole, to be edited apart.
        _fork("fork_copies", 8, 2, 1500, 40, True, 24, 2, 64, 16),
        # A busy pool after many replies ended.
        _compact("compact_pool", 300, 900, 90, 24, 2, 64, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (8, 8, 64), (4, 4, 128), (16, 1, 128), (4, 1, 64), (40, 2, 64)]


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "fork", "compact"])
    heads, kv, hd = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["f32", "f16"])
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 6000)])
        seqs = min(_log(rng, 1, 64), max(1, 24000 // new))
        return _append(None, seqs, new, rng.choice([0, _log(rng, 1, 3000)]), kv, hd, page, dtype)
    if kind == "attend":
        new = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 2500)])
        seqs = min(_log(rng, 1, 64), max(1, 6000 // new))
        old = rng.choice([0, _log(rng, 1, 200), min(_log(rng, 200, 100000), 250000 // seqs)])
        causal = rng.random() < 0.85
        # no more work than the longest listed prompts
        while seqs * new * heads * hd * (new / 2 + old) > 4 * 2000 * 32 * 128 * 6000:
            old, new = old // 2, max(1, new // 2)
        return _attend(None, seqs, new, old, heads, kv, hd, page, dtype, causal)
    layers = _log(rng, 1, 24)
    if kind == "fork":
        return _fork(None, _log(rng, 1, 8), _log(rng, 1, 4), _log(rng, 1, 2000), _log(rng, 1, 200), rng.random() < 0.5,
                     layers, min(kv, 2), hd if kv == 1 else 64, page)
    seqs = _log(rng, 2, 200)
    return _compact(None, seqs, _log(rng, 4, 900), rng.randint(1, seqs - 1), layers, min(kv, 2), 64, page)


# --------------------------------------------------------------------------------- what a case's sizes come to

def _plan(case):
    """Host-side sizes of a case, the same for every seed: per sequence the tokens cached before (old) and new."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    if case["kind"] in ("append", "attend"):
        n = case["seqs"]
        # the longest sequence has the case's sizes, the others spread below it
        new = [case["new"]] + [max(1, int(case["new"] * rng.uniform(0.1, 1))) for _ in range(n - 1)]
        if case["new"] <= 8:
            new = [case["new"]] * n
        old = [case["old"]] + [int(case["old"] * rng.uniform(0.02, 1)) for _ in range(n - 1)]
        lens = [a + b for a, b in zip(old, new)]
        return {"old": old, "new": new, "lens": lens}
    if case["kind"] == "fork":
        return {"lens": [case["tokens"]] + [max(1, int(case["tokens"] * rng.uniform(0.3, 1)))
                                            for _ in range(case["parents"] - 1)]}
    lens = [max(1, int(case["tokens"] * rng.uniform(0.1, 1))) for _ in range(case["seqs"])]
    order = list(range(case["seqs"]))
    rng.shuffle(order)
    # pages as a pool has them after some time: taken in turns, by whichever sequence grew
    need = [-(-l // case["page"]) for l in lens]
    turns = [s for s in range(case["seqs"]) for _ in range(need[s])]
    rng.shuffle(turns)
    return {"lens": lens, "ended": sorted(order[:case["ended"]]), "turns": turns}


def _pages_of(tokens, page):
    return -(-tokens // page)


def _page_bytes(case):
    raw = 2 * case["kv"] * case["page"] * case["hd"] + 8 * case["kv"] * (case["page"] // BLOCK)
    return (raw + 127) // 128 * 128


def work(case):
    p, kv, hd = _plan(case), case["kv"], case["hd"]
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "f32" else 2
        n = sum(p["new"])
        back = n + sum(o % BLOCK for o in p["old"])  # earlier tokens of the touched blocks, read back too
        blocks = sum(_pages_of(o % BLOCK + m, BLOCK) for o, m in zip(p["old"], p["new"]))
        return {"bytes": 2 * kv * (n * hd * (size + 1) + back * hd * (1 + size) + 8 * blocks), "flops": 4 * kv * hd * n}
    if case["kind"] == "attend":
        size, heads = (4 if case["dtype"] == "f32" else 2), case["heads"]
        n, keys = sum(p["new"]), sum(p["lens"])
        seen = sum(m * o + m * (m + 1) // 2 if case["causal"] else m * (o + m) for o, m in zip(p["old"], p["new"]))
        return {"bytes": 2 * n * heads * hd * size + 2 * kv * (keys * hd + 4 * keys // BLOCK),
                "flops": 4 * hd * heads * seen}
    if case["kind"] == "fork":
        c = case["children"]
        if case["copy"]:
            moved = sum(c * _pages_of(l, case["page"]) for l in p["lens"])
        else:
            moved = sum(c for l in p["lens"] if l % case["page"])
        taken = sum(c * _pages_of(l + case["grow"], case["page"]) for l in p["lens"])
        return {"bytes": 2 * moved * case["layers"] * _page_bytes(case) + 12 * taken, "flops": 0}
    need = [_pages_of(l, case["page"]) for l in p["lens"]]
    ended = set(p["ended"])
    live = sum(n for s, n in enumerate(need) if s not in ended)
    moved = sum(1 for i, s in enumerate(p["turns"]) if s not in ended and i >= live)
    return {"bytes": 2 * moved * case["layers"] * _page_bytes(case) + 8 * sum(need), "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _rows(gen, n, kv, hd):
    """Keys and values of n tokens, f32: keys with one channel in sixteen wider than the rest, values by head."""
    k = torch.randn(n, kv, hd, generator=gen, device=DEVICE)
    k *= 1.0 + 5.0 * (torch.arange(hd, device=DEVICE) % 16 == 3)
    v = torch.randn(n, kv, hd, generator=gen, device=DEVICE)
    v *= 0.25 * (1 + torch.arange(kv, device=DEVICE).view(1, kv, 1))
    return k, v


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _inputs(case, seed):
    """Old and new key / value rows, and the query rows, of an append or attend case: the same on every tree."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    p, dtype = _plan(case), _dtype(case)
    k0, v0 = (t.to(dtype) for t in _rows(gen, sum(p["old"]), case["kv"], case["hd"]))
    k1, v1 = (t.to(dtype) for t in _rows(gen, sum(p["new"]), case["kv"], case["hd"]))
    q = None
    if case["kind"] == "attend":
        q = torch.randn(sum(p["new"]), case["heads"], case["hd"], generator=gen, device=DEVICE).to(dtype)
    # the order in which the pool hands out pages
    n_pages = sum(_pages_of(l, case["page"]) for l in p["lens"])
    order = torch.randperm(n_pages, generator=gen, device=DEVICE)
    return p, k0, v0, k1, v1, q, order


def _touched(old, new, rows, page_of, page):
    """The 16-token blocks that new rows fall in: block number in the pool, the row of each of its 16 tokens (-1: not
    a new one) and how many earlier tokens it holds."""
    blocks, index, held = [], [], []
    first = 0
    for s, (o, m) in enumerate(zip(old, new)):
        for b in range(o // BLOCK, _pages_of(o + m, BLOCK)):
            at = b * BLOCK
            blocks.append(page_of[s][at // page] * (page // BLOCK) + at % page // BLOCK)
            index.append([first + t - o if o <= t < o + m else -1 for t in range(at, at + BLOCK)])
            held.append(max(0, min(o - at, BLOCK)))
        first += m
    return {"block": torch.tensor(blocks, device=DEVICE), "row": torch.tensor(index, device=DEVICE),
            "held": torch.tensor(held, device=DEVICE)}


def _prepare_cache(case, seed):
    p, k0, v0, k1, v1, q, order = _inputs(case, seed)
    n, page = len(p["lens"]), case["page"]
    need = [_pages_of(l, page) for l in p["lens"]]
    st = {"case": case, "start": _ints(_starts(p["new"])), "q": q, "n_new": sum(p["new"])}
    # new rows as a fused projection leaves them: keys and values side by side in one row
    kvrow = torch.cat([k1, v1], dim=1)
    st["k"], st["v"] = kvrow[:, :case["kv"]], kvrow[:, case["kv"]:]
    back = [o % BLOCK + m for o, m in zip(p["old"], p["new"])]
    st["back"], st["n_back"] = _ints(_starts(back)), sum(back)
    single = all(m == 1 for m in p["new"])
    if own:
        qh = _package()
        cache = qh.KV8Cache(1, sum(need), page, case["kv"], case["hd"], n, max(need), device=DEVICE)
        seqs = torch.arange(n, dtype=torch.int32, device=DEVICE)
        if sum(p["old"]):
            cache.resize(seqs, _ints(p["old"]))
            cache.append(0, k0, v0, start=_ints(_starts(p["old"])))
        cache.resize(seqs, _ints(p["lens"]))
        if case["kind"] == "attend":
            cache.append(0, k1, v1, start=st["start"])
        st["cache"] = cache
        st["start"] = None if single else st["start"]
        return st
    order = order.tolist()
    page_of = []
    for c in need:
        page_of.append(order[:c])
        order = order[c:]
    st["page_of"] = [torch.tensor(x, device=DEVICE) for x in page_of]
    shape = (sum(need) * (page // BLOCK), case["kv"], BLOCK, case["hd"])
    st["codes"] = [torch.zeros(shape, dtype=torch.int8, device=DEVICE) for _ in range(2)]
    st["scales"] = [torch.zeros(shape[:2], device=DEVICE) for _ in range(2)]
    if sum(p["old"]):
        _plain_append(st, _touched([0] * n, p["old"], k0, page_of, page), k0, v0)
    st["touched"] = _touched(p["old"], p["new"], k1, page_of, page)
    if case["kind"] == "attend":
        _plain_append(st, st["touched"], k1, v1)
    # rows of the pool that hold the tokens read back, and the cached tokens of each sequence
    slot = [[pg * page + t for pg in pages for t in range(page)] for pages in page_of]
    st["back_slots"] = torch.tensor([x for s in range(n) for x in slot[s][p["lens"][s] - back[s]:p["lens"][s]]],
                                    device=DEVICE)
    st["plan"] = p
    return st


def _prepare_pool(case, seed):
    """Page tables, counts and page contents of a fork or compact case."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    p, page = _plan(case), case["page"]
    need = [_pages_of(l, page) for l in p["lens"]]
    if case["kind"] == "fork":
        c, n = case["children"], case["parents"]
        grown = [_pages_of(l + case["grow"], page) for l in p["lens"]]
        n_seqs, n_pages = n * (1 + c), sum(need) + c * (sum(need if case["copy"] else [0]) + sum(grown)) + 3
        turns = [s for s in range(n) for _ in range(need[s])]
        random.Random(sum(need)).shuffle(turns)
        src = [s for s in range(n) for _ in range(c)]
        lists = {"src": _ints(src), "dst": _ints(list(range(n, n_seqs))),
                 "grown": _ints([p["lens"][s] + case["grow"] for s in src])}
        width = max(grown)
    else:
        n_seqs, n_pages, turns, width = case["seqs"], len(p["turns"]) + 5, p["turns"], max(need)
        lists = {"ended": _ints(p["ended"]), "none": _ints([0] * len(p["ended"]))}
    table = [[-1] * width for _ in range(n_seqs)]
    filled = [0] * n_seqs
    refs = [0] * n_pages
    for i, s in enumerate(turns):
        table[s][filled[s]] = i
        filled[s] += 1
        refs[i] = 1
    lens = p["lens"] + [0] * (n_seqs - len(p["lens"]))
    pages = torch.randint(0, 256, (case["layers"], n_pages, _page_bytes(case)), generator=gen, device=DEVICE,
                          dtype=torch.uint8)
    st = {"case": case, "lists": lists, "first": (_ints(table), _ints(lens), _ints(refs))}
    if own:
        cache = _package().KV8Cache(case["layers"], n_pages, page, case["kv"], case["hd"], n_seqs, width, device=DEVICE)
        cache.pages.copy_(pages)
        st["cache"] = cache
        st["held"] = (cache.table, cache.lens, cache.refs)
        st["pages"] = cache.pages
    else:
        st["held"] = tuple(torch.empty_like(t) for t in st["first"])
        st["pages"] = pages
    for a, b in zip(st["held"], st["first"]):
        a.copy_(b)
    return st


def prepare(case, seed):
    if case["kind"] in ("append", "attend"):
        return _prepare_cache(case, seed)
    return _prepare_pool(case, seed)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if kind == "append":
        return _own_append(state) if own else _plain_append_pass(state)
    if kind == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if kind == "fork":
        return _own_fork(state) if own else _plain_fork(state)
    return _own_compact(state) if own else _plain_compact(state)


def _own_append(st):
    cache = st["cache"]
    cache.append(0, st["k"], st["v"], start=st["start"])
    return cache.read(0, st["n_back"], start=st["back"], dtype=st["k"].dtype)


def _own_attend(st):
    return st["cache"].attention(0, st["q"], start=st["start"], causal=st["case"]["causal"])


def _own_fork(st):
    cache, lists = st["cache"], st["lists"]
    cache.fork(lists["src"], lists["dst"], copy=st["case"]["copy"])
    cache.resize(lists["dst"], lists["grown"])
    return {"table": cache.table, "lens": cache.lens, "refs": cache.refs, "pages": cache.pages}


def _own_compact(st):
    for a, b in zip(st["held"], st["first"]):  # the state before, so that every pass has the same pages to move
        a.copy_(b)
    cache, lists = st["cache"], st["lists"]
    cache.resize(lists["ended"], lists["none"])
    live = cache.compact()
    return {"live": live, "table": cache.table, "lens": cache.lens, "refs": cache.refs, "pages": cache.pages}


# ------------------------------------------------------------------------------------------------ plain forms

def _nearest(x):
    """Nearest integer, halves away from zero (64-bit x: quotients next to a half keep their side)."""
    return torch.sign(x) * torch.floor(x.abs() + 0.5)


def _block_scale(amax):
    """amax / 127 rounded once (a division by a number would be a product with its reciprocal)."""
    return (amax.double() / torch.full_like(amax, 127.0, dtype=torch.float64)).float()


def _plain_append(st, touched, k, v):
    block, row, held = touched["block"], touched["row"], touched["held"]
    if block.numel() == 0:
        return
    is_new = (row >= 0).view(-1, 1, BLOCK, 1)
    is_old = (torch.arange(BLOCK, device=row.device) < held.view(-1, 1)).view(-1, 1, BLOCK, 1)
    for which, x in enumerate((k, v)):
        x = x.float()[row.clamp(min=0)].transpose(1, 2) * is_new  # [blocks][kv][16][hd]
        codes, scales = st["codes"][which], st["scales"][which]
        before = scales[block] * (held > 0).view(-1, 1)
        now = torch.maximum(before, _block_scale(x.abs().amax((2, 3))))
        at = now.double().clamp(min=1e-300).view(now.shape + (1, 1))
        fresh = _nearest(x.double() / at)
        kept = _nearest(codes[block].double() * before.double().view(before.shape + (1, 1)) / at)
        codes[block] = torch.where(is_new, fresh, torch.where(is_old, kept, torch.zeros_like(kept))).to(torch.int8)
        scales[block] = now


def _plain_append_pass(st):
    _plain_append(st, st["touched"], st["k"], st["v"])
    case, out = st["case"], []
    for codes, scales in zip(st["codes"], st["scales"]):
        c = codes.transpose(1, 2).reshape(-1, case["kv"], case["hd"])[st["back_slots"]]
        d = scales[st["back_slots"] // BLOCK]
        out.append((c.float() * d.unsqueeze(-1)).to(st["k"].dtype))
    return tuple(out)


def _plain_attend(st):
    case, p = st["case"], st["plan"]
    kv, hd, group = case["kv"], case["hd"], case["heads"] // case["kv"]
    per = case["page"] // BLOCK
    out = torch.empty_like(st["q"])
    first = 0
    for s, (m, length) in enumerate(zip(p["new"], p["lens"])):
        blocks = (st["page_of"][s].view(-1, 1) * per + torch.arange(per, device=DEVICE)).view(-1)
        keys, values = ((c[blocks].float() * d[blocks].view(-1, kv, 1, 1)).transpose(0, 1).reshape(kv, -1, hd)[:, :length]
                        for c, d in zip(st["codes"], st["scales"]))
        q = st["q"][first:first + m].float().view(m, kv, group, hd).permute(1, 2, 0, 3).reshape(kv, group * m, hd)
        scores = torch.matmul(q, keys.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(hd))
        if case["causal"]:
            hidden = torch.arange(length, device=DEVICE) > torch.arange(length - m, length, device=DEVICE).view(m, 1)
            scores = scores.view(kv, group, m, length).masked_fill(hidden, -math.inf).view(kv, group * m, length)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(e, values.contiguous()) / e.sum(-1, keepdim=True)
        out[first:first + m] = o.view(kv, group, m, hd).permute(2, 0, 1, 3).reshape(m, kv * group, hd).to(out.dtype)
        first += m
    return out


def _drop_refs(refs, rows):
    """One count less for each page in rows (-1: none)."""
    held = rows.reshape(-1).long()
    refs.index_add_(0, held.clamp(min=0), -(held >= 0).to(torch.int32))


def _plain_resize(st, seqs, lens_new):
    table, lens, refs = st["held"]
    page, width = st["case"]["page"], table.shape[1]
    column = torch.arange(width, device=DEVICE)
    seqs = seqs.long()
    before, after = lens[seqs], lens_new
    n_before, n_after = (before + page - 1) // page, (after + page - 1) // page
    rows = table[seqs]
    gone = (column >= n_after.view(-1, 1)) & (column < n_before.view(-1, 1))
    _drop_refs(refs, torch.where(gone, rows, -1))
    rows = torch.where(gone, -1, rows)
    # a partly filled last page that others hold too is replaced by a copy where its sequence grows
    last = (n_before - 1).clamp(min=0).long().view(-1, 1)
    old_last = rows.gather(1, last).view(-1)
    split = (after > before) & (before % page != 0) & (refs[old_last.long().clamp(min=0)] > 1)
    wants = ((column >= n_before.view(-1, 1)) & (column < n_after.view(-1, 1))) | (split.view(-1, 1) & (column == last))
    free = torch.nonzero(refs == 0).view(-1)
    where = torch.nonzero(wants)
    assert where.shape[0] <= free.shape[0], "the cases have pages enough"
    taken = free[:where.shape[0]]
    _drop_refs(refs, torch.where(split, old_last, -1))
    rows[where[:, 0], where[:, 1]] = taken.to(torch.int32)
    refs[taken] = 1
    table[seqs], lens[seqs] = rows, after
    who = torch.nonzero(split).view(-1)
    if who.numel():
        st["pages"][:, rows[who, last.view(-1)[who]].long()] = st["pages"][:, old_last[who].long()]


def _plain_fork(st):
    table, lens, refs = st["held"]
    case, lists = st["case"], st["lists"]
    src, dst = lists["src"].long(), lists["dst"].long()
    _drop_refs(refs, table[dst])
    rows = table[src]
    if case["copy"]:
        where = torch.nonzero(rows >= 0)
        taken = torch.nonzero(refs == 0).view(-1)[:where.shape[0]]
        st["pages"][:, taken] = st["pages"][:, rows[where[:, 0], where[:, 1]].long()]
        rows[where[:, 0], where[:, 1]] = taken.to(torch.int32)
        refs[taken] = 1
    else:
        held = rows.reshape(-1).long()
        refs.index_add_(0, held.clamp(min=0), (held >= 0).to(torch.int32))
    table[dst], lens[dst] = rows, lens[src]
    _plain_resize(st, lists["dst"], lists["grown"])
    return {"table": table, "lens": lens, "refs": refs, "pages": st["pages"]}


def _plain_compact(st):
    for a, b in zip(st["held"], st["first"]):
        a.copy_(b)
    table, lens, refs = st["held"]
    _plain_resize(st, st["lists"]["ended"], st["lists"]["none"])
    live = (refs > 0).sum()
    index = torch.arange(refs.numel(), device=DEVICE)
    high = torch.nonzero((refs > 0) & (index >= live)).view(-1)
    hole = torch.nonzero((refs == 0) & (index < live)).view(-1)
    st["pages"][:, hole] = st["pages"][:, high]
    goes = index.to(torch.int32)
    goes[high] = hole.to(torch.int32)
    refs[hole] = refs[high]
    refs[high] = 0
    table.copy_(torch.where(table >= 0, goes[table.long().clamp(min=0)], table))
    return {"live": live.to(torch.int32).view(1), "table": table, "lens": lens, "refs": refs, "pages": st["pages"]}


# ------------------------------------------------------------------------------------------------ from the definition

def _exact_sequence(old, new):
    """One sequence's stored values of one KV head batch, 64 bits: rows old [o][kv][hd], then rows new behind them."""
    def blocks_of(x, head):  # tokens grouped in blocks, the first of which has `head` places taken
        n, kv, hd = x.shape
        tail = -(head + n) % BLOCK
        pad = torch.zeros(head, kv, hd, dtype=torch.float64, device=x.device)
        end = torch.zeros(tail, kv, hd, dtype=torch.float64, device=x.device)
        return torch.cat([pad, x.double(), end]).view(-1, BLOCK, kv, hd)

    def scale(blocks):
        top = blocks.abs().amax(dim=(1, 3))  # [blocks][kv]
        return torch.div(top, 127.0 * torch.ones_like(top)).float().double()

    def codes(values, d):
        ratio = values / torch.where(d > 0, d, torch.ones_like(d))[:, None, :, None]
        return torch.trunc(ratio + torch.copysign(torch.full_like(ratio, 0.5), ratio))

    o = old.shape[0]
    a = blocks_of(old, 0)
    da = scale(a)
    ca = codes(a, da)
    head = o % BLOCK
    b = blocks_of(new, head)
    db = scale(b)
    cb = codes(b, db)
    if head:
        d = torch.maximum(da[-1:], db[:1])
        cb[:1] = codes(b[:1], d)
        cb[:1, :head] = codes(ca[-1:] * da[-1:][:, None, :, None], d)[:, :head]
        db[:1] = d
        ca, da = ca[:-1], da[:-1]
    values = torch.cat([ca * da[:, None, :, None], cb * db[:, None, :, None]])
    return values.reshape(-1, old.shape[1], old.shape[2])[:o + new.shape[0]]


def exact(case, seed):
    if case["kind"] not in ("append", "attend"):
        return None  # whole numbers only
    p, k0, v0, k1, v1, q, _ = _inputs(case, seed)
    kv, hd = case["kv"], case["hd"]
    a = b = 0
    back, outs = ([], []), []
    for o, m in zip(p["old"], p["new"]):
        keys, values = (_exact_sequence(x[a:a + o], y[b:b + m]) for x, y in ((k0, k1), (v0, v1)))
        if case["kind"] == "append":
            for to, x in zip(back, (keys, values)):
                to.append(x[o - o % BLOCK:])
        else:
            group, length = case["heads"] // kv, o + m
            rows = q[b:b + m].double()
            out = torch.empty(m, case["heads"], hd, dtype=torch.float64, device=q.device)
            limit = torch.arange(o, length, device=q.device).view(m, 1)
            for h in range(case["heads"]):
                g = h // group
                s = rows[:, h] @ keys[:, g].t().contiguous() / math.sqrt(hd)
                if case["causal"]:
                    s = torch.where(torch.arange(length, device=q.device) <= limit, s, -math.inf)
                w = torch.softmax(s, dim=-1)
                out[:, h] = w @ values[:, g]
            outs.append(out)
        a, b = a + o, b + m
    if case["kind"] == "append":
        return tuple(torch.cat(x) for x in back)
    return torch.cat(outs)
