"""What a step of many sequences does around the 8-bit paged cache: its cost over the range it is used in.

Five kinds of pass:

* norm: root-mean-square norm of rows, with the residual's addition before it, into rows of the same type or into 8-bit
  blocks of 32 with a scale each, as the quantized matmuls take them;
* rope: rotary positions of the query and key heads, as a fused projection leaves them in one row;
* attend: causal attention of whole prompts, packed end to end, over their own keys and values before those are rounded to
  8 bits (or of new rows behind kept ones, or over states that are not their own);
* beam: the best continuations of each prompt's beams over beams and vocabulary;
* reorder: the cache's sequences become those beams' sequences, and room for each beam's next token.

Sizes follow the repository's benchmark (rows of 896, 14 query heads over 2 KV heads of 64, a vocabulary of 151,936, 24
layers) or are generic.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

BLOCK = 32
EPS = 1e-6
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

def _norm(name, tokens, width, dtype, residual, form):
    return {"name": name, "kind": "norm", "tokens": tokens, "width": width, "dtype": dtype, "residual": residual,
            "form": form}


def _rope(name, tokens, heads, kv, hd, rot, interleaved, scaling, last, dtype):
    return {"name": name, "kind": "rope", "tokens": tokens, "heads": heads, "kv": kv, "hd": hd, "rot": rot,
            "interleaved": interleaved, "scaling": scaling, "last": last, "dtype": dtype}


def _attend(name, seqs, new, behind, heads, kv, hd, causal, dtype):
    return {"name": name, "kind": "attend", "seqs": seqs, "new": new, "behind": behind, "heads": heads, "kv": kv, "hd": hd,
            "causal": causal, "dtype": dtype}


def _beam(name, prompts, beams, vocab, k, dtype):
    return {"name": name, "kind": "beam", "prompts": prompts, "beams": beams, "vocab": vocab, "k": k, "dtype": dtype}


def _reorder(name, prompts, beams, tokens, layers, kv, hd, page):
    return {"name": name, "kind": "reorder", "prompts": prompts, "beams": beams, "tokens": tokens, "layers": layers,
            "kv": kv, "hd": hd, "page": page}


def listed():
    return [
        # One decode step of one conversation on the benchmark's rows, where only latency counts.
        _norm("norm_step", 1, 896, "f32", True, "q8"),
        # A batch of long prompts on the rows of a larger model, into what its quantized projections take.
        _norm("norm_prompts", 4001, 5120, "f32", True, "q8"),
        # The same for unquantized projections, in f16: the largest norm.
        _norm("norm_rows", 16000, 4096, "f16", True, "rows"),
        # A server's decode step: one token each of conversations of mixed lengths, the benchmark's heads.
        _rope("rope_step", 48, 14, 2, 64, 64, False, "none", 5000, "f32"),
        # Long prompts in contexts stretched past the trained length.
        _rope("rope_prompts", 8000, 32, 8, 128, 128, False, "parts", 130000, "f16"),
        # The benchmark's 512-token prompt, in the type that the quantized projections give.
        _attend("attend_prompt", 1, 512, 0, 14, 2, 64, True, "f32"),
        # A batch of prompts of mixed lengths, packed.
        _attend("attend_packed", 16, 2000, 0, 14, 2, 64, True, "f32"),
        # A long document on the heads of a larger model.
        _attend("attend_long", 1, 12001, 0, 32, 8, 128, True, "f16"),
        # Four beams of one prompt over the benchmark's vocabulary.
        _beam("beam_step", 1, 4, 151936, 8, "f32"),
        # A batch of prompts.
        _beam("beam_batch", 24, 8, 151936, 16, "f32"),
        # The four beams' sequences in the cache.
        _reorder("reorder_step", 1, 4, 600, 24, 2, 64, 64),
        # A batch's, in small pages.
        _reorder("reorder_batch", 64, 8, 3000, 4, 2, 64, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (8, 8, 64), (4, 4, 128), (16, 1, 256), (4, 1, 80), (40, 2, 64)]


def draw(rng):
    kind = rng.choice(["norm", "norm", "rope", "rope", "attend", "attend", "attend", "beam", "beam", "reorder"])
    dtype = rng.choice(["f32", "f16"])
    heads, kv, hd = rng.choice(_HEADS)
    if kind == "norm":
        form = rng.choice(["q8", "rows"])
        width = 32 * _log(rng, 1, 256) if form == "q8" else _log(rng, 1, 8192)
        return _norm(None, min(_log(rng, 1, 16000), 30000000 // width), width, dtype, rng.random() < 0.75, form)
    if kind == "rope":
        rot = rng.choice([hd, hd, 2 * rng.randint(1, hd // 2)])
        return _rope(None, min(_log(rng, 1, 8000), 32000000 // ((heads + kv) * hd)), heads, kv, hd, rot,
                     rng.random() < 0.4, rng.choice(["none", "linear", "base", "parts"]), _log(rng, 100, 1000000), dtype)
    if kind == "attend":
        hd = 64 if hd == 64 else 128
        new, behind = _log(rng, 1, 6000), rng.choice([0, 0, _log(rng, 1, 4000)])
        seqs = max(1, min(_log(rng, 1, 64), 500000000 // (heads * new * (new + behind))))
        return _attend(None, seqs, new, behind, heads, kv, hd, rng.random() < 0.8, dtype)
    if kind == "beam":
        beams, vocab = _log(rng, 1, 40), _log(rng, 40, 200000)
        k = min(rng.choice([1, beams, 2 * beams, _log(rng, 1, 256)]), beams * vocab, 256)
        return _beam(None, min(_log(rng, 1, 64), max(1, 28000000 // (beams * vocab))), beams, vocab, k, dtype)
    prompts, beams = _log(rng, 1, 64), _log(rng, 1, 12)
    page = rng.choice([16, 32, 64, 128, 256])
    layers = max(1, min(_log(rng, 1, 24), 500000 // (prompts * beams * page)))
    return _reorder(None, prompts, beams, _log(rng, 1, 24000 // (prompts + 7)), layers, min(kv, 2),
                    64 if hd == 64 else 128, page)


# --------------------------------------------------------------------------------- what a case's sizes come to

def _ceil(a, b):
    return -(-a // b)


def _page_bytes(case):
    raw = 2 * case["kv"] * case["page"] * case["hd"] + 8 * case["kv"] * (case["page"] // 16)
    return _ceil(raw, 128) * 128


def _lengths(case):
    """Rows and keys of each sequence of an attend case, the same for every seed: the longest has the case's sizes."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    new = [case["new"]] + [max(1, int(case["new"] * rng.uniform(0.1, 1))) for _ in range(case["seqs"] - 1)]
    return new, [m + int(case["behind"] * (rng.uniform(0, 1) if i else 1)) for i, m in enumerate(new)]


def _plan(case):
    """Host-side sizes of a reorder case, the same for every seed: each prompt's beams share its whole pages and hold what
    was generated since; `parent` names the sequence that each one continues."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    beams, page = case["beams"], case["page"]
    tokens = [case["tokens"]] + [max(1, int(case["tokens"] * rng.uniform(0.2, 1))) for _ in range(case["prompts"] - 1)]
    shared = [int(t * 0.85) // page for t in tokens]
    lens = [t for t in tokens for _ in range(beams)]
    n = len(lens)
    table, taken, refs = [[] for _ in range(n)], 0, []
    for p, t in enumerate(tokens):
        first = list(range(taken, taken + shared[p]))
        taken += shared[p]
        refs += [beams] * shared[p]
        for b in range(beams):
            rest = _ceil(t, page) - shared[p]
            table[p * beams + b] = first + list(range(taken, taken + rest))
            taken += rest
            refs += [1] * rest
    # as beam search has them: a few beams continued several times, others by nothing
    parent = [p * beams + b for p in range(len(tokens)) for b in sorted(rng.choices(range(beams), k=beams))]
    return {"lens": lens, "table": table, "refs": refs, "n_pages": taken + 2 * n, "parent": parent}


def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "norm":
        each = size * (4 if case["residual"] else 2) if case["form"] == "rows" else (
            size * (3 if case["residual"] else 1) + 1 + 4 / BLOCK)
        return {"bytes": case["tokens"] * case["width"] * each + 4 * case["width"],
                "flops": 6 * case["tokens"] * case["width"]}
    if case["kind"] == "rope":
        heads = case["heads"] + case["kv"]
        return {"bytes": case["tokens"] * (2 * size * heads * case["hd"] + 4) + 4 * case["rot"],
                "flops": 3 * case["tokens"] * heads * case["rot"]}
    if case["kind"] == "attend":
        new, keys = _lengths(case)
        seen = sum(m * (l - m) + m * (m + 1) // 2 if case["causal"] else m * l for m, l in zip(new, keys))
        return {"bytes": 2 * size * case["hd"] * (sum(new) * case["heads"] + sum(keys) * case["kv"]),
                "flops": 4 * case["hd"] * case["heads"] * seen}
    if case["kind"] == "beam":
        rows = case["prompts"] * case["beams"]
        return {"bytes": rows * (size * case["vocab"] + 4) + 12 * case["prompts"] * case["k"],
                "flops": 4 * rows * case["vocab"]}
    p, page = _plan(case), case["page"]
    old, new = sum(len(r) for r in p["table"]), sum(len(p["table"][s]) for s in p["parent"])
    # a partly filled last page that several beams continue: all of them but one get a copy
    copies = sum(p["parent"].count(s) - 1 for s in set(p["parent"]) if p["lens"][s] % page)
    return {"bytes": 4 * (old + 2 * new) + 8 * p["n_pages"] + 2 * copies * case["layers"] * _page_bytes(case), "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _gen(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_norm(case, seed):
    gen, dtype, shape = _gen(seed), _dtype(case), (case["tokens"], case["width"])
    # a residual stream with a few channels much wider than the others, and a block's smaller output
    x = torch.randn(shape, generator=gen, device=DEVICE)
    x *= 1.0 + 20.0 * (torch.arange(case["width"], device=DEVICE) % 97 == 5)
    w = 1.0 + 0.3 * torch.randn(case["width"], generator=gen, device=DEVICE)
    st = {"case": case, "w": w, "x": x.to(dtype), "residual": None}
    if case["residual"]:
        st["residual"], st["x"] = st["x"], (0.3 * torch.randn(shape, generator=gen, device=DEVICE)).to(dtype)
    return st


_THETA, _FACTOR, _CONTEXT, _LOW, _HIGH = 1e6, 4.0, 32768, 1.0, 32.0


def _magnitude(case):
    return 0.1 * math.log(_FACTOR) + 1.0 if case["scaling"] == "parts" else 1.0


def _turns(case):
    """Turns per position of each pair, on the host in 64 bits."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64)
    theta = _THETA
    if case["scaling"] == "base" and case["rot"] > 2:
        theta *= _FACTOR ** (case["rot"] / (case["rot"] - 2))
    f = theta ** (-2.0 * i / case["rot"]) / (2 * math.pi)
    if case["scaling"] == "linear":
        f = f / _FACTOR
    if case["scaling"] == "parts":
        keep = ((_CONTEXT * f - _LOW) / (_HIGH - _LOW)).clamp(0, 1)
        f = f * (keep + (1 - keep) / _FACTOR)
    return f


def _rope_inputs(case, seed):
    gen, n = _gen(seed), case["tokens"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    # one row of queries, keys and values, as a fused projection leaves it
    row = torch.randn(n, (heads + 2 * kv) * hd, generator=gen, device=DEVICE).to(_dtype(case))
    # a few prompts' tokens, each a run of positions somewhere in its context
    run = max(1, n // 5)
    first = torch.randint(0, max(1, case["last"] - run), (_ceil(n, run),), generator=gen, device=DEVICE)
    pos = (first.view(-1, 1) + torch.arange(run, device=DEVICE)).view(-1)[:n].to(torch.int32)
    q = row[:, :heads * hd].view(n, heads, hd)
    k = row[:, heads * hd:(heads + kv) * hd].view(n, kv, hd)
    return q, k, pos


def _prepare_rope(case, seed):
    q, k, pos = _rope_inputs(case, seed)
    st = {"case": case, "q": q, "k": k, "pos": pos}
    if own:
        scaling = None if case["scaling"] == "none" else case["scaling"]
        st["rope"] = _package().Rope(case["hd"], rot_dim=case["rot"], interleaved=case["interleaved"], theta=_THETA,
                                     scaling=scaling, factor=_FACTOR, context=_CONTEXT, low=_LOW, high=_HIGH,
                                     magnitude=_magnitude(case), device=DEVICE)
    else:
        st["turns"] = _turns(case).to(DEVICE)
    return st


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _attend_inputs(case, seed):
    gen, (new, keys) = _gen(seed), _lengths(case)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    q = torch.randn(sum(new), heads, hd, generator=gen, device=DEVICE)
    # keys with a few channels wider than the others, as rotated keys have; keys and values side by side in one row
    row = torch.randn(sum(keys), 2 * kv, hd, generator=gen, device=DEVICE)
    row[:, :kv] *= 1.0 + 3.0 * (torch.arange(hd, device=DEVICE) % 16 == 3)
    row = row.to(_dtype(case))
    return q.to(_dtype(case)), row[:, :kv], row[:, kv:]


def _prepare_attend(case, seed):
    new, keys = _lengths(case)
    q, k, v = _attend_inputs(case, seed)
    return {"case": case, "q": q, "k": k, "v": v, "start": _ints(_starts(new)), "longest": max(new), "most": max(keys),
            "kstart": _ints(_starts(keys)) if case["behind"] else None}


def _prepare_beam(case, seed):
    gen, rows = _gen(seed), case["prompts"] * case["beams"]
    # logits as a model's head gives them: a wide bulk, and a few ids well above it
    logits = 2.0 * torch.randn(rows, case["vocab"], generator=gen, device=DEVICE)
    top = torch.randint(0, case["vocab"], (rows, 6), generator=gen, device=DEVICE)
    logits.scatter_add_(1, top, 4.0 + 3.0 * torch.randn(rows, 6, generator=gen, device=DEVICE))
    scores = -20.0 * torch.rand(rows, generator=gen, device=DEVICE) - 5.0
    return {"case": case, "logits": logits.to(_dtype(case)), "scores": scores}


def _prepare_reorder(case, seed):
    gen, p = _gen(seed), _plan(case)
    n, n_pages = len(p["lens"]), p["n_pages"]
    width = _ceil(max(p["lens"]) + 1, case["page"])
    # which page each number of the plan is: pools hand them out in any order
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    plan = torch.full((n, width), -1, dtype=torch.int64)
    for s, row in enumerate(p["table"]):
        plan[s, :len(row)] = torch.tensor(row)
    plan = plan.to(DEVICE)
    table = torch.where(plan >= 0, order[plan.clamp(min=0)], -1).to(torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEVICE)
    refs[order[:len(p["refs"])].long()] = _ints(p["refs"])
    pages = torch.randint(0, 256, (case["layers"], n_pages, _page_bytes(case)), generator=gen, device=DEVICE,
                          dtype=torch.uint8)
    st = {"case": case, "first": [table, _ints(p["lens"]), refs], "src": _ints(p["parent"]), "dst": _ints(list(range(n))),
          "grown": _ints([p["lens"][s] + 1 for s in p["parent"]])}
    if own:
        cache = _package().KV8Cache(case["layers"], n_pages, case["page"], case["kv"], case["hd"], n, width, device=DEVICE)
        cache.pages.copy_(pages)
        st["cache"], st["pages"] = cache, cache.pages
        st["held"] = [cache.table, cache.lens, cache.refs]
    else:
        st["held"], st["pages"] = [torch.empty_like(t) for t in st["first"]], pages
    return st


def prepare(case, seed):
    return {"norm": _prepare_norm, "rope": _prepare_rope, "attend": _prepare_attend, "beam": _prepare_beam,
            "reorder": _prepare_reorder}[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if kind == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    if kind == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if kind == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if kind == "beam":
        return _own_beam(state) if own else _plain_beam(state)
    # the state before, so that every pass has the same beams to reorder
    torch._foreach_copy_(state["held"], state["first"])
    if own:
        _own_reorder(state)
    else:
        _plain_reorder(state)
    table, lens, refs = state["held"]
    return {"table": table, "lens": lens, "refs": refs, "pages": state["pages"]}


def _values(q, d):
    """What 8-bit codes stand for."""
    return (q.view(*d.shape, BLOCK) * d.unsqueeze(-1)).view(q.shape)


def _own_norm(st):
    qh, residual = _package(), st["residual"]
    if st["case"]["form"] == "rows":
        return qh.rmsnorm(st["x"], st["w"], EPS, residual=residual)
    got = qh.rmsnorm_q8(st["x"], st["w"], EPS, residual=residual)
    return (*got[:-2], _values(*got[-2:]))


def _own_rope(st):
    return st["rope"](st["q"], st["k"], pos=st["pos"])


def _own_attend(st):
    return _package().attention(st["q"], st["k"], st["v"], st["start"], kstart=st["kstart"], causal=st["case"]["causal"])


def _own_beam(st):
    return _package().beam_select(st["logits"], st["scores"], st["case"]["beams"], st["case"]["k"])


def _own_reorder(st):
    st["cache"].reorder(st["src"], st["dst"])
    st["cache"].resize(st["dst"], st["grown"])


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_norm(st):
    x, residual = st["x"], st["residual"]
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    # the row in 64 bits: a result next to a border between two codes keeps its side
    wide = h.double()
    scale = 1.0 / torch.sqrt((wide * wide).sum(-1, keepdim=True) / wide.shape[-1] + EPS)
    y = (wide * scale * st["w"].double()).float()
    if st["case"]["form"] == "rows":
        out = (y.to(x.dtype),)
    else:
        blocks = y.view(y.shape[0], -1, BLOCK)
        top = blocks.abs().amax(-1)
        d = top / torch.full_like(top, 127.0)
        inverse = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
        t = blocks * inverse.unsqueeze(-1)
        whole = torch.trunc(t)
        code = whole + torch.where((t - whole).abs() >= 0.5, torch.sign(t), torch.zeros_like(t))
        out = (_values(code.to(torch.int8).view(y.shape), d),)
    return out[0] if residual is None and st["case"]["form"] == "rows" else out if residual is None else (h, *out)


def _plain_rope(st):
    case = st["case"]
    angle = st["pos"].double().view(-1, 1) * st["turns"]  # in turns; far positions need the 64 bits
    angle = (angle - torch.round(angle)) * (2 * math.pi)
    m = _magnitude(case)
    c, s = (m * torch.cos(angle)).float().unsqueeze(1), (m * torch.sin(angle)).float().unsqueeze(1)
    return tuple(_plain_turn(t, c, s, case["rot"], case["interleaved"]) for t in (st["q"], st["k"]))


def _plain_turn(x, c, s, rot, interleaved):
    wide = x.float()
    if interleaved:
        a, b = wide[..., 0:rot:2], wide[..., 1:rot:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = wide[..., :rot // 2], wide[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((turned, wide[..., rot:]), dim=-1).to(x.dtype)


def _padded(x, start, length):
    """Packed rows as [sequences][heads][length][head_dim] in 32 bits, and which of them are there."""
    place = start[:-1].long().view(-1, 1) + torch.arange(length, device=DEVICE)
    there = place < start[1:].long().view(-1, 1)
    return x[place.clamp(max=x.shape[0] - 1)].float().transpose(1, 2).contiguous(), there


def _plain_attend(st):
    case, start = st["case"], st["start"]
    kstart = start if st["kstart"] is None else st["kstart"]
    q, rows = _padded(st["q"], start, st["longest"])
    k, cols = _padded(st["k"], kstart, st["most"])
    v, _ = _padded(st["v"], kstart, st["most"])
    n, kv, most, hd = k.shape
    q = q.view(n * kv, -1, hd)
    scores = torch.matmul(q, k.view(n * kv, most, hd).transpose(1, 2).contiguous()).view(n, kv, -1, st["longest"], most)
    hidden = ~cols.view(n, 1, most)
    if case["causal"]:
        # a sequence's rows are its last ones
        at = torch.arange(st["longest"], device=DEVICE) + (cols.sum(1) - rows.sum(1)).view(n, 1)
        hidden = hidden | (torch.arange(most, device=DEVICE) > at.unsqueeze(-1))
    scores = (scores * (1.0 / math.sqrt(hd))).masked_fill_(hidden.view(n, 1, 1, -1, most), -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(n * kv, -1, most), v.view(n * kv, most, hd)).view(n, -1, st["longest"], hd)
    return out.transpose(1, 2)[rows].to(st["q"].dtype)


def _plain_beam(st):
    case = st["case"]
    wide = st["logits"].double()  # candidates of different beams meet in the order of their sums
    top = wide.amax(-1, keepdim=True)
    total = torch.log(torch.exp(wide - top).sum(-1, keepdim=True)) + top
    each = (wide + st["scores"].double().view(-1, 1) - total).view(case["prompts"], -1)
    best, at = torch.sort(each, dim=-1, descending=True, stable=True)  # equal ones in the order of their places
    best, at = best[:, :case["k"]], at[:, :case["k"]]
    first = case["beams"] * torch.arange(case["prompts"], device=DEVICE).view(-1, 1)
    parent = torch.div(at, case["vocab"], rounding_mode="floor")
    return (first + parent).to(torch.int32), (at - parent * case["vocab"]).to(torch.int32), best.float()


def _add_refs(refs, rows, by):
    """`by` more for each page in rows (-1: none)."""
    held = rows.reshape(-1).long()
    refs.index_add_(0, held.clamp(min=0), by * (held >= 0).to(torch.int32))


def _plain_reorder(st):
    table, lens, refs = st["held"]
    page, src, dst = st["case"]["page"], st["src"].long(), st["dst"].long()
    rows, before = table[src], lens[src]
    _add_refs(refs, table[dst], -1)
    _add_refs(refs, rows, 1)
    # room for the next token: a new page where the last is full, a copy of it where others hold it too
    column = torch.arange(table.shape[1], device=DEVICE)
    have, want = (before + page - 1) // page, (st["grown"] + page - 1) // page
    last = (have - 1).clamp(min=0).long().view(-1, 1)
    old = rows.gather(1, last).view(-1)
    split = (before % page != 0) & (refs[old.long().clamp(min=0)] > 1)
    needs = ((column >= have.view(-1, 1)) & (column < want.view(-1, 1))) | (split.view(-1, 1) & (column == last))
    where = torch.nonzero(needs)
    taken = torch.nonzero(refs == 0).view(-1)[:where.shape[0]]
    _add_refs(refs, torch.where(split, old, -1), -1)
    rows[where[:, 0], where[:, 1]] = taken.to(torch.int32)
    refs[taken] = 1
    table[dst], lens[dst] = rows, st["grown"]
    who = torch.nonzero(split).view(-1)
    st["pages"][:, rows[who, last.view(-1)[who]].long()] = st["pages"][:, old[who].long()]


# ------------------------------------------------------------------------------------------------ from the definition

def _exact_norm(case, seed):
    st = _prepare_norm(case, seed)
    h = st["x"].double()
    if st["residual"] is not None:
        h = h + st["residual"].double()
    kept = h.to(_dtype(case)).double()  # what the norm sees is what the sum holds
    y = st["w"].double() * kept * torch.rsqrt(kept.square().mean(dim=1, keepdim=True) + EPS)
    if case["form"] == "q8":
        rows = y.to(torch.float32).reshape(-1, BLOCK)
        d = rows.double().abs().max(dim=1, keepdim=True).values.div(127.0 * torch.ones(1, 1, dtype=torch.float64,
                                                                                       device=DEVICE)).float()
        per = torch.where(d > 0, torch.ones_like(d) / d, d)
        code = (rows * per).double()
        code = torch.copysign(torch.floor(code.abs() + 0.5), code)
        y = (code * d.double()).view(h.shape)
    if st["residual"] is None:
        return y if case["form"] == "rows" else (y,)
    return h, y


def _exact_rope(case, seed):
    q, k, pos = _rope_inputs(case, seed)
    rot, half = case["rot"], case["rot"] // 2
    out = [q.double().clone(), k.double().clone()]
    for i in range(half):
        base = _THETA
        if case["scaling"] == "base" and rot > 2:
            base = _THETA * math.pow(_FACTOR, rot / (rot - 2))
        rate = math.pow(base, -2 * i / rot)
        if case["scaling"] == "linear":
            rate /= _FACTOR
        elif case["scaling"] == "parts":
            share = (_CONTEXT * rate / math.tau - _LOW) / (_HIGH - _LOW)
            share = min(1.0, max(0.0, share))
            rate = share * rate + (1.0 - share) * rate / _FACTOR
        z = torch.polar(torch.full_like(pos, 1, dtype=torch.float64) * _magnitude(case), pos.double() * rate).view(-1, 1)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        for t in out:
            turned = torch.complex(t[..., first].contiguous(), t[..., second].contiguous()) * z
            t[..., first], t[..., second] = turned.real, turned.imag
    return tuple(out)


def _exact_attend(case, seed):
    q, k, v = _attend_inputs(case, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group, a, b = case["heads"] // case["kv"], 0, 0
    for m, l in zip(*_lengths(case)):
        limit = torch.arange(l - m, l, device=q.device).unsqueeze(1)
        for h in range(case["heads"]):
            s = q[a:a + m, h].double() @ k[b:b + l, h // group].double().t().contiguous() / case["hd"] ** 0.5
            if case["causal"]:
                s = torch.where(torch.arange(l, device=q.device) <= limit, s, -math.inf)
            out[a:a + m, h] = torch.softmax(s, dim=1) @ v[b:b + l, h // group].double()
        a, b = a + m, b + l
    return out


def _exact_beam(case, seed):
    st = _prepare_beam(case, seed)
    logp = torch.log_softmax(st["logits"].double(), dim=-1) + st["scores"].double().unsqueeze(1)
    best = torch.topk(logp.reshape(case["prompts"], -1), case["k"], dim=-1).values
    return None, None, best


def exact(case, seed):
    if case["kind"] == "reorder":
        return None  # whole numbers only
    return {"norm": _exact_norm, "rope": _exact_rope, "attend": _exact_attend, "beam": _exact_beam}[case["kind"]](case, seed)
