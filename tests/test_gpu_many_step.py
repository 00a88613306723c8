"""The operators of a step of many sequences together, as a serving loop uses them: prompts read packed (norm into 8-bit blocks,
quantized projections, rotary positions, attention over their own keys and values, the 8-bit cache's store), then beam search over
the cache (the same with the cache's attention, the selection, the reordering and the room for the next token). Every result of
the new operators is checked on the inputs that it meets there, and a captured step against eager ones."""
import math

import numpy as np
import pytest
import torch

from test_gpu_beam import plain_select
from test_gpu_prompt import check as check_attention, formula as attention_formula, ints, starts
from test_gpu_rows import check_rope, check_rounded, norm_formula

pytestmark = pytest.mark.gpu

DIM, HEADS, KV, HD, FFN, LAYERS, VOCAB, PAGE = 256, 4, 2, 64, 512, 2, 1500, 16
BEAMS = 4


class Model:
    """Two layers of quantized matrices with random weights, over the package's operators."""

    def __init__(self, qh, synth, dev):
        self.qh, self.dev = qh, dev
        rng = np.random.default_rng(3)
        q8 = lambda seed, r, c: qh.DeviceTensor.upload(synth.q8_tensor(seed, r, c), qh.Q8_0, r, c, device=dev)  # noqa: E731
        self.embed = torch.from_numpy(rng.standard_normal((VOCAB, DIM)).astype(np.float32)).to(dev)
        norm = lambda: torch.from_numpy((1 + 0.2 * rng.standard_normal(DIM)).astype(np.float32)).to(dev)  # noqa: E731
        self.layers = [dict(n1=norm(), n2=norm(), qkv=q8(10 * l + 1, (HEADS + 2 * KV) * HD, DIM), o=q8(10 * l + 2, DIM, DIM),
                            gate=q8(10 * l + 3, FFN, DIM), up=q8(10 * l + 4, FFN, DIM), down=q8(10 * l + 5, DIM, FFN))
                       for l in range(LAYERS)]
        self.norm, self.head = norm(), q8(99, VOCAB, DIM)
        self.rope = qh.Rope(HD, rot_dim=48, theta=1e4, device=dev)
        self.check = False

    def normed(self, x, w, res):
        got = self.qh.rmsnorm_q8(x, w, 1e-6, residual=res)
        h = x if res is None else got[0]
        if self.check:
            assert res is None or torch.equal(h, x + res)
            y = self.qh.rmsnorm(h, w, 1e-6)
            check_rounded(y, norm_formula(h, w, 1e-6), torch.float32)
            q, d = self.qh.quantize_q8(y)
            assert torch.equal(q, got[-2]) and torch.equal(d, got[-1])
        return h, got[-2], got[-1]

    def layers_of(self, x, pos, attend):
        """Every layer over rows x at positions pos; attend(l, q, k, v) -> rows."""
        qh, delta = self.qh, None
        for l, w in enumerate(self.layers):
            x, q8, d8 = self.normed(x, w["n1"], delta) if delta is None else self.normed(delta, w["n1"], x)
            row = qh.matmul_q(w["qkv"], q8, d8)
            n = row.shape[0]
            q, k, v = (t.view(n, -1, HD) for t in row.split([HEADS * HD, KV * HD, KV * HD], dim=1))
            q0, k0 = q.clone(), k.clone()
            qh_q, qh_k = self.rope(q, k, pos=pos, q_out=q, k_out=k)  # in place, in the projection's rows
            if self.check:
                check_rope(qh_q, q0, pos, self.rope.turns, 48, False)
                check_rope(qh_k, k0, pos, self.rope.turns, 48, False)
            a = attend(l, q, k, v).reshape(n, HEADS * HD)
            delta = qh.matmul_q(w["o"], *qh.quantize_q8(a))
            x, q8, d8 = self.normed(delta, w["n2"], x)
            g, u = qh.matmul_q(w["gate"], q8, d8), qh.matmul_q(w["up"], q8, d8)
            delta = qh.matmul_q(w["down"], *qh.quantize_q8(torch.nn.functional.silu(g) * u))
        return delta, x

    def logits(self, delta, x):
        _, q8, d8 = self.normed(delta, self.norm, x)
        return self.qh.matmul_q(self.head, q8, d8) * 0.05


def new_cache(qh, dev, n_seqs):
    return qh.KV8Cache(LAYERS, 40 * n_seqs, PAGE, KV, HD, n_seqs, 16, device=dev)


def read_prompts(model, cache, prompts):
    """The prompts into sequences 0, BEAMS, 2 BEAMS ..; the logits behind their last tokens."""
    qh, dev = model.qh, model.dev
    lens = [len(p) for p in prompts]
    st = starts(lens)
    start = ints(st, dev)
    seqs = ints([BEAMS * i for i in range(len(prompts))], dev)
    cache.resize(seqs, ints(lens, dev))
    x = model.embed[torch.cat([torch.as_tensor(p, device=dev) for p in prompts])]
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in lens])

    def attend(l, q, k, v):
        cache.append(l, k, v, start=start, seqs=seqs)
        out = qh.attention(q, k, v, start)
        if model.check:
            check_attention(out, *attention_formula(q, k, v, st, st, True, HD ** -0.5))
        return out

    delta, x = model.layers_of(x, pos, attend)
    last = ints([s - 1 for s in st[1:]], dev).long()
    return model.logits(delta[last], x[last])


def step(model, cache, tokens):
    """One token of every sequence (room for it is there) -> logits."""
    pos = cache.lens - 1

    def attend(l, q, k, v):
        cache.append(l, k, v)
        return cache.attention(l, q)

    return model.logits(*model.layers_of(model.embed[tokens.long()], pos, attend))


def select(model, logits, scores, beams):
    got = model.qh.beam_select(logits, scores, beams, BEAMS)
    if model.check:
        want = plain_select(logits, scores, beams, BEAMS, logits.shape[1])
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
        assert np.allclose(got[2].cpu().numpy(), want[2], rtol=2.0 ** -24, atol=1e-11)
    return got


def contents(cache, s):
    n = int(cache.lens[s])
    return [torch.stack(cache.read(l, n, start=ints([0, n], cache.device), seqs=ints([s], cache.device))) for l in range(LAYERS)]


def test_beam_search_over_the_cache(qh, synth, gpu):
    model = Model(qh, synth, gpu)
    model.check = True
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, VOCAB, n) for n in (37, 5, 64)]
    n = BEAMS * len(prompts)
    cache = new_cache(qh, gpu, n)
    logits = read_prompts(model, cache, prompts)
    # the first choice: one row to a prompt, whose sequence the beams continue
    row, token, score = select(model, logits, None, 1)
    parent = (row * BEAMS).view(-1)
    taken = [[int(t)] for t in token.view(-1)]
    for turn in range(5):
        before = {int(s): contents(cache, int(s)) for s in set(parent.tolist())}
        lens = cache.lens[parent.long()] + 1
        cache.reorder(parent)
        cache.resize(torch.arange(n, dtype=torch.int32, device=gpu), lens)
        assert int(cache.status) == 0
        for s, p in enumerate(parent.tolist()):  # the parents' tokens, behind which there is room for one
            for got, want in zip(contents(cache, s), before[p]):
                assert torch.equal(got[:, :-1], want)
        logits = step(model, cache, token.view(-1))
        assert bool(torch.isfinite(logits).all())
        parent, token, score = select(model, logits, score.view(-1), BEAMS)
        parent = parent.view(-1)
        taken = [taken[p] + [int(t)] for p, t in zip(parent.tolist(), token.view(-1).tolist())]
        assert bool((score[:, :-1] >= score[:, 1:]).all())
    # sequences of different beams differ, and every prompt's beams stayed its own
    assert len({(i // BEAMS, tuple(t)) for i, t in enumerate(taken)}) == n
    assert all(p // BEAMS == i // BEAMS for i, p in enumerate(parent.tolist()))
    held = torch.zeros_like(cache.refs)
    held.index_add_(0, cache.table[cache.table >= 0].long(), torch.ones_like(cache.table[cache.table >= 0]))
    assert torch.equal(held, cache.refs)


def test_captured_beam_search(qh, synth, gpu):
    """A whole step in a graph, replayed: the same tokens, parents, scores and cache as eager steps from the same state."""
    model = Model(qh, synth, gpu)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, VOCAB, n) for n in (20, 33)]
    n = BEAMS * len(prompts)
    cache = new_cache(qh, gpu, n)
    row, token, score = select(model, read_prompts(model, cache, prompts), None, 1)
    state = dict(parent=(row * BEAMS).view(-1).contiguous(), token=token.view(-1).contiguous(), score=score.view(-1).contiguous())
    everyone = torch.arange(n, dtype=torch.int32, device=gpu)
    kept = [t.clone() for t in (cache.table, cache.lens, cache.refs, cache.pages, *state.values())]

    def one():
        lens = cache.lens[state["parent"].long()] + 1
        cache.reorder(state["parent"], everyone)
        cache.resize(everyone, lens)
        got = select(model, step(model, cache, state["token"]), state["score"], BEAMS)
        for name, t in zip(("parent", "token", "score"), got):
            state[name].copy_(t.reshape(-1))

    def run(f):
        out = []
        for t, v in zip((cache.table, cache.lens, cache.refs, cache.pages, *state.values()), kept):
            t.copy_(v)
        for _ in range(4):
            f()
            torch.cuda.synchronize()
            out.append([t.clone() for t in (*state.values(), cache.table, cache.lens, cache.refs)])
        return out

    eager = run(one)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for again in (run(graph.replay), run(one), run(graph.replay)):
        assert all(torch.equal(a, b) for x, y in zip(again, eager) for a, b in zip(x, y))
    assert int(cache.status) == 0 and not math.isnan(float(state["score"].sum()))
