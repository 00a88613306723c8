"""The decoder over a bound 8-bit paged cache (qh_decoder_bind_kv8).

The first layer's keys and values depend on the token ids alone, so the cache's layer 0 is checked bit for bit: the f32
cache of the plain decoder, put through the plain model of the 8-bit cache in the same stretches. What later layers and
the logits may differ by is not bounded tightly (each rounding to 8 bits feeds every later quantization); there the final
hidden state has to agree with the f32 cache's within what 8-bit rounding amounts to, and everything that must not depend
on where tokens lie (forks, copies, page sizes, graphs) has to give equal bits."""
import numpy as np
import pytest

from conftest import bits
from decoder_util import qnt_module
from kv8_util import PlainKV8

pytestmark = pytest.mark.gpu


def model(seed=3, **kw):
    qnt = qnt_module()
    args = dict(vocab_size=2048, n_layers=2)
    args.update(kw)
    hp = qnt.HParams(**args)
    return hp, qnt.synthetic_q4mix(seed, hp)


NARROW = dict(vocab_size=1024, dim=256, n_heads=4, n_kv_heads=1, head_dim=64, ffn_dim=512)
WIDE = dict(vocab_size=1024, dim=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn_dim=512)

MANY = dict(vocab_size=1024, dim=2560, n_heads=40, n_kv_heads=1, head_dim=64, ffn_dim=512)


def cache_for(qh, hp, n_pages=40, page=32, seqs=4, seq_pages=10):
    c = qh.KV8Cache(hp.n_layers, n_pages, page, hp.n_kv_heads, hp.head_dim, seqs, seq_pages)
    c.pages.fill_(0x7f)
    return c


def ints(x):
    import torch
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def stored(cache, layer, seq, n):
    k, v = cache.read(layer, n, start=ints([0, n]), seqs=ints([seq]))
    return k.cpu().numpy(), v.cpu().numpy()


@pytest.mark.parametrize("stack", [32, 96])
@pytest.mark.parametrize("shape", [NARROW, WIDE])
def test_first_layer_bit_for_bit(qh, gpu, shape, stack):
    hp, tens = model(**shape)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp)
    dec.set_prefill_stack(stack)
    dec.bind_kv8(cache, 2)
    rng = np.random.default_rng(1)
    ids = rng.integers(0, hp.vocab_size, 75).astype(np.int32)
    dec.prefill(ids, 0)
    dec.begin(20)
    for _ in range(7):
        dec.step()
    more = rng.integers(0, hp.vocab_size, 33).astype(np.int32)
    dec.prefill(more, 82)
    assert dec.status() == 0 and int(cache.status) == 0 and int(cache.lens[2]) == 115
    tokens = np.concatenate([ids, dec.outputs(7), more])
    plain = PlainKV8(1, 40, 32, hp.n_kv_heads, hp.head_dim, 4, 10)
    ref = qh.Decoder(hp, tens, ctx_len=256, kv_f32=True)
    ref.prefill(tokens, 0)
    k, v = (x.reshape(-1, hp.n_kv_heads, hp.head_dim) for x in ref.kv(0, 115))
    at = 0
    stretches = [min(stack, 75 - i) for i in range(0, 75, stack)] + [1] * 7 + [min(stack, 33 - i) for i in range(0, 33, stack)]
    for m in stretches:
        plain.resize([2], [at + m])
        plain.append(0, [2], [m], k[at:at + m], v[at:at + m])
        at += m
    for got, want in zip(stored(cache, 0, 2, 115), plain.values(0, 2)):
        assert (got == want).all()  # a code of 0 has no sign
    dec.close()
    ref.close()


@pytest.mark.parametrize("shape,dtype", [(NARROW, None), (WIDE, None), (NARROW, 1), ({}, None)])
def test_hidden_states_agree_with_the_f32_cache(qh, gpu, shape, dtype):
    """A code is off by at most 1/254 of its block's largest value, about 1/80 of the block's root mean square for the
    values here (their largest is some three times that): keys, values and, behind them, every later 8-bit activation
    each carry about as much, and two layers add up to a few per cent. A wrong head, position, bias or page would be of
    the order of the state itself."""
    qnt = qnt_module()
    args = dict(vocab_size=2048, n_layers=2)
    args.update(shape)
    hp = qnt.HParams(**args)
    tens = qnt.synthetic_q4mix(5, hp) if dtype is None else qnt.synthetic_dense(5, hp, dtype)
    dec, ref = qh.Decoder(hp, tens, ctx_len=256), qh.Decoder(hp, tens, ctx_len=256, kv_f32=True)
    cache = cache_for(qh, hp, page=16, seq_pages=16)
    dec.bind_kv8(cache, 1)
    k = 1 if dtype is None else 0
    ids = np.random.default_rng(2).integers(0, hp.vocab_size, 130).astype(np.int32)
    at = 0
    for m in (70, 1, 1, 40, 1, 17):
        for d in (dec, ref):
            d.prefill(ids[at:at + m], at, top_k=k)
        at += m
        a, b = dec.hidden().astype(np.float64), ref.hidden().astype(np.float64)
        assert np.linalg.norm(a - b) <= 0.15 * np.linalg.norm(b), (at, np.linalg.norm(a - b) / np.linalg.norm(b))
    assert dec.status() == 0
    dec.close()
    ref.close()


@pytest.mark.parametrize("shape,pages", [(NARROW, 80), (WIDE, 80), (NARROW, 130), (MANY, 8), (MANY, 130)])
def test_steps_agree_over_every_attention_kernel(qh, gpu, shape, pages):
    """Tables of more than 1,024 and 2,048 positions, where a step's attention is joined from shares, and more query heads
    to a KV head than its kernels take: the 8-bit outputs come from another place each. Bounds as above."""
    hp, tens = model(5, **shape)
    dec, ref = qh.Decoder(hp, tens, ctx_len=256), qh.Decoder(hp, tens, ctx_len=256, kv_f32=True)
    dec.bind_kv8(cache_for(qh, hp, page=16, seq_pages=pages), 1)
    ids = np.random.default_rng(2).integers(0, hp.vocab_size, 120).astype(np.int32)
    at = 0
    for m in (100, 1, 1, 1):
        for d in (dec, ref):
            d.prefill(ids[at:at + m], at)
        at += m
        a, b = dec.hidden().astype(np.float64), ref.hidden().astype(np.float64)
        assert np.linalg.norm(a - b) <= 0.15 * np.linalg.norm(b), (at, np.linalg.norm(a - b) / np.linalg.norm(b))
    assert dec.status() == 0
    dec.close()
    ref.close()


def continue_from(dec, cache, seq, ids, steps=6):
    dec.bind_kv8(cache, seq)
    dec.prefill(ids[-1:], len(ids) - 1)
    first = dec.hidden()
    dec.begin(steps + 1)
    for _ in range(steps):
        dec.step()
    return dec.outputs(steps + 1).tolist(), first, dec.hidden()


@pytest.mark.parametrize("copy", [False, True])
def test_replies_from_forks(qh, gpu, copy):
    """A prompt read once; continuations of shared and copied forks equal the continuation of the prompt's own sequence,
    and none changes what the others hold."""
    hp, tens = model(**NARROW)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp)
    ids = np.random.default_rng(3).integers(0, hp.vocab_size, 77).astype(np.int32)
    dec.bind_kv8(cache, 0)
    dec.prefill(ids, 0)
    cache.fork(ints([0, 0]), ints([1, 3]), copy=copy)
    before = [stored(cache, l, 0, 77) for l in range(2)]
    results = [continue_from(dec, cache, s, ids) for s in (1, 3)]
    for l in range(2):
        for got, want in zip(stored(cache, l, 0, 77), before[l]):
            assert (bits(got) == bits(want)).all()
    results.append(continue_from(dec, cache, 0, ids))
    for tokens, first, last in results[1:]:
        assert tokens == results[0][0]
        assert (bits(first) == bits(results[0][1])).all() and (bits(last) == bits(results[0][2])).all()
    assert dec.status() == 0 and int(cache.status) == 0 and cache.lens.tolist() == [83, 83, 0, 83]
    # after the pages have moved, still the same
    cache.resize(ints([0]), ints([0]))
    cache.compact()
    assert continue_from(dec, cache, 3, ids)[0] == results[0][0]
    dec.close()


def test_a_captured_step_follows_the_bound_sequence(qh, gpu):
    import torch
    hp, tens = model(**NARROW)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, hp.vocab_size, n).astype(np.int32) for n in (40, 66)]
    want = []
    for s, ids in enumerate(prompts):
        dec.bind_kv8(cache, s)
        dec.prefill(ids, 0)
        dec.begin(12)
        for _ in range(11):
            dec.step()
        want.append((dec.outputs(12).tolist(), [stored(cache, l, s, len(ids) + 11) for l in range(2)]))
    cache.reset()
    dec.bind_kv8(cache, 0)
    dec.prefill(prompts[0], 0)
    dec.begin(12)
    dec.step()  # outside the graph first
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        dec.step()
    for _ in range(10):
        g.replay()
        torch.ones(100, device="cuda").sum().item()
    assert dec.outputs(12).tolist() == want[0][0] and dec.status() == 0
    dec.bind_kv8(cache, 1)
    dec.prefill(prompts[1], 0)
    dec.begin(12)
    for _ in range(11):
        g.replay()
    assert dec.outputs(12).tolist() == want[1][0] and dec.status() == 0
    for s, ids in enumerate(prompts):
        for l in range(2):
            for a, b in zip(stored(cache, l, s, len(ids) + 11), want[s][1][l]):
                assert (bits(a) == bits(b)).all()
    dec.close()


def test_no_place_is_reported_and_harms_nothing(qh, gpu):
    hp, tens = model(**NARROW)
    dec = qh.Decoder(hp, tens, ctx_len=128)
    cache = cache_for(qh, hp, n_pages=4, page=16, seqs=3, seq_pages=8)
    ids = np.random.default_rng(5).integers(0, hp.vocab_size, 100).astype(np.int32)
    dec.bind_kv8(cache, 0)
    dec.prefill(ids[:30], 0)
    dec.bind_kv8(cache, 1)
    dec.prefill(ids[:20], 0)
    assert dec.status() == 0
    kept = stored(cache, 0, 0, 30)
    dec.begin(20)
    for _ in range(12):
        dec.step()  # fills the second page
    assert dec.status() == 0 and cache.lens.tolist() == [30, 32, 0]
    dec.step()
    assert dec.status() == 4 and int(cache.status) == qh.KV8_NO_PAGES and cache.lens.tolist() == [30, 32, 0]
    # a step at another position than the sequence's end, a prompt behind it, one past the table row
    cache.status.zero_()
    dec.bind_kv8(cache, 0)
    dec.step()
    assert dec.status() & 4 and cache.lens.tolist() == [30, 32, 0]
    dec.prefill(ids[:3], 31)
    assert dec.status() == 4 and cache.lens.tolist() == [30, 32, 0]
    assert int(cache.status) == 0
    for a, b in zip(stored(cache, 0, 0, 30), kept):
        assert (bits(a) == bits(b)).all()
    # and the decoder's own cache again, as it was never used: from the start
    dec.bind_kv8(None)
    ref = qh.Decoder(hp, tens, ctx_len=128)
    for d in (dec, ref):
        d.prefill(ids[:40], 0)
    assert (bits(dec.hidden()) == bits(ref.hidden())).all() and dec.status() == 0
    # the context's end
    big = cache_for(qh, hp, n_pages=20, page=16, seqs=1, seq_pages=12)
    dec.bind_kv8(big, 0)
    dec.prefill(np.resize(ids, 127), 0)
    dec.begin(4)
    dec.step()
    assert dec.status() == 0 and int(big.lens[0]) == 128
    dec.step()
    assert dec.status() == 1 and int(big.lens[0]) == 128
    dec.close()
    ref.close()


def test_bind_refusals(qh, gpu):
    hp, tens = model(**NARROW)
    dec = qh.Decoder(hp, tens, ctx_len=128)
    good = cache_for(qh, hp)
    for bad, seq in ((good, 4), (good, -1), (qh.KV8Cache(3, 4, 16, 1, 64, 1, 4), 0), (qh.KV8Cache(2, 4, 16, 2, 64, 1, 4), 0),
                     (qh.KV8Cache(2, 4, 16, 1, 128, 1, 4), 0)):
        with pytest.raises(qh.QHError):
            dec.bind_kv8(bad, seq)
    assert qh.lib().qh_decoder_bind_kv8(None, good._ref, 0) == qh.ERR_ARG
    ids = np.arange(40, dtype=np.int32)
    for after in range(3):  # each of its allocations fails once: the decoder stays on its own cache
        assert qh.lib().qh_fault_alloc(after) == 0
        assert qh.lib().qh_decoder_bind_kv8(dec.h, good._ref, 0) == qh.ERR_NOMEM
    dec.prefill(ids, 0)
    assert int(good.lens[0]) == 0
    dec.bind_kv8(good, 0)
    dec.prefill(ids, 0)
    assert int(good.lens[0]) == 40 and dec.status() == 0
    dec.close()
