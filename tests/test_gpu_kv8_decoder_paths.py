"""The decoder over a bound 8-bit cache on the paths that its other tests do not take: one launch per operation, the options of
the model, single tokens as prompts, timed steps, sampling; and its attention against the f32 cache's over the same values."""
import ctypes as C

import numpy as np
import pytest

from conftest import bits
from decoder_util import qnt_module
from test_gpu_kv8_decoder import NARROW, WIDE, cache_for, ints, model, stored

pytestmark = pytest.mark.gpu


def run(qh, hp, tens, n=70, steps=6, seq_pages=10, **kw):
    """Hidden states and the cache's values after a prompt and after steps, and the tokens."""
    dec = qh.Decoder(hp, tens, ctx_len=256, **kw)
    cache = cache_for(qh, hp, seq_pages=seq_pages, n_pages=seq_pages + 20)
    dec.bind_kv8(cache, 1)
    k = 1 if tens["model.embed_tokens.weight"].dtype == qh.Q8_0 else 0
    ids = np.random.default_rng(2).integers(0, hp.vocab_size, n).astype(np.int32)
    dec.prefill(ids, 0, top_k=k)
    out = [dec.hidden()]
    dec.begin(steps + 1, top_k=k)
    for _ in range(steps):
        dec.step(top_k=k)
    out += [dec.hidden()] + [x for l in range(hp.n_layers) for x in stored(cache, l, 1, n + steps)]
    tokens = dec.outputs(steps + 1).tolist()
    assert dec.status() == 0 and int(cache.status) == 0
    dec.close()
    return tokens, out


def equal(a, b):
    assert a[0] == b[0]
    for x, y in zip(a[1], b[1]):
        assert (bits(x) == bits(y)).all()


@pytest.mark.parametrize("seq_pages", [10, 80])
@pytest.mark.parametrize("shape,options", [(NARROW, {}), (WIDE, {}), (NARROW, dict(tied_embeddings=False, flags=1)),
                                           (WIDE, dict(flags=1))])
def test_one_launch_per_operation(qh, gpu, monkeypatch, shape, options, seq_pages):
    hp, tens = model(4, **shape, **options)
    fused = run(qh, hp, tens, seq_pages=seq_pages)
    monkeypatch.setenv("QH_DECODER_FUSE", "0")
    equal(fused, run(qh, hp, tens, seq_pages=seq_pages))


@pytest.mark.parametrize("shape", [NARROW, WIDE])
def test_the_decoders_own_cache_plays_no_part(qh, gpu, shape):
    hp, tens = model(4, **shape)
    equal(run(qh, hp, tens), run(qh, hp, tens, kv_f32=True))


@pytest.mark.parametrize("shape,dtype", [(NARROW, None), (WIDE, None), (NARROW, 0), (NARROW, 1)])
def test_a_prompt_of_one_token_is_a_step(qh, gpu, shape, dtype):
    qnt = qnt_module()
    hp = qnt.HParams(**dict(dict(vocab_size=2048, n_layers=2), **shape))
    tens = qnt.synthetic_q4mix(4, hp) if dtype is None else qnt.synthetic_dense(4, hp, dtype)
    k = 1 if dtype is None else 0
    tokens, want = run(qh, hp, tens, steps=4)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp, n_pages=30)
    dec.bind_kv8(cache, 1)
    ids = np.random.default_rng(2).integers(0, hp.vocab_size, 70).astype(np.int32)
    dec.prefill(ids, 0, top_k=k)
    for i, t in enumerate(tokens[:4]):
        dec.prefill(np.array([t], np.int32), 70 + i, top_k=k)
    got = [dec.hidden()] + [x for l in range(hp.n_layers) for x in stored(cache, l, 1, 74)]
    for x, y in zip(got, want[1:]):
        assert (bits(x) == bits(y)).all()
    dec.close()


@pytest.mark.parametrize("seq_pages,joins", [(10, 0), (80, 1)])
def test_a_timed_step(qh, gpu, seq_pages, joins):
    """The same step; the launches that make room count to the first layer's projections."""
    import torch
    hp, tens = model(4, **NARROW)
    tokens, want = run(qh, hp, tens, steps=1, seq_pages=seq_pages)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp, seq_pages=seq_pages, n_pages=seq_pages + 20)
    dec.bind_kv8(cache, 1)
    dec.prefill(np.random.default_rng(2).integers(0, hp.vocab_size, 70).astype(np.int32), 0)
    dec.begin(2)
    us, stage, n = np.zeros(64, np.float32), np.full(64, -7, np.int32), C.c_int32(-1)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert qh.lib().qh_decoder_step_timed(dec.h, 1, stream, us.ctypes.data, stage.ctypes.data, 64, C.byref(n)) == 0
    assert dec.outputs(2).tolist() == tokens and (bits(dec.hidden()) == bits(want[1])).all()
    per = [qh.STAGE_QKV, qh.STAGE_ATTENTION] + [qh.STAGE_ATTENTION] * (1 + joins) + [qh.STAGE_O, qh.STAGE_GATE_UP, qh.STAGE_DOWN]
    ids = [qh.STAGE_QKV] * 4 + [l * qh.STAGES_PER_LAYER + s for l in range(hp.n_layers) for s in per]
    assert stage[:n.value].tolist() == ids + [qh.STAGE_FINAL_NORM, qh.STAGE_HEAD, qh.STAGE_HEAD]
    assert (us[:n.value] > 0).all()
    dec.close()


def test_sampled_replies(qh, gpu):
    """The sampler over two forks of a prompt: one seed gives one reply, wherever its tokens lie."""
    hp, tens = model(4, **NARROW)
    dec = qh.Decoder(hp, tens, ctx_len=256)
    cache = cache_for(qh, hp)
    ids = np.random.default_rng(3).integers(0, hp.vocab_size, 50).astype(np.int32)
    dec.bind_kv8(cache, 0)
    dec.prefill(ids, 0)
    cache.fork(ints([0, 0, 0]), ints([1, 2, 3]))
    p = qh.sampler_params(temperature=5.0, top_k=20, top_p=1.0)
    replies = []
    for seq, seed in ((1, 7), (2, 7), (3, 8)):
        dec.bind_kv8(cache, seq)
        dec.set_query(p)
        dec.set_sampler(p, seed)
        dec.prefill(ids, 0, top_k=20)
        dec.begin(13, top_k=20)
        for _ in range(12):
            dec.step(top_k=20)
        replies.append(dec.outputs(13).tolist())
    assert dec.status() == 0 and int(cache.status) == 0
    assert replies[0] == replies[1] != replies[2]
    dec.close()


@pytest.mark.parametrize("shape", [NARROW, WIDE, {}])
@pytest.mark.parametrize("n", [40, 200])
def test_attention_agrees_with_the_f32_caches_over_the_same_values(qh, gpu, shape, n):
    """A decoder with an f32 cache, whose rows are overwritten by the bound cache's values in every layer, and the next token by
    both: what is left is that token's own keys and values in 8 bits (a rounding of a value is rms 0.0025 of it here, see the
    sizes below, with one of n weights) and its effect on the 8-bit activations behind it: a change of e shifts e / step of
    the codes by a step (about 0.024 of an activation's rms), so its rms is sqrt(0.024 e), 0.003 for e = 0.0025 * 4 / n at
    n = 40. Ten such roundings in two layers, taken as if they all pointed the same way, are 0.03 of the state. A wrong
    position, head, page or scale would be of the order of the state."""
    hp, tens = model(5, **shape)
    dec, ref = qh.Decoder(hp, tens, ctx_len=256), qh.Decoder(hp, tens, ctx_len=256, kv_f32=True)
    cache = cache_for(qh, hp)
    dec.bind_kv8(cache, 2)
    ids = np.random.default_rng(2).integers(0, hp.vocab_size, n + 1).astype(np.int32)
    for d in (dec, ref):
        d.prefill(ids[:n], 0)
    kvd = hp.n_kv_heads * hp.head_dim
    for l in range(hp.n_layers):
        for base, x in zip((ref.views.kcache_f32, ref.views.vcache_f32), stored(cache, l, 2, n)):
            x = np.ascontiguousarray(x, np.float32)
            assert qh.lib().qh_memcpy_h2d(C.c_void_p(base + 4 * l * 256 * kvd), x.ctypes.data, x.nbytes, None) == 0
            assert qh.lib().qh_stream_sync(None) == 0
    for d in (dec, ref):
        d.prefill(ids[n:], n)
    a, b = dec.hidden().astype(np.float64), ref.hidden().astype(np.float64)
    assert np.linalg.norm(a - b) <= 0.03 * np.linalg.norm(b), np.linalg.norm(a - b) / np.linalg.norm(b)
    dec.close()
    ref.close()
