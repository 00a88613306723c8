"""Beam search's selection (qh_beam_select) with scores of any finite size, to f32's ends: what is added to a logit is then so large
that candidates round to the same 64-bit score, and go to the lower beam, then the lower id.

The 64-bit score is (logit - largest logit of its row) + (score - log of the row's sum); the kernel's log differs from the exact one
by 2^-38 and what its own rounding adds, some 4e-12. Parents and tokens are equal where no border between two 64-bit scores lies in that
distance: a border is one in every 2^-52 of the score's size, so that the chance of it is below 1e-5 a row at 1e10 and less above, and
below 1e10 a score's step is so small that two candidates differ by more."""
import math

import pytest
import torch

from test_gpu_beam import TYPES, check, make

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min
SIZES = [-1e10, -1e12, -1e15, -1e16, -1e18, -1e30, LOWEST, 1e12, 1e17, -LOWEST]


@pytest.mark.parametrize("score", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("prompts,beams,vocab,k", [(2, 1, 1, 3), (3, 4, 1000, 8), (1, 1, 5003, 40), (2, 3, 50257, 8), (1, 4, 151936, 8),
                                                  (1, 4, 151936, 33), (1, 8, 30000, 256)])
def test_all_scores_large(qh, gpu, dtype, score, prompts, beams, vocab, k):
    """Every beam has the same score; then each one of its own, some next to each other."""
    rows = prompts * beams
    logits, _ = make(gpu, rows, vocab, dtype, seed=vocab + k)
    scores = torch.full((rows,), score, device=gpu)
    check(qh, logits, scores, beams, k)
    if abs(score) < 1e38:
        scores *= 1 + torch.arange(rows, device=gpu) % 3 * 0.25
        check(qh, logits, scores, beams, k)


@pytest.mark.parametrize("score", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("k", [1, 8, 256])
def test_some_scores_large(qh, gpu, dtype, score, k):
    """A prompt's first, middle or last beams with a large score, the others ordinary: fewer ids in those than k, so that both kinds
    are chosen, and more."""
    for vocab in (5, 60, 7000):
        logits, scores = make(gpu, 12, vocab, dtype, seed=k)
        scores[[0, 5, 6, 7, 11]] = score
        check(qh, logits, scores, 4, k)
        check(qh, logits, scores, 12, k)


@pytest.mark.parametrize("score", [-1e16, -1e30, LOWEST])
def test_many_beams_large(qh, gpu, score):
    """So many candidates of one 64-bit score that the pool of those held overflows again and again."""
    logits, _ = make(gpu, 32, 50257, "f16", spread=0.5)
    check(qh, logits, torch.full((32,), score, device=gpu), 16, 64)
    check(qh, logits, torch.full((32,), score, device=gpu), 32, 256)


@pytest.mark.parametrize("score", [-1e16, LOWEST])
def test_masks_with_large_scores(qh, gpu, score):
    """Forbidden ids, rows of them alone and rows that are out, among beams of one large score."""
    logits, _ = make(gpu, 8, 3001, "f32")
    logits[0, 5:] = -math.inf
    logits[1] = -math.inf
    logits[2, ::2] = torch.finfo(torch.float32).min
    logits[3, 7] = math.nan
    scores = torch.full((8,), score, device=gpu)
    scores[4] = -math.inf
    for k in (1, 8, 256):
        check(qh, logits, scores, 4, k)
        check(qh, logits, scores, 8, k)
