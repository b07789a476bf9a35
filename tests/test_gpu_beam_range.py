"""Beam selection over the whole range of finite logits: masks of large negative numbers, large offsets, large maxima."""
import numpy as np
import pytest

import plain_cache4 as P

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of binary32
# Scores: terms of a sum of exponentials are 2^-22 off by themselves, and by their argument's roundings (the difference, the factor, the product:
# 2.25 U of it, whose mean under the softmax is at most the logarithm of the vocabulary, 10.4 here); sixteen are added up in binary32
# (15 U), a chunk's sum is rounded (U) and scaled (2^-22 and 3 U): 2^-18.2 together at worst.  The result is rounded once.
SUM = 2.0 ** -18


def best(logits, scores, n_out):
    """One group in binary64: differences from a beam's maximum before anything is lost."""
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    beams, vocab = x.shape
    top = x.max(-1, keepdims=True)
    total = ((x - top) - np.log(np.exp(x - top).sum(-1, keepdims=True))) + scores.astype(np.float64)[:, None]
    beam, token = np.repeat(np.arange(beams), vocab), np.tile(np.arange(vocab), beams)
    order = np.lexsort((token, -x.ravel(), beam, -total.ravel()))[:n_out]
    return beam[order], token[order], total.ravel()[order]


def run(lcu, x, scores, n_out, dtype):
    """x [groups, beams, vocab] in binary32, rounded to the type."""
    logits = x if dtype == "float32" else P.float_to_bits(x, dtype)
    x64 = x.astype(np.float64) if dtype == "float32" else P.bits_to_float(logits, dtype)
    parents, tokens, out = lcu.beam_select(logits, scores, n_out, dtype)
    for g in range(len(x)):
        p, t, s = best(x64[g], scores[g], n_out)
        apart = (p[1:] != p[:-1]) & (s[1:] != s[:-1])
        assert (np.abs(np.diff(s))[apart] > 2 * SUM).all()  # (no neighbours of different beams that rounding could turn)
        assert parents[g].tolist() == p.tolist() and tokens[g].tolist() == t.tolist(), g
        with np.errstate(over="ignore"):
            want = s.astype(np.float32)
        fine = np.isfinite(want)
        assert np.array_equal(out[g][~fine], want[~fine])
        assert (np.abs(out[g][fine] - s[fine]) <= SUM + U * np.abs(s[fine])).all(), float(np.abs(out[g][fine] - s[fine]).max())


MASKS = [("float32", -1e30), ("float32", -1e20), ("float32", -3.4028235e38), ("float32", -2.4e38), ("bfloat16", -1e30), ("bfloat16", -3.3895314e38), ("float16", -65504.0)]


@pytest.mark.parametrize("dtype,mask", MASKS)
@pytest.mark.parametrize("vocab", [4096, 9000])
def test_masks_of_finite_numbers(lcu, dtype, mask, vocab):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((5, 3, vocab)) * 2.5).astype(np.float32)
    scores = np.array([[-1.0, -1.25, -0.5]] * 5, np.float32)
    x[0, 1, :4096] = mask                            # a whole chunk
    x[1, 1, vocab - vocab % 4096 or 5:] = mask       # the short last chunk
    x[2, :, 100:] = mask                             # few tokens are left
    x[3, 2] = mask                                   # a beam with nothing but masks: all its tokens are as likely
    scores[3] = [-20.0, -20.5, 9.0]
    x[4] = mask                                      # two tokens are left in all
    x[4, 0, 7] = 1.0
    x[4, 2, vocab - 1] = -2.0
    for n_out in (1, 4, 40):
        run(lcu, x, scores, n_out, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [700, 32000])
def test_offsets_change_nothing(lcu, dtype, vocab):
    """Beams whose logits lie around 0, 100, 1000 and 30000, either sign."""
    rng = np.random.default_rng(vocab + 1)
    x = (rng.standard_normal((2, 4, vocab)) * 2.5).astype(np.float32)
    offsets = np.array([[0.0, 100.0, 1000.0, 30000.0], [-30000.0, -100.0, 0.37, -1000.0]], np.float32)
    x += offsets[..., None]
    run(lcu, x, np.array([[-1.0, -1.3, -0.7, -1.1]] * 2, np.float32), 9, dtype)


@pytest.mark.parametrize("dtype,large", [("float32", 3.4028235e38), ("float32", 2.4e38), ("float32", 1e20), ("bfloat16", 3.3895314e38), ("float16", 65504.0)])
def test_large_maxima(lcu, dtype, large):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((1, 3, 5000)) * 2.5).astype(np.float32)
    x[0, 0, 4999] = large
    x[0, 1, [3, 4097, 4098]] = large
    x[0, 2, 17] = -large
    run(lcu, x, np.array([[-1.0, -1.5, 0.0]], np.float32), 6, dtype)
