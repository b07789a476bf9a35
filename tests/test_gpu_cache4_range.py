"""Attention over 4-bit caches where one row takes nearly everything, and a cache that is evicted twice."""
import numpy as np
import pytest
import torch

import plain_cache4 as P
from test_gpu_cache4 import Cache, bits, i32, near_attention, tensor

pytestmark = pytest.mark.gpu


def behind_a_dominant_row(lcu, dtype, seqs, m, heads, kv, held):
    """Row 0 of every head is 17.5 nats ahead of all others, which are alike, and holds zeros: an output is what the others leave, n 2^-25.2
    of their value.  An operand of the product with the values is a probability rounded to a half, at least 2^7 for the largest: off by
    2^-11 of itself or 2^-25, 2^-32 of the largest; the rest as in near_attention."""
    hd, bs = 128, 32
    rng = np.random.default_rng(held)
    n = held + m
    cache = Cache(lcu, seqs, kv, hd, n, bs, dtype)
    k = rng.integers(0, 16, hd).astype(np.uint8)
    k[0] = 0
    cache.codes[0][:] = torch.from_numpy(P.pack(k[None])).cuda()[0]
    k[0] = 15
    cache.codes[0][:, :, 0] = torch.from_numpy(P.pack(k[None])).cuda()[0]
    cache.scales[0][:] = 2.0
    v = rng.integers(8, 16, (n, hd)).astype(np.uint8)
    cache.codes[1][:] = torch.from_numpy(P.pack(v)).cuda()
    cache.scales[1][:] = 2.0
    cache.scales[1][:, :, 0] = 0.0
    qb = np.zeros((seqs * m, heads * hd), np.uint16)
    qb[:, ::hd] = P.float_to_bits(np.float32(6.6), dtype)
    q = float(P.bits_to_float(qb[0, 0], dtype))
    e = np.exp(-30.0 * q / np.sqrt(hd))
    assert 2.0 ** -25.6 < e < 2.0 ** -25.1
    out = P.bits_to_float(bits(cache.attend(tensor(qb, dtype), i32([held] * seqs), m, heads)), dtype).reshape(seqs, m, heads, hd)
    values = (v.astype(np.float64) - 7.5) * 2.0
    values[0] = 0.0
    seen = held + 1 + np.arange(m)
    want = (e * np.cumsum(values, 0)[seen - 1] / (1 + (seen - 1)[:, None] * e))[None, :, None]
    ds = 2 * hd * 2.0 ** -24 * 30 * q / np.sqrt(hd) + 2.0 ** -20
    tol = (P.step_of(dtype) + 1.01 * (2.0 ** -11 + 2 * ds + 2.0 ** -20)) * want + 2.0 ** -24 + (held + m) * 2.0 ** -32 * 15.0
    assert (np.abs(out - want) <= tol).all(), float((np.abs(out - want) / tol).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("seqs,m,heads,kv,held", [
    (16, 1, 16, 16, 5600), (16, 1, 64, 16, 5600), (2, 4, 16, 8, 20000),  # few rows, one and several heads per key
    (1, 500, 64, 16, 3000), (1, 130, 2, 1, 32000)])                      # prompts, whole items and shared tiles
def test_rows_far_behind_the_largest_count(lcu, dtype, seqs, m, heads, kv, held):
    behind_a_dominant_row(lcu, dtype, seqs, m, heads, kv, held)


@pytest.mark.parametrize("dtype,hd,bs", [("float16", 128, 32), ("bfloat16", 128, 64), ("float16", 64, 64), ("bfloat16", 128, 128)])
@pytest.mark.parametrize("seqs,m,lengths,heads,kv", [
    (2, 1, [150, 7], 4, 2), (1, 4, [150], 8, 2), (1, 1, [30001], 6, 2), (2, 1, [800, 3333], 24, 1), (1, 130, [150], 4, 2), (1, 40, [2500], 8, 4), (2, 200, [0, 91], 4, 4)])
def test_scores_of_tens_of_thousands(lcu, dtype, hd, bs, seqs, m, lengths, heads, kv):
    """Keys of odd whole numbers up to 15 in pairs of equal ones, and queries that are 64 times a key that the row sees: every product and sum is a
    whole number below 2^24, so scores are as exact as their scaling; the pair's are tens of thousands ahead of all others (or, of a pair whose
    second row is hidden, the first's), so what a score is off by is the same for all that count.  Tolerances of outputs: a probability
    rounded to a half, sums 2^-20, one rounding of the output.  A weight is 2 to the difference of a score and the logarithm of its row's
    sum, binary32 numbers of which one has been rounded before: below 2^17, by 2^-8 at most, and 2^(2^-8) is 1 + 0.00272."""
    rng = np.random.default_rng(m + heads + hd)
    ctx = max(lengths) + m + 1
    group = heads // kv
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    cache.codes[0][:, :, 1::2] = cache.codes[0][:, :, 0:ctx - ctx % 2:2]
    cache.scales[0][:], cache.scales[1][:] = 2.0, 0.5
    k, v = cache.values(0), cache.values(1)
    q = np.zeros((seqs, m, heads, hd))
    for s, held in enumerate(lengths):
        for i in range(m):
            for h in range(heads):
                q[s, i, h] = 64 * k[s, h // group, rng.integers(0, held + i + 1)]
    qb = P.float_to_bits(q.reshape(seqs * m, heads * hd), dtype)
    assert np.array_equal(P.bits_to_float(qb, dtype).reshape(q.shape), q) and 64 * (k ** 2).sum(-1).max() * 1.4427 / np.sqrt(hd) < 2 ** 17
    for weights in (None, torch.zeros(seqs, kv, ctx, device="cuda")):
        out = P.bits_to_float(bits(cache.attend(tensor(qb, dtype), i32(lengths), m, heads, weights=weights)), dtype).reshape(q.shape)
        for s, held in enumerate(lengths):
            rows = held + m
            o, p, spread, _ = P.attention(q[s], k[s][:, :rows], v[s][:, :rows], held, group)
            assert ((p > 0.49) | (p < 1e-30)).all()
            tol = P.step_of(dtype) * np.abs(o) + (2.0 ** -11 + 2.0 ** -20) * spread * 1.01
            assert (np.abs(out[s] - o) <= tol).all(), float((np.abs(out[s] - o) / tol).max())
            if weights is not None:
                want = p.reshape(kv, group * m, rows).sum(1)
                w = weights[s].double().cpu().numpy()
                assert (np.abs(w[:, :rows] - want) <= (0.00272 + 2.0 ** -19) * want + 1e-28).all() and (w[:, rows:] == 0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,held,heads,kv", [(1, 200, 6, 2), (4, 3000, 8, 2), (130, 0, 4, 2), (40, 2500, 8, 4), (300, 40, 16, 16)])
def test_scores_up_to_the_end_of_their_range(lcu, dtype, m, held, heads, kv):
    """Scores (powers of two) up to 2^26, of queries that are 8192 times a key's steps, exact as above; the rows that see one key alone have it with the
    other sign.  Outputs are the key's values: a probability rounded to a half, sums 2^-20, one rounding."""
    rng = np.random.default_rng(m)
    cache = Cache(lcu, 1, kv, 128, held + m, 32, dtype)
    cache.scales[0][:], cache.scales[1][:] = 16.0, 0.5
    k, v = cache.values(0)[0], cache.values(1)[0]
    q, want = np.zeros((m, heads, 128)), np.zeros((m, heads, 128))
    for i in range(m):
        for h in range(heads):
            d = rng.integers(0, held + i + 1)
            q[i, h] = k[h // (heads // kv), d] * (512 if held + i else -512)
            want[i, h] = v[h // (heads // kv), d]
            score = k[h // (heads // kv), :held + i + 1] @ q[i, h] * (1.4426950408889634 / np.sqrt(128))
            assert 2 ** 24 < abs(score[d]) < 2 ** 26 and (np.delete(score, d) < score[d] - 2 ** 20).all()
    qb = P.float_to_bits(q.reshape(m, heads * 128), dtype)
    assert np.array_equal(P.bits_to_float(qb, dtype).reshape(q.shape), q)
    for weights in (None, torch.zeros(1, kv, held + m, device="cuda")):
        out = P.bits_to_float(bits(cache.attend(tensor(qb, dtype), i32([held]), m, heads, weights=weights)), dtype).reshape(q.shape)
        assert (np.abs(out - want) <= (P.step_of(dtype) + (2.0 ** -11 + 2.0 ** -20) * 1.01) * np.abs(want)).all(), float(np.abs(out - want).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,held,heads,kv", [(1, 200, 4, 2), (3, 900, 8, 2), (140, 60, 4, 2)])
def test_values_below_the_normal_halves(lcu, dtype, m, held, heads, kv):
    """Scales from 2^-24 to 2^-17 under queries of thousands.  A value is off by 2^-24 at most, an output below the normal halves by 2^-25 more; keys as
    halves (prompts) are off by 2^-25, scores by the queries' sum of that, 8e-4, and the outputs by twice that of values of 1e-5, below 2^-25."""
    rng = np.random.default_rng(held)
    cache = Cache(lcu, 1, kv, 128, held + m, 32, dtype)
    cache.fill(rng, held + m)
    for which in range(2):
        steps = torch.from_numpy(rng.integers(1, 128, tuple(cache.scales[0].shape)).astype(np.float32)).cuda()
        cache.scales[which][:] = steps * 2.0 ** -24
    assert ((cache.scales[0] > 0) & (cache.scales[0] < 2.0 ** -17)).all()
    qb = P.float_to_bits(rng.standard_normal((m, heads * 128)) * 3000, dtype)
    w = torch.zeros(1, kv, held + m, device="cuda")
    q = P.bits_to_float(qb, dtype).reshape(m, heads, 128)
    o, p, spread, big = P.attention(q, cache.values(0)[0], cache.values(1)[0], held, heads // kv)
    assert np.abs(q).sum(-1).max() * 2.0 ** -25 / np.sqrt(128) < 1e-3 and np.abs(cache.values(1)).max() < 6e-5
    ds = (2 * 128 * 2.0 ** -24 * big + 8 * 2.0 ** -24 * (1 + big))[..., None]
    for weights in (None, w):
        out = P.bits_to_float(bits(cache.attend(tensor(qb, dtype), i32([held]), m, heads, weights=weights)), dtype).reshape(o.shape)
        tol = P.step_of(dtype) * np.abs(o) + (2.0 ** -11 + 2 * ds + 2.0 ** -20 + (2e-3 if m * heads // kv > 64 else 0)) * spread * 1.01 + 2.0 ** -24 + 2.0 ** -25
        assert (np.abs(out - o) <= tol).all(), float((np.abs(out - o) / tol).max())
    want = p.reshape(kv, -1, held + m).sum(1)
    assert (np.abs(w[0].double().cpu().numpy() - want) <= (2 * ds.max() + 2.0 ** -19 + 2e-3) * want + 2.0 ** -40).all()


def test_a_cache_is_evicted_twice(lcu):
    """A cache that fills up two times: positions run further ahead of lengths each time, kept rows and their weights follow the lists."""
    seqs, kv, heads, hd, bs, ctx, keep, recent, dtype = 2, 2, 4, 64, 32, 40, 17, 5, "float16"
    rng = np.random.default_rng(12)
    cache = lcu.Cache4(seqs, kv, hd, ctx, bs, dtype)
    weights = np.zeros((seqs, kv, ctx))
    position = evictions = 0
    for turn, m in enumerate([20] + [1] * 60):
        if cache.lengths.max() == ctx:
            got = cache.planes[4].to_host(np.float32, (seqs, kv, ctx))
            before = [P.bits_to_float(a, dtype) for a in cache.read(ctx)]
            kept = cache.evict(keep, recent)
            after = [P.bits_to_float(a, dtype) for a in cache.read(keep)]
            for s in range(seqs):
                for h in range(kv):
                    rows = P.evict(got[s, h], ctx, keep, recent)
                    assert kept[s, h].tolist() == rows
                    assert all(np.array_equal(a[s, h], b[s, h, rows]) for a, b in zip(after, before))
                    weights[s, h, :keep] = weights[s, h, rows]
            evictions += 1
            assert (cache.lengths == keep).all()
        held = int(cache.lengths[0])
        assert (cache.positions == position).all() and position - held == evictions * (ctx - keep)
        q, k, v = (P.float_to_bits(rng.standard_normal((seqs, m, c * hd)), dtype) for c in (heads, kv, kv))
        q_rot = cache.append(q, k, v)
        at = position + np.arange(m)
        turned = P.rotate(P.bits_to_float(q, dtype).reshape(seqs * m, heads, hd), np.tile(at, seqs), 10000.0).reshape(seqs, m, heads, hd)
        q64 = P.bits_to_float(q_rot, dtype).reshape(seqs, m, heads, hd)
        pair = np.repeat(np.hypot(turned[..., 0::2], turned[..., 1::2]), 2, -1)
        assert (np.abs(q64 - turned) <= 2.0 ** -11 * np.abs(turned) + 6 * 2.0 ** -24 * pair + 2.0 ** -25).all()
        cache.attend(q_rot)
        kk, vv = (P.bits_to_float(a, dtype) for a in cache.read(held + m))
        for s in range(seqs):
            _, p, _, _ = P.attention(q64[s], kk[s], vv[s], held, heads // kv)
            weights[s, :, held:] = 0
            weights[s, :, :held + m] += p.reshape(kv, -1, m, held + m).sum((1, 2))
        got = cache.planes[4].to_host(np.float32, (seqs, kv, ctx))
        # (sums of up to 61 steps, each within 2^-17 of itself: the scores' 2 x 64 x 2^-24 of sums of products up to 30, and 2^-19)
        assert (np.abs(got - weights)[:, :, :held + m] <= 2.0 ** -11 * weights[:, :, :held + m]).all()
        cache.advance(m)
        position += m
    assert evictions == 2
