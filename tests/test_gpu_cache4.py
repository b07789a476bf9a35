"""The operators over 4-bit caches on the GPU against the definitions in binary64."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_cache4 as P

pytestmark = pytest.mark.gpu
TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16}
U = 2.0 ** -24  # half a step of binary32


def tensor(bits, dtype):
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16).copy()).cuda().view(TORCH[dtype])


def bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Cache:
    """Planes filled with NaN scales and random codes, so that rows nothing was written to would show."""

    def __init__(self, lcu, seqs, kv, hd, ctx, bs, dtype="float16", seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lcu, self.seqs, self.kv, self.hd, self.ctx, self.bs, self.dtype = lcu, seqs, kv, hd, ctx, bs, dtype
        self.codes = [torch.randint(0, 256, (seqs, kv, ctx, hd // 2), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.full((seqs, kv, ctx, hd // bs), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
        self.planes = [self.codes[0], self.scales[0], self.codes[1], self.scales[1]]

    def ptrs(self):
        return [p.data_ptr() for p in self.planes]

    def shape(self):
        return self.kv, self.hd, self.bs, self.ctx

    def fill(self, rng, rows, scale=1.0):
        """`rows` random rows per sequence."""
        for which in range(2):
            x = (rng.standard_normal((self.seqs, self.kv, rows, self.hd)) * scale).astype(np.float32)
            s = P.scales_of(x, self.bs)
            self.codes[which][:, :, :rows] = torch.from_numpy(P.pack(P.codes_of(x, s, self.bs))).cuda()
            self.scales[which][:, :, :rows] = torch.from_numpy(s).cuda()

    def values(self, which):
        return P.values_of(P.unpack(self.codes[which].cpu().numpy()), self.scales[which].cpu().numpy(), self.bs)

    def append(self, q, k, v, lengths, positions, m, heads, theta, q_out=None, stream=None):
        lcu = self.lcu
        q_out = torch.empty(q.shape[0], heads * self.hd, dtype=q.dtype, device="cuda") if q_out is None else q_out
        lcu.check(lcu.lib.lcu_cache4_append(*self.ptrs(), q_out.data_ptr(), q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0), lengths.data_ptr(),
                                            None if positions is None else positions.data_ptr(), self.seqs, m, heads, *self.shape(), theta,
                                            lcu.OP_DTYPES[self.dtype], stream))
        return q_out

    def attend(self, q, lengths, m, heads, most=None, weights=None, beta=0.0, out=None, ws=None, stream=None):
        lcu = self.lcu
        most = most or self.ctx
        out = torch.full((q.shape[0], heads * self.hd), 77.0, dtype=q.dtype, device="cuda") if out is None else out
        need = lcu.lib.lcu_attention_cache4_workspace(self.seqs, m, heads, self.kv, self.hd, most, int(weights is not None))
        ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda") if ws is None else ws
        lcu.check(lcu.lib.lcu_attention_cache4(out.data_ptr(), out.stride(0), None if weights is None else weights.data_ptr(), beta, q.data_ptr(), q.stride(0), *self.ptrs(),
                                               lengths.data_ptr(), self.seqs, m, heads, *self.shape(), most, lcu.OP_DTYPES[self.dtype], ws.data_ptr(), need, stream))
        if stream is None:
            torch.cuda.synchronize()
            assert (ws[need:] == 255).all()  # (nothing behind the workspace)
        return out


def near_attention(cache, out, q_bits, lengths, m, heads, weights=None, old=None, beta=0.0, limit=None):
    """Tolerances: one rounding of the output; every probability rounded to a half once (2^-11 of it); scores in binary32 over hd products
    (their rounding and the order of their sum: 2 hd U of sum |q k|, and the factors of the softmax a few U); sums of probabilities 2^-20."""
    hd, seqs = cache.hd, cache.seqs
    q = P.bits_to_float(q_bits, cache.dtype).reshape(seqs, m, heads, hd)
    got = P.bits_to_float(bits(out), cache.dtype).reshape(seqs, m, heads, hd)
    k, v = cache.values(0), cache.values(1)
    group = heads // cache.kv
    for s, held in enumerate(lengths):
        rows = min(cache.ctx, limit or cache.ctx, max(0, held + m)) if held >= 0 else 0
        o, p, spread, big = P.attention(q[s], k[s][:, :rows], v[s][:, :rows], held, group)
        ds = (2 * hd * U * big + 8 * U * (1 + big))[..., None]
        tol = P.step_of(cache.dtype) * np.abs(o) + (2.0 ** -11 + 2 * ds + 2.0 ** -20) * spread * 1.01 + 2.0 ** -24
        assert (np.abs(got[s] - o) <= tol).all(), (s, float((np.abs(got[s] - o) / tol).max()))
        if weights is not None:
            w = weights[s].double().cpu().numpy()
            want = p.reshape(cache.kv, group * m, rows).sum(1)
            tol = (2 * ds.max() + 2.0 ** -19) * want + 2.0 ** -40
            before = old[s].double().cpu().numpy()
            want[:, :max(0, held)] += beta * before[:, :max(0, held)]
            assert (np.abs(w[:, :rows] - want) <= tol + 2.0 ** -22 * np.abs(want)).all(), (s, float((np.abs(w[:, :rows] - want) / tol).max()))
            assert np.array_equal(w[:, rows:], before[:, rows:], equal_nan=True)


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd,bs", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("heads,kv,m,theta", [(1, 1, 1, 10000.0), (6, 3, 5, 10000.0), (32, 32, 1, 0.0), (7, 1, 37, 500000.0)])
def test_append_and_read(lcu, dtype, hd, bs, heads, kv, m, theta):
    seqs, ctx = 3, 64
    rng = np.random.default_rng(hd + bs + heads + m)
    lengths, positions = np.array([0, 11, 27]), np.array([0, 100007, 5])
    ldq, ldkv = heads * hd + 8, kv * hd + 16
    qb, kb, vb = (P.float_to_bits(rng.standard_normal((seqs * m, n)) * 2.0, dtype) for n in (ldq, ldkv, ldkv))
    kb[:, :hd // 2] = 0
    vb[0, :hd] = 0  # blocks of zeros
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    before = [p.clone() for p in cache.planes]
    q, k, v = tensor(qb, dtype), tensor(kb, dtype), tensor(vb, dtype)
    q_out = cache.append(q[:, :heads * hd], k[:, :kv * hd], v[:, :kv * hd], i32(lengths), i32(positions), m, heads, theta)
    torch.cuda.synchronize()
    at = (positions[:, None] + np.arange(m)).ravel()
    q64 = P.rotate(P.bits_to_float(qb[:, :heads * hd], dtype).reshape(-1, heads, hd), at, theta)
    got = P.bits_to_float(bits(q_out), dtype).reshape(q64.shape)
    pair = np.repeat(np.hypot(q64[..., 0::2], q64[..., 1::2]), 2, -1)
    # cosine and sine rounded to binary32 (U each), two products and a sum: 4 U of the pair's length; one rounding
    assert (np.abs(got - q64) <= P.step_of(dtype) * np.abs(q64) + 6 * U * pair + 2.0 ** -25).all()
    # (the rotated keys as binary32 numbers, within 6 U of the pair's length of the formula's)
    k64 = P.rotate(P.bits_to_float(kb[:, :kv * hd], dtype).reshape(-1, kv, hd), at, theta).reshape(seqs, m, kv, hd).transpose(0, 2, 1, 3)
    v64 = P.bits_to_float(vb[:, :kv * hd], dtype).reshape(seqs, m, kv, hd).transpose(0, 2, 1, 3)
    for s in range(seqs):
        n = slice(lengths[s], lengths[s] + m)
        vs = P.scales_of(v64[s], bs)
        assert np.array_equal(cache.scales[1][s, :, n].cpu().numpy(), vs)
        assert np.array_equal(cache.codes[1][s, :, n].cpu().numpy(), P.pack(P.codes_of(v64[s], vs, bs)))
        ks = cache.scales[0][s, :, n].cpu().numpy()
        if theta == 0:
            assert np.array_equal(ks, P.scales_of(k64[s], bs))
            assert np.array_equal(cache.codes[0][s, :, n].cpu().numpy(), P.pack(P.codes_of(k64[s], ks, bs)))
        else:
            a = np.abs(k64[s]).reshape(kv, m, -1, bs).max(-1)
            # 7 bits: half a step is 2^-7 of the value at most (2^-8 just below a power of two); halves below 2^-14 in steps of 2^-24
            assert (np.abs(ks.astype(np.float64) - a / 7.5) <= 2.0 ** -7 * a / 7.5 * (1 + 1e-5) + 2.0 ** -24).all()
            held = P.values_of(P.unpack(cache.codes[0][s, :, n].cpu().numpy()), ks, bs)
            step = np.repeat(ks.astype(np.float64), bs, -1)
            over = np.maximum(0, np.abs(k64[s]) - 8 * step)  # (nothing lies above the last code's half step)
            length = np.repeat(np.hypot(k64[s][..., 0::2], k64[s][..., 1::2]), 2, -1)
            assert (over <= 6 * U * length + 2.0 ** -24).all()
            assert (np.abs(held - k64[s]) <= 0.5 * step * (1 + 1e-5) + 6 * U * length).all()
    # read: the values, rounded to the type (bfloat16) or as they are (halves); rows outside the cache are zeros
    for count, first in ((m, lengths), (9, np.array([-4, 60, 20]))):
        outs = [torch.full((seqs, kv, count, hd), 5.0, dtype=TORCH[dtype], device="cuda") for _ in range(2)]
        lcu.check(lcu.lib.lcu_cache4_read(outs[0].data_ptr(), outs[1].data_ptr(), *cache.ptrs(), i32(first).data_ptr(), seqs, count, *cache.shape(), lcu.OP_DTYPES[dtype], None))
        torch.cuda.synchronize()
        for which in range(2):
            val, got = cache.values(which), P.bits_to_float(bits(outs[which]), dtype)
            for s in range(seqs):
                for i in range(count):
                    j = first[s] + i
                    want = P.bits_to_float(P.float_to_bits(val[s, :, j], dtype), dtype) if 0 <= j < ctx else np.zeros((kv, hd))
                    assert np.array_equal(got[s, :, i], want, equal_nan=True), (which, s, i)
    # rows that the call does not own
    for p, old in zip(cache.planes, before):
        for s in range(seqs):
            for r in (slice(0, lengths[s]), slice(lengths[s] + m, ctx)):
                assert torch.equal(p[s, :, r].contiguous().view(torch.uint8), old[s, :, r].contiguous().view(torch.uint8))


def test_append_borders_and_numbers_that_are_none(lcu):
    """Half-way values, the largest and smallest halves, huge bfloat16, infinities and NaN; no queries; in-place queries; rows behind the cache's
    end and unused sequences."""
    hd, bs, ctx = 64, 32, 4
    for dtype in ("float16", "bfloat16"):
        x = np.zeros((8, hd), np.float32)
        x[0] = np.arange(hd) % 16 - 7.5
        x[1] = np.where(np.arange(hd) % 2, 0.5, 7.5) * 2.0 ** -20
        x[2] = 65504.0
        x[3] = np.linspace(-3, 3, hd)
        x[3, 5] = np.inf
        x[4] = np.linspace(-3, 3, hd)
        x[4, 40] = np.nan
        x[5] = 3e38 if dtype == "bfloat16" else 60000.0
        x[6, 0], x[6, 1] = 1e-7, -6e-8
        x[7] = np.linspace(-1, 1, hd)
        b = P.float_to_bits(x, dtype)
        x64 = P.bits_to_float(b, dtype)
        cache = Cache(lcu, 4, 1, hd, ctx, bs, dtype)
        old = [p.clone() for p in cache.planes]
        q = tensor(np.tile(b, (1, 2)), dtype)
        same = q.clone()
        lengths = i32([2, 0, -1, 3])  # rows 2, 3; 0, 1; none; 3 and one behind the end
        cache.append(q, tensor(b, dtype), tensor(b, dtype), lengths, None, 2, 2, 0.0, q_out=q)
        torch.cuda.synchronize()
        assert torch.equal(q.view(torch.int16), same.view(torch.int16))  # no rotation
        for s, first, rows in ((0, 2, (0, 1)), (1, 0, (2, 3)), (3, 3, (6,))):
            for which in range(2):
                w = x64[list(rows)][None]
                n = slice(first, first + len(rows))
                sc = P.scales_of(w, bs)
                assert np.array_equal(cache.scales[which][s, :, n].cpu().numpy(), sc, equal_nan=True)
                assert np.array_equal(cache.codes[which][s, :, n].cpu().numpy(), P.pack(P.codes_of(w, sc, bs)))
        for p, o in zip(cache.planes, old):
            assert torch.equal(p[2].contiguous().view(torch.uint8), o[2].contiguous().view(torch.uint8))
            assert torch.equal(p[3, :, :3].contiguous().view(torch.uint8), o[3, :, :3].contiguous().view(torch.uint8))
        lcu.check(lcu.lib.lcu_cache4_append(*cache.ptrs(), None, None, 0, tensor(b, dtype).data_ptr(), tensor(b, dtype).data_ptr(), hd, lengths.data_ptr(), None, 4, 2, 0,
                                            *cache.shape(), 0.0, lcu.OP_DTYPES[dtype], None))
        torch.cuda.synchronize()


# ------------------------------------------------------------------ attention
CASES = [
    # seqs, m, lengths before, heads, kv
    (1, 1, [0], 1, 1),
    (1, 1, [16], 4, 4),
    (2, 1, [130, 7], 8, 2),
    (3, 1, [1023, -1, 255], 7, 1),
    (1, 1, [2500], 24, 2),
    (2, 1, [64, 63], 40, 2),
    (1, 2, [0], 2, 2),
    (2, 3, [15, 16], 8, 4),
    (2, 5, [200, -3], 14, 2),
    (1, 17, [0], 3, 3),
    (1, 64, [64], 4, 4),
    (2, 65, [0, 127], 4, 2),
    (1, 129, [300], 7, 1),
    (1, 200, [57], 4, 1),
    (1, 300, [0], 2, 2),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd,bs", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("seqs,m,lengths,heads,kv", CASES)
def test_attention(lcu, dtype, hd, bs, seqs, m, lengths, heads, kv):
    rng = np.random.default_rng(m + heads + hd)
    ctx = max(lengths) + m + 3
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    for s, n in enumerate(lengths):  # (rows behind the last one keep codes at random and scales that are no numbers)
        one = Cache(lcu, 1, kv, hd, ctx, bs, dtype)
        if n >= 0:
            one.fill(rng, n + m)
        for p, o in zip(cache.planes, one.planes):
            p[s] = o[0]
    qb = P.float_to_bits(rng.standard_normal((seqs * m, heads * hd + 8)) * 1.5, dtype)
    q = tensor(qb, dtype)[:, :heads * hd]
    out = torch.full((seqs * m, heads * hd + 16), 9.0, dtype=TORCH[dtype], device="cuda")
    plain = cache.attend(q, i32(lengths), m, heads, out=out[:, :heads * hd])
    assert (out[:, heads * hd:] == 9.0).all()
    near_attention(cache, plain, qb[:, :heads * hd], lengths, m, heads)
    old = torch.rand(seqs, kv, ctx, device="cuda")
    for s, n in enumerate(lengths):
        old[s, :, max(0, n):] = float("nan")  # (entries of the call's own rows are not read)
    for beta in (0.0, 0.75):
        w = old.clone()
        again = cache.attend(q, i32(lengths), m, heads, weights=w, beta=beta)
        near_attention(cache, again, qb[:, :heads * hd], lengths, m, heads, weights=w, old=old, beta=beta)
        twice = old.clone()
        third = cache.attend(q, i32(lengths), m, heads, weights=twice, beta=beta)
        assert torch.equal(third.view(torch.int16), again.view(torch.int16)) and torch.equal(twice.view(torch.int32), w.view(torch.int32))


LONG = [
    # seqs, m, lengths before, heads, kv: runs of chunks over several sequences and heads, columns in several blocks, tiles shared by CTAs
    (3, 1, [3000, 0, 1700], 4, 2),
    (4, 1, [900, -1, 2100, 31], 12, 1),
    (1, 1, [4500], 40, 1),
    (2, 5, [1500, 2222], 16, 4),
    (1, 13, [3333], 8, 2),
    (1, 40, [2500], 8, 4),
    (3, 33, [1200, -1, 100], 6, 2),
]


@pytest.mark.parametrize("dtype,hd,bs", [("float16", 128, 32), ("bfloat16", 128, 64), ("float16", 128, 128), ("bfloat16", 64, 32), ("float16", 64, 64)])
@pytest.mark.parametrize("seqs,m,lengths,heads,kv", LONG)
def test_attention_of_long_caches(lcu, dtype, hd, bs, seqs, m, lengths, heads, kv):
    rng = np.random.default_rng(m + heads + hd + bs)
    ctx = max(lengths) + m + 1  # (an odd number of rows where blocks are whole rows: scales between words)
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    for s, n in enumerate(lengths):
        one = Cache(lcu, 1, kv, hd, ctx, bs, dtype)
        if n >= 0:
            one.fill(rng, n + m)
        for p, o in zip(cache.planes, one.planes):
            p[s] = o[0]
    qb = P.float_to_bits(rng.standard_normal((seqs * m, heads * hd)) * 1.5, dtype)
    old = torch.rand(seqs, kv, ctx, device="cuda")
    plain = cache.attend(tensor(qb, dtype), i32(lengths), m, heads)
    near_attention(cache, plain, qb, lengths, m, heads)
    w = old.clone()
    out = cache.attend(tensor(qb, dtype), i32(lengths), m, heads, weights=w, beta=0.5)
    near_attention(cache, out, qb, lengths, m, heads, weights=w, old=old, beta=0.5)
    # a block of values, and one of keys, without numbers: all dimensions of the rows that see the key, that block of those that see the values
    group = heads // kv
    row_v, row_k = lengths[0] // 3, lengths[0] + m // 2
    cache.scales[1][0, 0, row_v, 0] = float("nan")
    cache.scales[0][0, kv - 1, row_k, hd // bs - 1] = float("nan")
    odd = cache.attend(tensor(qb, dtype), i32(lengths), m, heads).float().view(seqs, m, heads, hd)
    want = plain.float().view(seqs, m, heads, hd).clone()
    want[0, :, :group, :bs] = float("nan")
    want[0, m // 2:, heads - group:] = float("nan")
    assert torch.equal(torch.isnan(odd), torch.isnan(want))
    assert torch.equal(odd[~torch.isnan(want)], want[~torch.isnan(want)])


def test_captured_prompts_and_two_calls_at_once(lcu):
    """A prompt's attention with weights captured and replayed on other rows; the same on two streams at the same time, a workspace each."""
    hd, bs, kv, heads, dtype, m, held = 128, 32, 2, 8, "float16", 70, 130
    rng = np.random.default_rng(6)
    caches = [Cache(lcu, 1, kv, hd, held + m, bs, dtype) for _ in range(2)]
    bits_of, qs, outs, ws, weights, streams = [], [], [], [], [], [torch.cuda.Stream() for _ in range(2)]
    need = lcu.lib.lcu_attention_cache4_workspace(1, m, heads, kv, hd, held + m, 1)
    for c in caches:
        c.fill(rng, held + m)
        bits_of.append(P.float_to_bits(rng.standard_normal((m, heads * hd)), dtype))
        qs.append(tensor(bits_of[-1], dtype))
        outs.append(torch.zeros(m, heads * hd, dtype=torch.float16, device="cuda"))
        ws.append(torch.empty(need, dtype=torch.uint8, device="cuda"))
        weights.append(torch.zeros(1, kv, held + m, device="cuda"))
    lengths = i32([held])
    torch.cuda.synchronize()
    for _ in range(3):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                caches[k].attend(qs[k], lengths, m, heads, weights=weights[k], beta=0.0, out=outs[k], ws=ws[k], stream=streams[k].cuda_stream)
    torch.cuda.synchronize()
    zero = torch.zeros_like(weights[0])
    for k in range(2):
        near_attention(caches[k], outs[k], bits_of[k], [held], m, heads, weights=weights[k], old=zero)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        caches[0].attend(qs[0], lengths, m, heads, weights=weights[0], beta=0.0, out=outs[0], ws=ws[0], stream=torch.cuda.current_stream().cuda_stream)
    for n in (held, 60, 0):
        b = P.float_to_bits(rng.standard_normal((m, heads * hd)), dtype)
        qs[0].copy_(tensor(b, dtype))
        lengths.copy_(i32([n]))
        old = weights[0].clone()
        graph.replay()
        torch.cuda.synchronize()
        near_attention(caches[0], outs[0], b, [n], m, heads, weights=weights[0], old=old)


@pytest.mark.parametrize("m", [1, 4, 130])
def test_attention_of_extreme_scores(lcu, m):
    """Scores of thousands either way, one key that takes everything, equal keys, queries of zero, tiny and large bfloat16 queries."""
    hd, bs, kv, heads, held = 128, 32, 2, 4, 150
    rng = np.random.default_rng(5)
    for dtype in ("float16", "bfloat16"):
        for scale_q, scale_k in ((60.0, 30.0), (0.0, 1.0), (1e-4, 1.0), (3000.0, 5.0)):
            cache = Cache(lcu, 1, kv, hd, held + m, bs, dtype)
            cache.fill(rng, held + m, scale_k)
            qb = P.float_to_bits(rng.standard_normal((m, heads * hd)) * scale_q, dtype)
            w = torch.zeros(1, kv, held + m, device="cuda")
            out = cache.attend(tensor(qb, dtype), i32([held]), m, heads, weights=w)
            near_attention(cache, out, qb, [held], m, heads, weights=w, old=torch.zeros_like(w))


@pytest.mark.parametrize("m", [1, 3, 40, 140])
@pytest.mark.parametrize("hd,bs", [(64, 64), (128, 32)])
def test_numbers_that_are_none_stay_with_the_rows_that_see_them(lcu, m, hd, bs):
    kv, heads, held, dtype = 2, 6, 21, "float16"
    rng = np.random.default_rng(m)
    group = heads // kv
    for which, row in ((1, held + m - 1), (1, held + m // 2), (0, held + m // 2), (1, 3)):
        cache = Cache(lcu, 1, kv, hd, held + m + 2, bs, dtype)
        cache.fill(rng, held + m)
        qb = P.float_to_bits(rng.standard_normal((m, heads * hd)), dtype)
        fine = cache.attend(tensor(qb, dtype), i32([held]), m, heads)
        near_attention(cache, fine, qb, [held], m, heads)
        blk = hd // bs - 1
        cache.scales[which][0, 1, row, blk] = float("nan")
        out = cache.attend(tensor(qb, dtype), i32([held]), m, heads).float().view(m, heads, hd).cpu()
        want = fine.float().view(m, heads, hd).cpu().clone()
        first = max(0, row - held)
        if which:
            want[first:, group:, blk * bs:] = float("nan")
        else:
            want[first:, group:] = float("nan")
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(out[ok], want[ok])


def test_attention_reads_no_further_than_max_len(lcu):
    hd, bs, kv, heads, dtype = 128, 64, 1, 8, "bfloat16"
    rng = np.random.default_rng(8)
    for m, held, most in ((1, 99, 100), (1, 99, 37), (6, 90, 50), (140, 90, 200)):
        cache = Cache(lcu, 1, kv, hd, 256, bs, dtype)
        cache.fill(rng, held + m)
        qb = P.float_to_bits(rng.standard_normal((m, heads * hd)), dtype)
        out = cache.attend(tensor(qb, dtype), i32([held]), m, heads, most=most)
        near_attention(cache, out, qb, [held], m, heads, limit=most)


def test_long_caches_pass_32_bit_offsets(lcu):
    """Planes of more than 2^31 bytes: the last sequence's rows lie behind them."""
    hd, bs, kv, heads, dtype, ctx, seqs = 128, 32, 8, 8, "float16", 140000, 33
    rng = np.random.default_rng(2)
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    assert cache.codes[0].numel() > 1 << 31
    lengths = np.full(seqs, -1)
    lengths[-1] = 40
    one = Cache(lcu, 1, kv, hd, ctx, bs, dtype)
    one.fill(rng, 41)
    for p, o in zip(cache.planes, one.planes):
        p[-1, :, :41] = o[0, :, :41]
    del one
    qb = P.float_to_bits(rng.standard_normal((seqs, heads * hd)), dtype)
    w = torch.zeros(seqs, kv, ctx, device="cuda")
    out = cache.attend(tensor(qb, dtype), i32(lengths), 1, heads, most=64, weights=w)
    assert (out[:-1] == 0).all() and (w[:-1] == 0).all()
    tail = Cache(lcu, 1, kv, hd, 64, bs, dtype)
    for p, o in zip(tail.planes, cache.planes):
        p[0] = o[-1, :, :64]
    near_attention(tail, out[-1:], qb[-1:], [40], 1, heads, weights=w[-1:, :, :64], old=torch.zeros(1, kv, 64, device="cuda"))
    kb = P.float_to_bits(rng.standard_normal((seqs, kv * hd)), dtype)
    cache.append(tensor(qb, dtype), tensor(kb, dtype), tensor(kb, dtype), i32(lengths + (lengths >= 0) * (ctx - 41)), None, 1, heads, 0.0)
    x = P.bits_to_float(kb[-1:], dtype).reshape(1, kv, hd)[0]
    assert np.array_equal(cache.scales[1][-1, :, ctx - 1].cpu().numpy(), P.scales_of(x, bs))
    planes = (C.c_void_p * 1)(cache.codes[0].data_ptr())
    kept = torch.zeros(seqs, kv, 2, dtype=torch.int32, device="cuda")
    was = cache.codes[0][-1, :, ctx - 2:].clone()
    lcu.check(lcu.lib.lcu_cache_evict(planes, planes, (C.c_int * 1)(hd // 2), 1, w.data_ptr(), kept.data_ptr(), None, i32([-1] * (seqs - 1) + [ctx]).data_ptr(), seqs, kv, ctx,
                                      ctx, 2, 2, None))
    torch.cuda.synchronize()
    assert torch.equal(cache.codes[0][-1, :, :2], was) and (kept[:-1] == -1).all()


def test_replayed_steps_follow_their_lengths(lcu):
    """A captured step (append and attention with weights) on a side stream, replayed with other lengths, positions and rows."""
    hd, bs, kv, heads, dtype, ctx, seqs = 128, 32, 2, 8, "float16", 96, 2
    rng = np.random.default_rng(4)
    cache = Cache(lcu, seqs, kv, hd, ctx, bs, dtype)
    cache.fill(rng, 90)
    q, k, v = (torch.zeros(seqs, n * hd, dtype=torch.float16, device="cuda") for n in (heads, kv, kv))
    q_out, out, w = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(seqs, kv, ctx, device="cuda")
    lengths, positions = i32([0, 0]), i32([0, 0])
    ws = torch.empty(lcu.lib.lcu_attention_cache4_workspace(seqs, 1, heads, kv, hd, ctx, 1) + 16, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()

    def step():
        s = torch.cuda.current_stream().cuda_stream
        cache.append(q, k, v, lengths, positions, 1, heads, 10000.0, q_out=q_out, stream=s)
        cache.attend(q_out, lengths, 1, heads, weights=w, beta=1.0, out=out, ws=ws, stream=s)

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for held in ([5, 40], [6, 41], [89, 12]):
        lengths.copy_(i32(held))
        positions.copy_(i32(held) + 1000)
        for t in (q, k, v):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape))))
        old = w.clone()
        graph.replay()
        torch.cuda.synchronize()
        near_attention(cache, out, bits(q_out), held, 1, heads, weights=w, old=old, beta=1.0)


# ------------------------------------------------------------------ eviction
def evict(lcu, dst, src, weights, lengths, ctx, dctx, keep, recent, lengths_out=None):
    seqs, kv = weights.shape[:2]
    arr = lambda ts: (C.c_void_p * max(1, len(ts)))(*[t.data_ptr() for t in ts])
    rb = (C.c_int * max(1, len(src)))(*[t.shape[-1] * t.element_size() for t in src])
    kept = torch.full((seqs, kv, keep), 99, dtype=torch.int32, device="cuda")
    lcu.check(lcu.lib.lcu_cache_evict(arr(dst), arr(src), rb, len(src), weights.data_ptr(), kept.data_ptr(), lengths_out.data_ptr() if lengths_out is not None else None,
                                      lengths.data_ptr(), seqs, kv, ctx, dctx, keep, recent, None))
    torch.cuda.synchronize()
    return kept


@pytest.mark.parametrize("kind", ["ordinary", "equal", "steps", "odd"])
@pytest.mark.parametrize("ctx,lengths,keep,recent", [
    (1, [1, 0], 1, 0), (2, [2, 1], 1, 1), (40, [40, 33, 7, -1], 16, 5), (300, [300, 299, 17], 16, 0), (300, [150, 300], 200, 200), (2048, [2048, 1500], 1024, 256),
    (5000, [5000, 4097], 1, 0), (5000, [4999], 4998, 3), (70000, [70000], 33333, 100), (64, [64, 70], 64, 3),
    (4097, [4097, 1, 4000], 700, 699), (16384, [16384, 12000], 16383, 0), (16385, [16385, 3], 1, 1), (65536, [65536, 40000], 20000, 1), (5000, [5000, 4000, 100, -1] * 7, 1234, 99),
    (17000, [17000, 16000] * 13, 16, 0)])
def test_evict(lcu, kind, ctx, lengths, keep, recent):
    rng = np.random.default_rng(ctx + keep)
    seqs, kv = len(lengths), 3
    w = np.exp(3 * rng.standard_normal((seqs, kv, ctx))).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "steps":
        w = np.floor(w).astype(np.float32)
    elif kind == "odd":
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.2] = -0.0
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.1] = -1.5
    g = torch.Generator(device="cuda").manual_seed(1)
    widths = [64, 8, 2, 4, 48, 6, 256]
    src = [torch.randint(0, 256, (seqs, kv, ctx, n), generator=g, device="cuda", dtype=torch.uint8) for n in widths]
    weights = torch.from_numpy(w).cuda()
    src.append(weights.view(torch.uint8).view(seqs, kv, ctx, 4).clone())
    ln = i32(lengths)
    keep_rows = min(keep + 3, ctx)
    away = [torch.full((seqs, kv, keep_rows, t.shape[-1]), 123, dtype=torch.uint8, device="cuda") for t in src]
    lo = i32([0] * seqs)
    kept = evict(lcu, away, src, weights, ln, ctx, keep_rows, keep, recent, lo)
    here = [t.clone() for t in src]
    lengths_here = ln.clone()
    kept2 = evict(lcu, here, here, weights, lengths_here, ctx, ctx, keep, recent, lengths_here)
    assert torch.equal(kept, kept2) and torch.equal(lo, lengths_here) and lo.tolist() == [min(n, keep, ctx) for n in lengths]
    assert torch.equal(evict(lcu, [], [], weights, ln, ctx, ctx, keep, recent), kept)
    for s in range(seqs):
        for h in range(kv):
            rows = P.evict(w[s, h], min(lengths[s], ctx), keep, recent)
            assert kept[s, h].tolist() == rows + [-1] * (keep - len(rows)), (s, h)
            at = torch.tensor(rows, dtype=torch.long, device="cuda")
            for t, a, b in zip(src, away, here):
                assert torch.equal(a[s, h, :len(rows)], t[s, h, at]) and (a[s, h, len(rows):] == 123).all()
                assert torch.equal(b[s, h, :len(rows)], t[s, h, at]) and torch.equal(b[s, h, len(rows):], t[s, h, len(rows):])


def test_evict_unaligned_planes(lcu):
    """Planes at addresses that only allow narrow copies."""
    rng = np.random.default_rng(3)
    ctx, keep = 500, 200
    w = torch.from_numpy(rng.random((1, 2, ctx)).astype(np.float32)).cuda()
    for off in (2, 4, 8):
        raw = torch.randint(0, 256, (2 * ctx * 64 + 64,), device="cuda", dtype=torch.uint8)
        plane = raw[off:off + 2 * ctx * 64].view(1, 2, ctx, 64)
        was, tail = plane.clone(), raw[off + 2 * ctx * 64:].clone()
        kept = evict(lcu, [plane], [plane], w, i32([ctx]), ctx, ctx, keep, 20).long()
        for h in range(2):
            assert torch.equal(plane[0, h, :keep], was[0, h, kept[0, h]]) and torch.equal(plane[0, h, keep:], was[0, h, keep:])
        assert torch.equal(raw[off + 2 * ctx * 64:], tail)


# ------------------------------------------------------------------ beams
@pytest.mark.parametrize("beams,vocab,n_out", [(1, 50, 6), (1, 4096, 64), (3, 9000, 64), (2, 70000, 17)])
@pytest.mark.parametrize("tiny", [1e-30, 1.0])
def test_beam_logits_whose_difference_a_score_loses(lcu, beams, vocab, n_out, tiny):
    """Equal scores, distinct logits: the lowest beam's, in the order of logits, then of tokens (scores of 1e30 lose any logit)."""
    rng = np.random.default_rng(vocab)
    x = (rng.integers(-300, 300, (1, beams, vocab)) * tiny).astype(np.float32)
    scores = np.full((1, beams), -1.0 if tiny < 1 else -1e30, np.float32)
    parents, tokens, out = lcu.beam_select(x, scores, n_out)
    order = np.lexsort((np.arange(vocab), -x[0, 0]))[:n_out]
    assert (parents == 0).all() and tokens[0].tolist() == order.tolist()
    lse = np.log(np.exp(x[0, 0].astype(np.float64) - x.max()).sum()) + x.max()
    assert np.allclose(out[0], -lse - 1 if tiny < 1 else -1e30, rtol=1e-6)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 50, 6), (1, 4, 4095, 4), (3, 2, 4097, 64), (2, 5, 32000, 10), (1, 32, 12289, 32), (1, 16, 128000, 32)])
def test_beam_select(lcu, dtype, groups, beams, vocab, n_out):
    rng = np.random.default_rng(vocab + n_out)
    x = rng.standard_normal((groups, beams, vocab)).astype(np.float32) * 3
    if dtype == "float32":
        logits = x
        x64 = x.astype(np.float64)
    else:
        logits = P.float_to_bits(x, dtype)
        x64 = P.bits_to_float(logits, dtype)
    scores = (rng.standard_normal((groups, beams)) - 5).astype(np.float32)
    parents, tokens, out = lcu.beam_select(logits, scores, n_out, dtype)
    for g in range(groups):
        p, t, s = P.beam_select(x64[g], scores[g].astype(np.float64), n_out)
        # scores: exponentials within 2^-22 of themselves, sums of sixteen, one rounding of a chunk's sum and of the result
        assert (np.abs(out[g] - s) <= 2.0 ** -19 + U * np.abs(s)).all()
        gaps = np.abs(np.diff(s)).min() if n_out > 1 else 1.0
        ties = n_out > 1 and (np.abs(np.diff(s)) < 1e-6) & (p[1:] != p[:-1])
        if not np.any(ties):
            assert parents[g].tolist() == p.tolist() and tokens[g].tolist() == t.tolist(), (g, gaps)


def test_beam_select_ties_and_numbers_that_are_none(lcu):
    v = 9000
    x = np.zeros((6, 3, v), np.float32)
    scores = np.full((6, 3), -1.0, np.float32)
    x[1, :, :] = -np.inf                       # no token allowed in a beam ...
    x[1, 2, 8000] = 3.0                        # ... but one
    scores[2, 0], scores[2, 1] = -np.inf, np.nan  # unused beams
    x[2, 2, 7] = 1.0
    x[3, 0, 5], x[3, 1, 5] = np.inf, np.nan    # a row without numbers; a logit without
    x[3, 1, 6] = 2.0
    scores[4] = -np.inf                        # nothing to go on with
    x[5, :, ::256] = 1.0                       # equal logits in one thread's places
    scores[5] = [-3.0, -2.0, -3.0]
    for n_out in (1, 3, 6, 40):
        parents, tokens, out = lcu.beam_select(x, scores, n_out)
        for g in range(6):
            x64 = x[g].astype(np.float64)
            p, t, s = P.beam_select(x64, scores[g].astype(np.float64), n_out)
            assert parents[g].tolist() == p.tolist() and tokens[g].tolist() == t.tolist(), (n_out, g)
            fine = np.isfinite(s)
            assert np.array_equal(np.isneginf(out[g]), ~fine) and (np.abs(out[g][fine] - s[fine]) <= 2.0 ** -19 + U * np.abs(s[fine])).all()


def test_beam_select_with_thousands_of_candidates_above_the_bound(lcu):
    """Eight of 32 beams are ahead of all others, so that the bound comes from the 64 threads that own their lists, and one of those has
    nothing in any of its four: nearly all entries of the other 252 lists lie above it."""
    rng = np.random.default_rng(77)
    vocab, beams, n_out = 32 * 4096, 32, 64
    x = rng.standard_normal((1, beams, vocab)).astype(np.float32)
    scores = np.full((1, beams), -100.0, np.float32)
    for b in (0, 1, 8, 9, 16, 17, 24, 25):
        scores[0, b] = 0.01 * b
        if b % 8 == 0:
            x[0, b, :4096] -= 20.0
    parents, tokens, out = lcu.beam_select(x, scores, n_out)
    p, t, s = P.beam_select(x[0].astype(np.float64), scores[0].astype(np.float64), n_out)
    assert np.abs(np.diff(s)).min() > 1e-6  # (nothing that rounding could turn)
    assert parents[0].tolist() == p.tolist() and tokens[0].tolist() == t.tolist() and (np.abs(out[0] - s) <= 2.0 ** -19 + U * np.abs(s)).all()


@pytest.mark.parametrize("groups,beams,kv,ctx,lengths", [
    (1, 1, 2, 5, [5]), (2, 4, 2, 70, [70, 69, 1, 33, 12, 0, -1, 80]), (1, 8, 3, 1000, [1000] * 8), (1, 13, 1, 301, [301] * 13), (1, 32, 1, 64, [40] * 32)])
def test_reorder(lcu, groups, beams, kv, ctx, lengths):
    rng = np.random.default_rng(beams)
    widths = [64, 8, 2, 4, 48, 6, 256]
    n = groups * beams
    src = [torch.randint(0, 256, (n, kv, ctx, w), device="cuda", dtype=torch.uint8) for w in widths]
    raw = torch.randint(0, 256, (n * kv * ctx * 16 + 2,), device="cuda", dtype=torch.uint8)
    src.append(raw[2:].view(n, kv, ctx, 16))  # an address that allows 2-byte copies only
    arr = lambda ts: (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])
    rb = (C.c_int * len(src))(*[t.shape[-1] for t in src])
    tables = [rng.integers(0, beams, (groups, beams)), np.tile(np.arange(beams)[::-1], (groups, 1)), np.roll(np.tile(np.arange(beams), (groups, 1)), 1, 1),
              np.zeros((groups, beams), int), np.where(rng.random((groups, beams)) < 0.5, -1, beams - 1)]
    tables.append(np.full((groups, beams), beams))  # outside: left as they are
    for parents in tables:
        here, away = [t.clone() for t in src[:-1]], [torch.full_like(t, 7) for t in src]
        last = torch.empty_like(raw)
        last.copy_(raw)
        here.append(last[2:].view(n, kv, ctx, 16))
        pr, ln = i32(parents), i32(lengths)
        for dst, frm in ((away, src), (here, here)):
            lcu.check(lcu.lib.lcu_cache_reorder(arr(dst), arr(frm), rb, len(src), pr.data_ptr(), ln.data_ptr(), groups, beams, kv, ctx, None))
        torch.cuda.synchronize()
        for i in range(n):
            parent = parents.ravel()[i]
            ok = 0 <= parent < beams
            frm = i // beams * beams + parent if ok else i
            rows = max(0, min(ctx, lengths[frm])) if ok else 0
            for s, a, h in zip(src, away, here):
                assert torch.equal(a[i, :, :rows], s[frm, :, :rows]) and (a[i, :, rows:] == 7).all()
                assert torch.equal(h[i, :, :rows], s[frm, :, :rows]) and torch.equal(h[i, :, rows:], s[i, :, rows:])


# ------------------------------------------------------------------ together
def test_a_beam_search_over_evicted_4_bit_caches(lcu):
    """Two groups of three beams: a prompt, steps with selection and reordering, an eviction in between, against the definitions step by step
    (the library's own rows are what later attention is held to, as rounding to codes may turn at a border)."""
    groups, beams, kv, heads, hd, bs, ctx, vocab, dtype = 2, 3, 2, 4, 64, 32, 48, 300, "float16"
    n = groups * beams
    rng = np.random.default_rng(11)
    cache = lcu.Cache4(n, kv, hd, ctx, bs, dtype)
    scores = np.where(np.arange(beams) == 0, 0.0, -np.inf)[None].repeat(groups, 0).astype(np.float32)
    tokens_so_far = [[[] for _ in range(beams)] for _ in range(groups)]
    weights = np.zeros((n, kv, ctx))

    def values():
        v = [np.stack([P.bits_to_float(x, dtype) for x in cache.read(ctx)])]
        return v[0][0], v[0][1]

    def attention_step(m):
        q, k, v = (rng.standard_normal((n, m, c * hd)) for c in (heads, kv, kv))
        qb, kb, vb = (P.float_to_bits(a, dtype) for a in (q, k, v))
        q_rot = cache.append(qb, kb, vb)
        out = P.bits_to_float(cache.attend(q_rot), dtype).reshape(n, m, heads, hd)
        kk, vv = values()
        q64 = P.bits_to_float(q_rot, dtype).reshape(n, m, heads, hd)
        for s in range(n):
            held = int(cache.lengths[s])
            # the new rows stand for the rotated keys, within half a step of their scale (which 7 bits put at most 2^-7 above maximum / 7.5)
            at = cache.positions[s] + np.arange(m)
            new = P.rotate(P.bits_to_float(kb[s], dtype).reshape(m, kv, hd), at, 10000.0).transpose(1, 0, 2)
            most = np.repeat(np.abs(new).reshape(kv, m, -1, bs).max(-1), bs, -1)
            assert (np.abs(kk[s, :, held:held + m] - new) <= 0.5 * most / 7.5 * (1 + 2.0 ** -6)).all()
            o, p, spread, big = P.attention(q64[s], kk[s, :, :held + m], vv[s, :, :held + m], held, heads // kv)
            ds = (2 * hd * U * big + 8 * U * (1 + big))[..., None]
            assert (np.abs(out[s] - o) <= P.step_of(dtype) * np.abs(o) + (2.0 ** -11 + 2 * ds + 2.0 ** -20) * spread * 1.01 + 2.0 ** -24).all()
            weights[s, :, held:] = 0
            weights[s, :, :held + m] += p.reshape(kv, -1, m, held + m).sum((1, 2))
            got = cache.planes[4].to_host(np.float32, (n, kv, ctx))[s]
            assert np.allclose(got[:, :held + m], weights[s, :, :held + m], rtol=1e-4, atol=1e-6)
        cache.advance(m)

    attention_step(20)
    for turn in range(30):
        logits = rng.standard_normal((groups, beams, vocab)).astype(np.float32)
        parents, tokens, new = lcu.beam_select(logits, scores, beams)
        for g in range(groups):
            p, t, s = P.beam_select(logits[g].astype(np.float64), scores[g].astype(np.float64), beams)
            assert parents[g].tolist() == p.tolist() and tokens[g].tolist() == t.tolist()
        scores = new
        before = values()
        lengths = cache.lengths.copy()
        cache.reorder(parents)
        at = (np.arange(groups)[:, None] * beams + parents).ravel()
        for a, b in zip(values(), before):
            for s in range(n):
                assert np.array_equal(a[s, :, :lengths[at[s]]], b[at[s], :, :lengths[at[s]]])
        weights = weights[at].copy()
        if cache.lengths.max() == ctx:
            got = cache.planes[4].to_host(np.float32, (n, kv, ctx))
            kept = cache.evict(24, 6)
            for s in range(n):
                for h in range(kv):
                    rows = P.evict(got[s, h], ctx, 24, 6)
                    assert kept[s, h].tolist() == rows
                    weights[s, h, :24] = weights[s, h, rows]
            assert (cache.lengths == 24).all() and (cache.positions == 48 + (turn > 30) * 24).all()
        attention_step(1)
