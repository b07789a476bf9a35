"""The 4-bit cache, attention over it, eviction, beam selection and reordering from their definitions, in binary64 (numpy)."""
import numpy as np


def bits_to_float(u, dtype):
    u = np.asarray(u, np.uint16)
    return u.view(np.float16).astype(np.float64) if dtype == "float16" else (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def float_to_bits(x, dtype):
    """Round to nearest even."""
    x = np.asarray(x, np.float32)
    if dtype == "float16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def step_of(dtype):
    """Largest relative error of one rounding."""
    return 2.0 ** -11 if dtype == "float16" else 2.0 ** -8


def seven_bits(s):
    m, e = np.frexp(s)
    return np.ldexp(np.rint(m * 128) / 128, e)


def scales_of(x, bs):
    """Scales [..., hd / bs] of rows x, a NaN for a block with a number that is not finite."""
    b = np.abs(x.reshape(*x.shape[:-1], -1, bs))
    a = np.where(np.isfinite(b).all(-1), np.where(np.isfinite(b), b, 0).max(-1), np.nan)
    # (the quotient is a binary32 number: the seven bits of a tie are those of what is rounded first)
    return np.minimum(seven_bits((a.astype(np.float32) / np.float32(7.5)).astype(np.float64)), 8704.0).astype(np.float16)


def codes_of(x, scales, bs):
    s = np.repeat(scales.astype(np.float32), bs, -1)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        c = np.clip(np.floor(x.astype(np.float32) / s + np.float32(8)), 0, 15)
    return np.where(s > 0, c, 8).astype(np.uint8)


def values_of(codes, scales, bs):
    return (codes.astype(np.float64) - 7.5) * np.repeat(scales.astype(np.float64), bs, -1)


def places(hd):
    """Nibble (0 ..) of a row's bytes for every dimension."""
    d = np.arange(hd)
    return ((d % 32) // 8 * (hd // 32) + d // 32) * 8 + d % 8


def pack(codes):
    hd = codes.shape[-1]
    nib = np.zeros_like(codes)
    nib[..., places(hd)] = codes
    return nib[..., 0::2] | nib[..., 1::2] << 4


def unpack(raw):
    nib = np.stack((raw & 15, raw >> 4), -1).reshape(*raw.shape[:-1], -1)
    return nib[..., places(nib.shape[-1])]


def rotate(x, positions, theta):
    """x [rows, heads, hd], neighbouring pairs."""
    if theta == 0:
        return x
    hd = x.shape[-1]
    a = np.asarray(positions, np.float64)[:, None, None] * np.float64(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(a), np.sin(a)
    return np.stack((x[..., 0::2] * c - x[..., 1::2] * s, x[..., 0::2] * s + x[..., 1::2] * c), -1).reshape(x.shape)


def attention(q, k, v, held, group):
    """q [m, heads, hd], k, v [kv, rows, hd] of one sequence: outputs, probabilities [heads, m, rows], and the spreads a tolerance needs:
    sum p |v| and the largest sum |q k| / sqrt(hd) over the keys seen."""
    m, heads, hd = q.shape
    rows = k.shape[1]
    out, spread, big = np.zeros((m, heads, hd)), np.zeros((m, heads, hd)), np.zeros((m, heads))
    p = np.zeros((heads, m, rows))
    for i in range(m):
        n = min(rows, held + i + 1)
        if held < 0 or n <= 0:
            continue
        for h in range(heads):
            kk, vv = k[h // group, :n], v[h // group, :n]
            s = kk @ q[i, h] / np.sqrt(hd)
            e = np.exp(s - s.max())
            p[h, i, :n] = e / e.sum()
            out[i, h] = p[h, i, :n] @ vv
            spread[i, h] = p[h, i, :n] @ np.abs(vv)
            big[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(hd)
    return out, p, spread, big


def evict(weights, length, keep, recent):
    """Rows kept, in order (lists may be shorter than keep)."""
    if length <= keep:
        return list(range(max(0, length)))
    w = np.where(np.isnan(weights[:length - recent]), -np.inf, weights[:length - recent] + 0.0)
    nan = np.isnan(weights[:length - recent])
    order = sorted(range(length - recent), key=lambda j: (-w[j], nan[j], j))  # (a NaN comes behind minus infinity)
    return sorted(order[:keep - recent]) + list(range(length - recent, length))


def beam_select(logits, scores, n_out):
    """One group: logits [beams, vocab], scores [beams] -> parents, tokens, scores (binary64)."""
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    top = x.max(-1)
    total = np.full(x.shape, -np.inf)
    for b in range(len(x)):
        if np.isfinite(top[b]) and np.isfinite(scores[b]):
            total[b] = x[b] - (np.log(np.exp(x[b] - top[b]).sum()) + top[b]) + scores[b]
    flat = total.ravel()
    order = np.argsort(-flat, kind="stable")[:n_out]
    return order // x.shape[1], order % x.shape[1], flat[order]
