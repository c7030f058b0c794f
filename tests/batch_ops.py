"""Plain restatements of a served batch's operators: 8-bit floating point weights and attention behind a shared prefix, in
64 bits where no format says otherwise."""
import math

import numpy as np

STEP = 2.0 ** -23  # a step of fp32, relative: the error of an addition that cuts instead of rounding

_half = np.arange(128)
_mag = np.where(_half >> 3 == 0, (_half & 7) * 2.0 ** -9, (8 + (_half & 7)) * 2.0 ** ((_half >> 3) - 10.0))
_mag[127] = np.nan
E4M3 = np.concatenate([_mag, -_mag])  # the value of each code


def to_e4m3(z):
    """Codes of float32 values up to 464 (and NaN), ties to even."""
    z = np.asarray(z, np.float32)
    a = np.abs(z).astype(np.float64)
    with np.errstate(invalid="ignore"):
        at = np.searchsorted(_mag[:127], a)  # the first value >= a
        lo, hi = np.clip(at - 1, 0, 126), np.clip(at, 0, 126)
        up = _mag[hi] - a < a - _mag[lo]
        tie = _mag[hi] - a == a - _mag[lo]
        code = np.where(up | (tie & (hi % 2 == 0)), hi, lo)
        code = np.where(np.isnan(a), 127, code)
    return (code | np.where(np.signbit(z), 128, 0)).astype(np.uint8)


def quantize(x, block_rows=1):
    """(codes, scales) by the format's steps, each rounded to 32 bits."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    f = np.float32
    p = np.zeros((-(-rows // block_rows) * block_rows, -(-cols // 128) * 128), f)
    p[:rows, :cols] = x
    b = p.reshape(p.shape[0] // block_rows, block_rows, -1, 128)
    with np.errstate(all="ignore"):
        s = np.abs(b).max(axis=(1, 3)) / f(448)
        s = np.where(s < f(2.0 ** -126), f(0), s).astype(f)
        inv = np.where(s == 0, f(0), f(1) / s).astype(f)
        z = b * inv[:, None, :, None]
    return to_e4m3(z).reshape(p.shape)[:rows, :cols], s


def spread(scales, rows, cols, block_rows):
    return np.repeat(np.repeat(scales, block_rows, 0)[:rows], 128, 1)[:, :cols]


def values(codes, scales, block_rows):
    with np.errstate(invalid="ignore"):
        return E4M3[codes] * spread(scales.astype(np.float64), *codes.shape, block_rows)


def product(x, codes, scales):
    """x w^T of the quantised x in 64 bits, and how far fp32 sums can be off: 128 additions in a block, one a block and a
    rounded scale, none of them off by more than a step of the sum of magnitudes."""
    qx = values(*quantize(x), 1)
    w = values(codes, scales, 128)
    blocks = -(-x.shape[1] // 128)
    return qx @ w.T, (130 + blocks) * STEP * (np.abs(qx) @ np.abs(w).T)


def gate(g, act):
    """act(g) and the largest |act'|, which is below 1.13 for either."""
    if act == 0:
        with np.errstate(over="ignore"):
            return g / (1 + np.exp(-g))
    return 0.5 * g * (1 + np.vectorize(math.erf)(g / math.sqrt(2)))


def gated(x, wg, wu, act):
    g, eg = product(x, *wg)
    u, eu = product(x, *wu)
    a = gate(g, act)
    # act itself: a handful of roundings of it, and of g where 1 + erf cancels
    ea = 1.13 * eg + 8 * STEP * np.abs(a) + 4 * STEP * np.abs(g)
    return a * u, ea * np.abs(u) + np.abs(a) * eu + ea * eu + STEP * np.abs(a * u)


def attend_shared(q, prefix, own, pos, n_tokens, heads, kv_heads):
    """Attention in 64 bits: prefix (k, v) [rows][kv_heads * hd], own the same per sequence (rows from the prefix's end on);
    also the sum of the magnitudes that an output adds up."""
    hd = q.shape[1] // heads
    cut = lambda x: x.astype(np.float64).reshape(len(x), kv_heads, hd)
    q = q.astype(np.float64).reshape(len(q), heads, hd)
    out, size = np.empty_like(q), np.empty_like(q)
    row, (pk, pv) = 0, map(cut, prefix)
    for (k, v), p, n in zip(own, pos, n_tokens):
        k, v = np.concatenate([pk, cut(k)]), np.concatenate([pv, cut(v)])
        for t in range(n):
            end = p + t + 1
            for h in range(heads):
                g = h // (heads // kv_heads)
                s = k[:end, g] @ q[row, h] / math.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                with np.errstate(invalid="ignore"):
                    out[row, h], size[row, h] = w @ v[:end, g], w @ np.abs(v[:end, g])
            row += 1
    return out.reshape(len(q), -1), size.reshape(len(q), -1)
