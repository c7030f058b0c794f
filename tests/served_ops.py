"""Plain restatements of the served token's operators, in 64 bits where no format says otherwise."""
import math

import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def angles(rot, base=10000.0, scaling=0, factor=1.0, orig_ctx=0.0, low=0.0, high=0.0):
    """Angle per position of each pair; scaling as MVH_ROPE_SCALE_*."""
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == 0:
            keep = 1.0
        elif scaling == 1:
            keep = 0.0
        elif scaling == 2:
            keep = min(max((orig_ctx * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
        else:
            a, b = (rot / 2 * math.log(orig_ctx / (2 * math.pi * t)) / math.log(base) for t in (high, low))
            a, b = max(math.floor(a), 0), min(math.ceil(b), rot - 1)
            keep = 1.0 - min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
        out.append(f * keep + f / factor * (1.0 - keep))
    return np.array(out)


def rotate(x, positions, f, rot, interleaved, scale=1.0):
    """x [tokens][heads][hd] rotated in 64 bits, and the largest error that the 32-bit steps can make: cos and sin
    rounded, two products and a sum rounded."""
    x = x.astype(np.float64)
    t = np.asarray(positions, np.float64)[:, None, None] * f
    c, s = scale * np.cos(t), scale * np.sin(t)
    y, err = x.copy(), np.zeros_like(x)
    i0 = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    i1 = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    err[..., i0] = EPS * (2 * (abs(x0 * c) + abs(x1 * s)) + abs(y[..., i0]))
    err[..., i1] = EPS * (2 * (abs(x0 * s) + abs(x1 * c)) + abs(y[..., i1]))
    # a cosine or sine near 0 is off by its angle's last place: 4 roundings of 2^-53 of the angle
    far = 4 * 2.0 ** -53 * abs(t) * scale * (abs(x0) + abs(x1))
    err[..., i0] += far
    err[..., i1] += far
    return y, 1.001 * err + 1e-30


def q4_values(x):
    """The values a 4-bit cache holds for rows x: the format's steps, each rounded to 32 bits."""
    x = np.ascontiguousarray(x, np.float32)
    b = x.reshape(x.shape[0], -1, 32)
    f = np.float32
    with np.errstate(all="ignore"):
        lo, hi = b.min(axis=2), b.max(axis=2)
        s = np.minimum((hi - lo) / f(15), f(512)).astype(np.float16).astype(f)
        c = np.clip(lo + f(8) * s, f(-65504), f(65504)).astype(np.float16).astype(f)
        n = np.clip(np.rint((b - c[..., None]) / s[..., None]) + f(8), f(0), f(15))
        n = np.where(s[..., None] > 0, n, f(8))
        v = s[..., None] * (n - f(8)) + c[..., None]
    v = np.where(np.isfinite(b).all(axis=2)[..., None], v, f(np.nan))
    return v.reshape(x.shape)


def attend(q, k, v, pos, group):
    """Causal attention of tokens at pos.. in 64 bits: q [tokens][heads][hd], k and v [rows][kv heads][hd]."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    out = np.empty_like(q)
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // group].T / math.sqrt(q.shape[2])
        for t in range(q.shape[0]):
            r = s[t, : pos + t + 1]
            w = np.exp(r - r.max())
            out[t, h] = w @ v[: pos + t + 1, h // group] / w.sum()
    return out


def log_softmax(x):
    x = x.astype(np.float64)
    m = x.max(axis=1, keepdims=True)
    with np.errstate(divide="ignore"):
        return x - m - np.log(np.exp(x - m).sum(axis=1, keepdims=True))
