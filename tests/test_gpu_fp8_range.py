"""Products on 8-bit floating point weights whose scales' product leaves fp32's normal numbers while the result does not."""
import numpy as np
import pytest

from batch_ops import STEP, product, quantize
from memvanta_amd import capi

pytestmark = pytest.mark.gpu

F = np.float32
TOP = float(np.finfo(F).max)
# batch, K, N: x quantised in the kernel, rows of 16 weights, tiles of 64 x 64, in parts, of 64 x 128, of 128 x 128
SHAPES = [(1, 400, 384), (3, 400, 384), (20, 400, 384), (60, 400, 384), (150, 400, 384), (70, 4096, 384), (333, 2048, 2560),
          (1100, 272, 9088)]


def _tensor(ctx, codes, scales):
    return ctx.upload("w", capi.MVH_TYPE_FP8_B128, codes.shape[1], codes.shape[0],
                      np.concatenate([codes.ravel(), scales.ravel().view(np.uint8)]))


def _sizes(rng, batch, k, n, sizes):
    """x of rows and weights of blocks of rows that are sizes[i] as large as ordinary ones, all positive, so that no sum is larger
    than the result; every seventh row of weights zeros."""
    x = np.abs(rng.standard_normal((batch, k))).astype(F)
    codes, scales = quantize(np.abs(rng.standard_normal((n, k))).astype(F), 128)
    codes = codes.copy()
    codes[::7] = 0
    pick = rng.integers(0, len(sizes), batch)
    pick[: min(batch, len(sizes))] = np.arange(min(batch, len(sizes)))
    x *= np.array([a for a, _ in sizes], F)[pick, None]
    return x, codes, scales * np.array([w for _, w in sizes], F)[np.arange(len(scales)) % len(sizes), None]


def _check(got, want, err, blocks):
    """err: what rounding may do, of numbers that fp32 holds; of subnormal ones a step each time."""
    g, w = np.clip(got.astype(np.float64), -TOP, TOP), np.clip(want, -TOP, TOP)
    off = np.abs(g - w) - err - (130 + blocks) * 2.0 ** -149
    assert not np.isnan(got).any()
    assert (off <= 0).all(), (off.max(), np.argwhere(off > 0)[:3])
    assert (want == 0).any() and (got[want == 0] == 0).all()


@pytest.mark.parametrize("batch,k,n", SHAPES)
# products of scales about 2^-126 to 2^-149, below, 2^128 to 2^140, far above, and both ends at once
@pytest.mark.parametrize("sizes", [[(2.0 ** -109, 2.0 ** -20), (2.0 ** -60, 2.0 ** -76)], [(2.0 ** -100, 2.0 ** -45), (2.0 ** -40, 2.0 ** -120)],
                                   [(2.0 ** 100, 2.0 ** 22), (2.0 ** 20, 2.0 ** 110)], [(2.0 ** 120, 2.0 ** 120), (2.0 ** 60, 2.0 ** 90)],
                                   [(2.0 ** 118, 2.0 ** -125), (2.0 ** -109, 2.0 ** 112), (1.0, 1.0)],
                                   [(2.0 ** -109, 2.0 ** -25), (2.0 ** 100, 2.0 ** 30), (1.0, 1.0)]])
def test_products(ctx, batch, k, n, sizes):
    x, codes, scales = _sizes(np.random.default_rng(k + batch), batch, k, n, sizes)
    t = _tensor(ctx, codes, scales)
    want, err = product(x, codes, scales)
    _check(ctx.matmul_fp8(t, x), want, err, -(-k // 128))
    t.free()


@pytest.mark.parametrize("batch,k,n", SHAPES)
def test_gated(ctx, batch, k, n):
    """The second product's scales alone: act(g) of ordinary size, u small or large."""
    rng = np.random.default_rng(k + batch)
    gate = quantize(rng.standard_normal((n, k)).astype(F), 128)
    for size, more in ((2.0 ** -100, 2.0 ** -40), (2.0 ** 90, 2.0 ** 45)):
        x, codes, scales = _sizes(rng, batch, k, n, [(size, more)])
        g_scales = (gate[1] * F(2.0 ** 6 / size / k ** 0.5)).astype(F)
        tg, tu = _tensor(ctx, gate[0], g_scales), _tensor(ctx, codes, scales)
        g, eg = product(x, gate[0], g_scales)
        u, eu = product(x, codes, scales)
        a = g / (1 + np.exp(-np.clip(g, -700, 700)))
        # silu's slope is below 1.13; its own error a handful of roundings, and where e^-g is beyond fp32 it is 0, less than 2^-121
        ea = 1.13 * eg + 8 * STEP * np.abs(a) + 2.0 ** -121
        err = ea * np.abs(u) + np.abs(a) * eu + ea * eu + STEP * np.abs(a * u) + (130 + -(-k // 128)) * 2.0 ** -149 * (1 + np.abs(a))
        got, want = ctx.gated_ffn_fp8(tg, tu, x), a * u
        held = (np.abs(u) + eu < TOP) & (np.abs(want) + err < TOP)
        assert held.mean() > 0.1
        assert (np.abs(got.astype(np.float64) - want) <= err)[held].all()
        assert (got[(u == 0) & (np.abs(g) < 1e30)] == 0).all()
        tg.free()
        tu.free()


@pytest.mark.parametrize("batch", [1, 3, 20, 60, 150, 2000])
def test_small_codes(ctx, batch):
    """Scales whose product is 2^132 or 2^-132, and sums of 2^-18 to 2^17 on them."""
    k, n = 256, 640
    for sx, sw in ((60, 72), (72, 60), (118, 14), (-60, -72), (-116, -16), (-10, -122)):
        x = np.zeros((batch, k), F)
        x[:, 128] = 448 * 2.0 ** sx  # against codes of 0: it sets the scale alone
        x[np.arange(batch), 129 + np.arange(batch) % 5] = np.array([1, 2, 5, 7, 448 * 512])[np.arange(batch) % 5] * 2.0 ** (sx - 9)
        codes = np.zeros((n, k), np.uint8)
        codes[np.arange(n), 129 + np.arange(n) % 5] = np.array([1, 3, 8, 60, 126])[np.arange(n) // 5 % 5]
        scales = np.full((n // 128, 2), 2.0 ** sw, F)
        t = _tensor(ctx, codes, scales)
        want, _ = product(x, codes, scales)
        got = ctx.matmul_fp8(t, x)
        # one product a sum: rounded once
        with np.errstate(over="ignore"):
            w = want.astype(F)
        assert (got == w).all(), (sx, sw, np.argwhere(got != w)[:3])
        t.free()
