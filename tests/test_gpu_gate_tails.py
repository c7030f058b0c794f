"""The gated feed-forward block where its activation is nearly 0: gates far below it, against 64 bits."""
import math

import numpy as np
import pytest

from batch_ops import E4M3
from memvanta_amd import capi

pytestmark = pytest.mark.gpu

F = np.float32
EPS = 2.0 ** -24  # half a step of fp32, relative


def _tensor(ctx, codes, scales):
    return ctx.upload("w", capi.MVH_TYPE_FP8_B128, codes.shape[1], codes.shape[0],
                      np.concatenate([codes.ravel(), scales.ravel().view(np.uint8)]))


def _run(ctx, batch, act, gates, u_size):
    """Gates -(448 or 336) 2^-9 |value of a code| gates, exactly, and ups u_size: each a single product.  (outputs, g, u)"""
    n, k = 640, 256
    col = np.zeros((n, k), np.uint8)
    col[:, 3] = np.arange(n) % 126 + 1
    one = np.zeros((n, k), np.uint8)
    one[:, 130] = 0x38  # 1
    x = np.zeros((batch, k), F)
    x[:, 3] = -np.where(np.arange(batch) % 2, 336, 448) * 2.0 ** -9
    x[:, 130] = 448
    tg = _tensor(ctx, col, np.full((n // 128, 2), gates, F))
    tu = _tensor(ctx, one, np.full((n // 128, 2), u_size / 448, F))
    y = ctx.gated_ffn_fp8(tg, tu, x, act)
    tg.free()
    tu.free()
    g = x[:, 3:4].astype(np.float64) * (E4M3[col[:, 3]] * gates)[None]
    return y, g, np.float64(F(u_size / 448)) * 448


BATCHES = [1, 3, 20, 60, 150, 2000]


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("gates", [0.5, 1.0])
def test_gelu(ctx, batch, gates):
    """g / sqrt(2) is off by two roundings, of the factor and of the product, which a result feels g^2 + 2 times; erfc by up to
    16 steps; three more roundings."""
    y, g, u = _run(ctx, batch, capi.MVH_GATE_GELU, gates, 2.0 ** 20)
    some = g > -12.5  # beyond, the activation is below fp32's normal numbers
    assert (g[some] < -5).any()
    want = 0.5 * g * np.vectorize(math.erfc)(-g / math.sqrt(2)) * u
    err = (2 * (g * g + 2) + 2 * 16 + 3) * EPS * np.abs(want) + 2.0 ** -149 * u
    assert (np.abs(y - want) <= err)[some].all(), np.abs((y - want) / want)[some].max()
    assert (y[~some] <= 0).all() and (np.abs(y[~some]) <= 1e-28).all()


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("gates", [0.5, 127 / 128])
def test_silu(ctx, batch, gates):
    """Down to where the activation is no normal number, -92: e^-g alone is beyond fp32 from -88.8 on.  16 steps for the
    exponential and its square, and as many for the quotient and products."""
    y, g, u = _run(ctx, batch, capi.MVH_GATE_SILU, gates, 2.0 ** 100)
    some = g > -91
    assert (g[some] < (-84, -89)[gates > 0.5] + 1).any()
    e = np.exp(np.maximum(g, -300))
    want = g * e / (1 + e) * u
    err = 32 * 2 * EPS * np.abs(want)
    assert (np.abs(y - want) <= err)[some].all(), np.abs((y - want) / want)[some].max()
    assert (y[~some] <= 0).all() and (np.abs(y[~some]) <= 2.0 ** -124 * u).all()


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("act", [capi.MVH_GATE_SILU, capi.MVH_GATE_GELU])
def test_infinite_gates(ctx, batch, act):
    """A gate beyond fp32's numbers has its activation's limit: 0 below, itself above."""
    n, k = 200, 128
    codes = np.zeros((n, k), np.uint8)
    codes[:, 0] = np.where(np.arange(n) % 2, 0x7e, 0xfe)  # +-448
    ups = np.zeros((n, k), np.uint8)
    ups[:, 0] = 0x38
    x = np.zeros((batch, k), F)
    x[:, 0] = F(2.0 ** 110)
    tg, tu = _tensor(ctx, codes, np.full((2, 1), 2.0 ** 60, F)), _tensor(ctx, ups, np.full((2, 1), 2.0 ** -110, F))
    y = ctx.gated_ffn_fp8(tg, tu, x, act)
    assert (y[:, ::2] == 0).all() and (y[:, 1::2] == np.inf).all()
    tg.free()
    tu.free()
