"""Weights in 8-bit floating point: quantisation bit for bit, products and the gated feed-forward block against 64 bits,
and their refusals."""
import numpy as np
import pytest

from batch_ops import gated, product, quantize, to_e4m3
from memvanta_amd import capi, synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F = np.float32


def _tensor(ctx, codes, scales):
    return ctx.upload("w", capi.MVH_TYPE_FP8_B128, codes.shape[1], codes.shape[0],
                      np.concatenate([codes.ravel(), scales.ravel().view(np.uint8)]))


def _rows(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
    x[:, rng.integers(0, cols, max(1, cols // 64))] *= 16
    return x.astype(F)


def _weights(rng, n, k):
    return quantize((rng.standard_normal((n, k)) * 0.02 * np.exp(rng.uniform(-1, 1, (n, 1)))).astype(F), 128)


def _check(got, want, err):
    assert got.shape == want.shape
    off = np.abs(got.astype(np.float64) - want) - err
    assert (off <= 0).all(), (float(off.max()), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (5, 144), (130, 400), (257, 2048)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(ctx, rows, cols, block_rows):
    x = _rows(np.random.default_rng(rows), rows, cols)
    x[rows // 2, : min(cols, 128)] = 0
    codes, scales = ctx.quantize_fp8(x, block_rows)
    want, want_s = quantize(x, block_rows)
    assert (scales.view(np.uint32) == want_s.view(np.uint32)).all()
    assert (codes == want).all()


def test_quantize_every_rounding(ctx):
    """A scale of 1: every code, the middle between each two and the numbers next to it."""
    from batch_ops import E4M3
    v = E4M3[:127].astype(F)
    mid = ((v[1:].astype(np.float64) + v[:-1]) / 2).astype(F)
    z = np.concatenate([v, mid, np.nextafter(mid, F(0)), np.nextafter(mid, F(500))])
    z = np.concatenate([z, -z])
    rows = np.zeros((-(-len(z) // 127), 128), F)
    for i in range(len(rows)):
        part = z[127 * i:127 * i + 127]
        rows[i, : len(part)] = part
        rows[i, 127] = 448
    codes, scales = ctx.quantize_fp8(rows)
    assert (scales == 1).all()
    assert (codes == to_e4m3(rows)).all()


def test_quantize_extremes(ctx):
    """Blocks of one size each, from numbers without a normal scale to the largest; infinities and NaN."""
    rng = np.random.default_rng(3)
    x = rng.uniform(-1, 1, (1, 128 * 12)).astype(F).reshape(12, 128)
    size = np.array([0, 1e-45, 1e-38, 5.2e-36, 5.4e-36, 1e-30, 1e-3, 1, 1e10, 1e38, 3.4e38, 1], F)
    with np.errstate(under="ignore"):
        x = x * size[:, None]
    x[11, 5], x[6, 77] = np.inf, np.nan
    codes, scales = ctx.quantize_fp8(x.reshape(1, -1))
    want, want_s = quantize(x.reshape(1, -1))
    assert (np.isnan(scales) == np.isnan(want_s)).all()
    fine = np.isfinite(want_s[0])
    assert (scales[0, fine] == want_s[0, fine]).all() and fine.sum() == 10 and scales[0, 11] == np.inf
    assert (codes.reshape(12, 128)[fine] == want.reshape(12, 128)[fine]).all()
    assert codes.reshape(12, 128)[11, 5] & 127 == 127 and (codes.reshape(12, 128)[6] & 127 == 127).all()


SHAPES = [(1, 16, 1), (1, 128, 17), (2, 144, 16), (7, 48, 129), (8, 4096, 64), (16, 272, 127), (17, 1024, 300), (33, 400, 33),
          (64, 288, 768), (65, 128, 128), (129, 656, 257), (130, 2048, 15), (300, 144, 515), (513, 384, 640),
          (3, 2064, 50), (2, 11008, 40), (40, 5632, 130), (60, 1040, 2100), (70, 8192, 90), (200, 4112, 1030), (700, 1040, 1030)]


@pytest.mark.parametrize("batch,k,n", SHAPES)
def test_matmul(ctx, batch, k, n):
    rng = np.random.default_rng(batch + k)
    w, x = _weights(rng, n, k), _rows(rng, batch, k)
    t = _tensor(ctx, *w)
    _check(ctx.matmul_fp8(t, x), *product(x, *w))
    t.free()


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("batch,k,n", SHAPES)
def test_gated_ffn(ctx, batch, k, n, act):
    rng = np.random.default_rng(batch + k + act)
    wg, wu, x = _weights(rng, n, k), _weights(rng, n, k), _rows(rng, batch, k)
    tg, tu = _tensor(ctx, *wg), _tensor(ctx, *wu)
    _check(ctx.gated_ffn_fp8(tg, tu, x, act), *gated(x, wg, wu, act))
    tg.free()
    tu.free()


@pytest.mark.parametrize("batch,k,n", [(1, 11008, 4096), (8, 2048, 32000), (20, 5632, 2048), (64, 4096, 11008),
                                       (333, 2048, 2560), (24, 4096, 32000), (129, 11008, 4097), (1100, 1024, 9000)])
def test_large(ctx, batch, k, n):
    """Sizes of the models, against 64 bits on the GPU's own double products."""
    rng = np.random.default_rng(n)
    x = _rows(rng, batch, k)
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * 0.02).numpy()
    t = ctx.upload_fp8("w", w)
    codes, scales = ctx.quantize_fp8(w, 128)
    from batch_ops import STEP, values
    xd = torch.from_numpy(values(*quantize(x), 1)).cuda()
    wd = torch.from_numpy(codes).cuda().view(torch.float8_e4m3fn).double()
    wd *= torch.from_numpy(scales).cuda().double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want, size = (xd @ wd.T.contiguous()).cpu().numpy(), (xd.abs() @ wd.abs().T.contiguous()).cpu().numpy()
    _check(ctx.matmul_fp8(t, x), want, (130 + -(-k // 128)) * STEP * size)
    t.free()


@pytest.mark.parametrize("batch", [1, 5, 40, 140])
def test_nan_stays_in_its_row_and_column(ctx, batch):
    """A NaN code of the weights makes its output column NaN, a NaN or infinity of x its token's row, and no other."""
    rng = np.random.default_rng(batch)
    k, n = 400, 200
    codes, scales = _weights(rng, n, k)
    codes = codes.copy()
    codes[37, 399] = 127
    x = _rows(rng, batch, k)
    x[batch // 2, 3] = np.nan if batch % 2 else np.inf
    t = _tensor(ctx, codes, scales)
    y = ctx.matmul_fp8(t, x)
    bad = np.zeros((batch, n), bool)
    bad[:, 37] = True
    bad[batch // 2] = True
    assert (np.isnan(y) == bad).all()
    t.free()


def test_device_rows_and_what_lies_around(ctx):
    """Device buffers: the rows given are read and written, nothing else."""
    rng = np.random.default_rng(9)
    for batch in (1, 3, 50, 150):
        k, n = 272, 130
        w, x = _weights(rng, n, k), _rows(rng, batch, k)
        t = _tensor(ctx, *w)
        big = torch.full((batch + 2, n), 7.0, device="cuda")
        xd = torch.full((batch + 2, k), float("nan"), device="cuda")
        xd[1:-1] = torch.from_numpy(x).cuda()
        torch.cuda.synchronize()
        ctx.matmul_fp8(t, xd[1:-1], big[1:-1])
        ctx.synchronize()
        y = big.cpu().numpy()
        assert (y[[0, -1]] == 7).all()
        assert (y[1:-1] == ctx.matmul_fp8(t, x)).all()
        t.free()


@pytest.mark.parametrize("batch,k,n", [(4, 8192, 100), (3, 10912, 1000), (4, 8192, 4100)])
def test_most_rows_quantised_in_the_kernel(ctx, batch, k, n):
    """Up to 32768 elements of x are held in LDS beside the waves' sums."""
    rng = np.random.default_rng(n)
    wg, wu, x = _weights(rng, n, k), _weights(rng, n, k), _rows(rng, batch, k)
    tg, tu = _tensor(ctx, *wg), _tensor(ctx, *wu)
    _check(ctx.gated_ffn_fp8(tg, tu, x, 0), *gated(x, wg, wu, 0))
    tg.free()
    tu.free()


@pytest.mark.parametrize("batch,k,n", [(3, 128, 64), (20, 256, 64), (70, 128, 260), (70, 8192, 256), (200, 2048, 512)])
def test_results_at_any_float(ctx, batch, k, n):
    """y needs a float's alignment only, also where rows of it are stored 16 bytes at a time."""
    rng = np.random.default_rng(n)
    w, x = _weights(rng, n, k), _rows(rng, batch, k)
    t = _tensor(ctx, *w)
    xd, flat = torch.from_numpy(x).cuda(), torch.full((batch * n + 8,), 7.0, device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_fp8(t, xd, flat[3:-5].reshape(batch, n))
    ctx.synchronize()
    got = flat.cpu().numpy()
    assert (got[:3] == 7).all() and (got[-5:] == 7).all()
    assert (got[3:-5].reshape(batch, n) == ctx.matmul_fp8(t, x)).all()
    t.free()


def test_empty(ctx):
    t = _tensor(ctx, *_weights(np.random.default_rng(0), 20, 32))
    assert ctx.matmul_fp8(t, np.zeros((0, 32), F)).shape == (0, 20)
    t.free()


def test_captured(ctx):
    """A call whose workspace is there is captured and replayed, with eager calls of other sizes between the replays."""
    rng = np.random.default_rng(4)
    own = capi.Context(0)
    w, wu = _weights(rng, 300, 400), _weights(rng, 300, 400)
    tg, tu = _tensor(own, *w), _tensor(own, *wu)
    stream = torch.cuda.ExternalStream(own.stream)
    for batch in (1, 70):
        x, y = torch.zeros((batch, 400), device="cuda"), torch.zeros((batch, 300), device="cuda")
        torch.cuda.synchronize()
        own.gated_ffn_fp8(tg, tu, x, 0, y)
        own.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            own.gated_ffn_fp8(tg, tu, x, 0, y)
        for i in range(4):
            rows = _rows(rng, batch, 400)
            x.copy_(torch.from_numpy(rows))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = y.cpu().numpy()
            assert (got == own.gated_ffn_fp8(tg, tu, rows)).all(), i
            own.matmul_fp8(tg, _rows(rng, 200, 400))  # a larger workspace
    tg.free()
    tu.free()
    own.close()


def test_profiled(ctx):
    t = _tensor(ctx, *_weights(np.random.default_rng(0), 64, 128))
    t2 = ctx.upload_fp8("blk.3.ffn_up.weight", np.ones((64, 128), F))
    capi.profile_reset()
    capi.profile_enable(True)
    ctx.matmul_fp8(t2, np.ones((3, 128), F))
    ctx.gated_ffn_fp8(t, t2, np.ones((2, 128), F))
    capi.profile_enable(False)
    got = [(e["tensor"], e["calls"], e["batch"]) for e in capi.profile_snapshot()]
    capi.profile_reset()
    assert got == [("blk.3.ffn_up.weight", 1, 3), ("w+blk.3.ffn_up.weight", 1, 2)]
    t.free()
    t2.free()


def test_refusals(ctx):
    rng = np.random.default_rng(0)
    t, t2 = _tensor(ctx, *_weights(rng, 20, 32)), _tensor(ctx, *_weights(rng, 20, 48))
    x = np.zeros((2, 32), F)
    q4 = ctx.upload("q", synth.Q4_0, 32, 4, synth.quantize_q4_0(rng.standard_normal((4, 32)).astype(F)))
    with pytest.raises(capi.MvhError, match="needs a FP8 tensor"):
        ctx.matmul_fp8(q4, np.zeros((2, 32), F))
    with pytest.raises(capi.MvhError, match="differ in shape"):
        ctx.gated_ffn_fp8(t, t2, x)
    with pytest.raises(capi.MvhError, match="gate activation"):
        ctx.gated_ffn_fp8(t, t, x, 2)
    for call in (lambda: ctx.matvec(t, x[0]), lambda: ctx.matmul_batch(t, x), lambda: ctx.matmul_batch_v06(t, x),
                 lambda: ctx.read_row(t, 0), lambda: ctx.matmul_q4_0_batch(t, x)):
        with pytest.raises(capi.MvhError, match="FP8"):
            call()
    with pytest.raises(capi.MvhError, match="multiple of 16"):
        ctx.quantize_fp8(np.zeros((2, 40), F))
    with pytest.raises(capi.MvhError, match="block_rows"):
        ctx.quantize_fp8(np.zeros((2, 32), F), 64, np.zeros(64, np.uint8), np.zeros(2, F))
    for shape, size in (((40, 4), 40 * 4 + 4), ((32, 4), 32 * 4), ((32, 129), 32 * 129 + 4)):
        with pytest.raises(capi.MvhError, match="byte size"):
            ctx.upload("w", capi.MVH_TYPE_FP8_B128, *shape, np.zeros(size, np.uint8))
    with pytest.raises(ValueError):
        ctx.matmul_fp8(t, np.zeros((2, 48), F))
    with pytest.raises(ValueError):
        ctx.matmul_fp8(t, torch.zeros((2, 32), device="cuda"), np.zeros((2, 20), F))
    xd = torch.zeros(4 * 32 + 4, device="cuda")
    with pytest.raises(capi.MvhError, match="16-byte aligned"):
        ctx.matmul_fp8(t, xd[1:65].reshape(2, 32), torch.zeros((2, 20), device="cuda"))
    flat = torch.zeros(256, device="cuda")
    with pytest.raises(capi.MvhError, match="must not overlap"):
        ctx.matmul_fp8(t, flat[:64].reshape(2, 32), flat[60:100].reshape(2, 20))
    raw = flat.view(torch.uint8)
    for codes, scales in ((raw[:64], flat[128:130]), (raw[512:576], flat[1:3]), (raw[512:576], flat[129:131])):
        with pytest.raises(capi.MvhError, match="must not overlap"):
            ctx.quantize_fp8(flat[:64].reshape(2, 32), 1, codes, scales)
    for a in (t, t2, q4):
        a.free()
