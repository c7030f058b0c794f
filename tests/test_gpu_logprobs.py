"""mvh_logprobs against a softmax in 64 bits."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import EPS, log_softmax

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NAMES = ("logprob", "entropy", "top_ids", "top_logprobs")


def _device(ctx, x, targets, top):
    rows = x.shape[0]
    d = torch.from_numpy(x).cuda()
    t = torch.from_numpy(targets).cuda() if targets is not None else None
    lp = torch.empty(rows, device="cuda") if targets is not None else None
    en = torch.empty(rows, device="cuda")
    ids = torch.empty((rows, top), dtype=torch.int32, device="cuda") if top else None
    tl = torch.empty((rows, top), device="cuda") if top else None
    torch.cuda.synchronize()
    ctx.logprobs(d, t, top, lp, en, ids, tl)
    ctx.synchronize()
    return {n: v.cpu().numpy() for n, v in zip(NAMES, (lp, en, ids, tl)) if v is not None}


def _check(got, x, targets, top):
    """log p = (l - m) - ln s: l - m rounded (2^-24 of it), ln s with s off by the exponentials' 2^-22 or so and sums of up
    to n / 256 terms in a row (a random walk: 2^-24 sqrt(n / 256)); entropy the same with terms of the entropy's size."""
    lp = log_softmax(x)
    n = x.shape[1]
    soft = 8 * EPS + 4 * EPS * max(1.0, (n / 256) ** 0.5)
    with np.errstate(invalid="ignore"):
        p = np.exp(lp)
        want_h = -np.where(p > 0, p * lp, 0.0).sum(axis=1)
    assert (abs(got["entropy"] - want_h) <= soft * (2 + 3 * abs(want_h))).all()

    def close(a, b):
        fin = np.isfinite(b)
        assert (np.isneginf(a) == np.isneginf(b)).all() and np.isfinite(a[fin]).all()
        assert (abs(a - b)[fin] <= (soft + 3 * EPS * abs(b) + 2 * EPS * abs(x[np.isfinite(x)]).max())[fin]).all()

    if targets is not None:
        close(got["logprob"], lp[np.arange(len(x)), targets])
    if top:
        order = np.argsort(-(x + 0.0), axis=1, kind="stable")[:, :top]
        assert (got["top_ids"] == order).all()
        close(got["top_logprobs"], np.take_along_axis(lp, order, axis=1))


# rows of one element, of no whole quad, of one batch and around it, of several parts; few and many rows
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (1, 63), (2, 64), (5, 65), (1, 1000), (4, 4095), (1, 4096), (3, 4097),
                                    (1, 32000), (7, 32003), (600, 513), (300, 5000), (2, 130001), (300, 9001), (520, 8500)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_random(ctx, rows, n, top):
    rng = np.random.default_rng(rows + n)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    t = rng.integers(0, n, rows).astype(np.int32)
    if top > n:
        with pytest.raises(capi.MvhError, match="top_k"):
            ctx.logprobs(x, t, top)
        return
    got = ctx.logprobs(x, t, top)
    _check(got, x, t, top)
    dev = _device(ctx, x, t, top)
    for name in got:
        assert (dev[name] == got[name]).all(), name


@pytest.mark.parametrize("n", [70, 5000, 40000])
def test_orders_and_ties(ctx, n):
    """Ascending and descending rows, rows of equal values, of few values, signed zeros, peaks in the last place."""
    rng = np.random.default_rng(n)
    x = np.zeros((9, n), np.float32)
    x[0] = np.arange(n) * np.float32(1e-3)
    x[1] = -x[0]
    x[3] = rng.integers(0, 3, n)
    x[4] = np.where(rng.random(n) < 0.5, 0.0, -0.0)
    x[5, -1] = 5
    x[6] = -3.4028235e38
    x[7] = rng.integers(0, 50, n)[np.argsort(rng.random(n))]
    x[8] = 1e4 * rng.standard_normal(n)
    t = np.array([n - 1, 0, n // 2, 1, 2, n - 1, 3, 5, int(x[8].argmax())], np.int32)
    for top in (1, 20, 64):
        got = ctx.logprobs(x[:8], t[:8], top)
        _check(got, x[:8], t[:8], top)
        got = ctx.logprobs(x[8:], t[8:], top)
        _check(got, x[8:], t[8:], top)


@pytest.mark.parametrize("n", [65, 4097, 33000])
def test_masked(ctx, n):
    """-inf everywhere but in a few places, fewer than top_k; a row of nothing else; the far end of a row."""
    rng = np.random.default_rng(n)
    x = np.full((5, n), -np.inf, np.float32)
    x[0, [3, n - 1, n // 2]] = 1.0, 2.0, 2.0
    x[1, n - 1] = -4.0
    x[2, 0] = 3e38
    x[3, rng.integers(0, n, 40)] = rng.standard_normal(40)
    t = np.array([n - 1, n - 1, 0, 1, 2], np.int32)
    t[3] = int(np.flatnonzero(np.isfinite(x[3]))[0])
    for top in (0, 5, 64):
        got = ctx.logprobs(x, t, top)
        _check({k: v[:4] for k, v in got.items()}, x[:4], t[:4], top)
        assert got["logprob"][4] == -np.inf and got["entropy"][4] == 0
        if top:
            assert (got["top_ids"][4] == np.arange(top)).all() and (got["top_logprobs"][4] == -np.inf).all()


@pytest.mark.parametrize("n", [100, 9000])
def test_nan_and_infinity(ctx, n):
    """A NaN or +inf makes the row's float results NaN, leaves ids in range and the other rows as they are."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((5, n)).astype(np.float32)
    t = np.full(5, 7, np.int32)
    clean = ctx.logprobs(x, t, 5)
    x[1, n - 1] = np.nan
    x[2, 0] = np.inf
    x[3, n // 2:] = -np.nan
    got = ctx.logprobs(x, t, 5)
    for name in NAMES:
        assert (got[name][[0, 4]] == clean[name][[0, 4]]).all()
        if name != "top_ids":
            assert np.isnan(got[name][1:4]).all(), name
    assert (got["top_ids"] >= 0).all() and (got["top_ids"] < n).all()


def test_one_kind_of_output_at_a_time(ctx):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    t = np.array([0, 4999, 17], np.int32)
    want = ctx.logprobs(x, t, 3)
    d, dt = torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()
    for name in NAMES:
        out = torch.full((3, 3) if name.startswith("top") else (3,), 9, device="cuda",
                         dtype=torch.int32 if name == "top_ids" else torch.float32)
        torch.cuda.synchronize()
        ctx.logprobs(d, dt if name == "logprob" else None, 3, **{name: out})
        ctx.synchronize()
        assert (out.cpu().numpy() == want[name]).all(), name
    # targets out of range on the device: NaN, nothing else
    bad = torch.tensor([-1, 5000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    lp, en = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    torch.cuda.synchronize()
    ctx.logprobs(d, bad, 0, logprob=lp, entropy=en)
    ctx.synchronize()
    assert torch.isnan(lp).all() and (en.cpu().numpy() == want["entropy"]).all()


def test_refusals(ctx):
    x, t = np.zeros((2, 10), np.float32), np.zeros(2, np.int32)

    def refused(code, text, *a):
        with pytest.raises(capi.MvhError, match=text) as e:
            ctx.logprobs(*a)
        assert e.value.code == code

    refused(1, "empty", np.zeros((2, 0), np.float32))
    refused(5, "top_k", x, t, 11)
    refused(5, "top_k", np.zeros((2, 100), np.float32), t, 65)
    refused(5, "target -1 of row 1", x, np.array([0, -1], np.int32))
    refused(5, "target 10 of row 0", x, np.array([10, 0], np.int32))
    lib, p = ctx.lib, x.ctypes.data
    assert lib.mvh_logprobs(ctx.h, p, 10, 2, None, 0, p, None, None, None, 0) == 1  # logprob without targets
    assert lib.mvh_logprobs(ctx.h, None, 10, 2, None, 0, None, p, None, None, 0) == 1
    assert lib.mvh_logprobs(ctx.h, p, 10, 2, None, 0, None, p, None, None, 5) == 1
    assert lib.mvh_logprobs(ctx.h, None, 10, 0, None, 0, None, None, None, None, 0) == 0  # no rows
    assert lib.mvh_logprobs(None, p, 10, 2, None, 0, None, p, None, None, 0) == 1
