"""Attention over a cache held in 4 bits against attention in 64 bits over the values that the cache holds."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import attend, q4_values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# Scores y in powers of two reach some 20 here: q in two fp16 leaves 2^-22 of each product, the fp32 sums a few 2^-24 of
# their terms (about twice the score's size): 20 * (2^-22 + 4 * 2^-24) = 1e-5 at worst in y, times ln 2 in a weight, a
# fourth of that in its rms; the weights' own two fp16 and the value sums add some 2^-22.  4e-6 covers both.
REL = 4e-6


def _case(ctx, rng, n_kv, hd, page, rows, layers=1, shift=1.0):
    kv = ctx.kv_cache(layers, n_kv * hd, page, rows, kv_type=capi.MVH_KV_Q4)
    k, v = (rng.standard_normal((rows, n_kv * hd), dtype=np.float32) for _ in range(2))
    k += np.float32(shift) * rng.standard_normal(n_kv * hd, dtype=np.float32)
    kv.write(layers - 1, 0, k, v)
    return kv, q4_values(k).reshape(rows, n_kv, hd), q4_values(v).reshape(rows, n_kv, hd)


def _check(got, want, what):
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= REL, (what, rel)
    rms = np.linalg.norm(want) / np.sqrt(want.size)
    assert abs(got - want).max() <= 40 * REL * max(rms, abs(want).max()), what


# head_dims of one block to eight, parts of blocks (48, 40, 24 ..: blocks shared by heads), more than eight blocks (288);
# groups of 1 to 12 heads; pages of 1 row, no whole groups, whole groups, whole steps
@pytest.mark.parametrize("n_head,n_kv,hd,page", [(8, 1, 64, 128), (4, 4, 128, 128), (2, 2, 32, 7), (6, 2, 96, 64), (6, 6, 48, 16),
                                                 (32, 4, 64, 20), (2, 1, 192, 32), (2, 1, 256, 8), (24, 2, 32, 1),
                                                 (5, 1, 128, 96), (4, 4, 40, 9), (2, 2, 80, 128), (2, 1, 160, 128),
                                                 (8, 8, 24, 128), (8, 4, 72, 20), (2, 2, 112, 32), (4, 4, 56, 16), (4, 4, 8, 128),
                                                 (4, 2, 16, 5), (1, 1, 224, 128), (2, 1, 288, 128)])
def test_decode(ctx, n_head, n_kv, hd, page):
    rng = np.random.default_rng(hd + page + n_head)
    kv, k, v = _case(ctx, rng, n_kv, hd, page, 1100)
    q = rng.standard_normal((1, n_head, hd), dtype=np.float32) * np.float32(1.5)
    for pos in (0, 1, 6, 7, 8, 15, 31, 32, 33, 63, 64, 127, 128, 129, 200, 511, 512, 700, 1023, 1024, 1099):
        got = kv.attn_decode(0, q.reshape(-1), pos, n_head, n_kv, hd).reshape(1, n_head, hd)
        _check(got, attend(q, k, v, pos, n_head // n_kv), pos)
    kv.close()


@pytest.mark.parametrize("n_head,n_kv,hd,page", [(8, 2, 64, 128), (4, 4, 128, 16), (12, 1, 32, 7), (6, 6, 48, 128),
                                                 (32, 8, 128, 128), (3, 3, 256, 20), (4, 2, 96, 1),
                                                 (8, 8, 24, 16), (16, 4, 72, 128), (4, 4, 56, 20), (2, 1, 160, 128), (2, 1, 288, 16)])
def test_batch(ctx, n_head, n_kv, hd, page):
    rng = np.random.default_rng(hd + page + n_head + 1)
    kv, k, v = _case(ctx, rng, n_kv, hd, page, 400)
    for pos, n in ((0, 1), (0, 2), (0, 40), (5, 3), (31, 33), (100, 7), (255, 64), (130, 129), (0, 300)):
        q = rng.standard_normal((n, n_head, hd), dtype=np.float32) * np.float32(1.5)
        got = kv.attn_batch(0, q.reshape(n, -1), pos, n, n_head, n_kv, hd).reshape(n, n_head, hd)
        _check(got, attend(q, k, v, pos, n_head // n_kv), (pos, n))
    kv.close()


# pages of one row (every row a group of 8 of its own), of no whole groups, of whole groups, steps and pairs of steps; one to
# 40 heads a kv head; rows, steps and pages on both sides of what the kernels split at
@pytest.mark.parametrize("hd,page", [(64, 20), (128, 96), (64, 9), (128, 1), (128, 128), (64, 64), (128, 16), (64, 32)])
def test_rows_and_steps(ctx, hd, page):
    rng = np.random.default_rng(hd * page)
    n_kv = 2
    kv, k, v = _case(ctx, rng, n_kv, hd, page, 2300)
    for group, pos, n in ((1, 990, 1), (1, 991, 1), (1, 992, 1), (1, 2200, 1), (4, 1500, 1), (4, 2111, 1), (2, 2000, 2), (1, 2100, 4),
                          (5, 2000, 1), (3, 2001, 5), (4, 2100, 4), (8, 1900, 40), (4, 2000, 200), (40, 2290, 9), (1, 1600, 700)):
        q = rng.standard_normal((n, group * n_kv, hd), dtype=np.float32) * np.float32(1.5)
        got = kv.attn_batch(0, q.reshape(n, -1), pos, n, group * n_kv, n_kv, hd).reshape(q.shape)
        _check(got, attend(q, k, v, pos, group), (group, pos, n))
    kv.close()


def test_page_past_4_gib(ctx):
    """Pages of 5 GiB: rows and heads beyond offsets of 32 bits."""
    rng = np.random.default_rng(40)
    n_kv, hd, rows = 64, 128, 2 ** 20
    kv = ctx.kv_cache(1, n_kv * hd, rows, rows, kv_type=capi.MVH_KV_Q4)
    k, v = (rng.standard_normal((41, n_kv * hd), dtype=np.float32) for _ in range(2))
    for pos in (0, rows - 41):
        kv.write(0, pos, k, v)
        for got, want in zip(kv.read(0, pos, 41), (k, v)):
            assert (got == q4_values(want)).all()
        k, v = v, k
    k, v = (q4_values(x).reshape(41, n_kv, hd) for x in (k, v))
    for n in (1, 3, 41):  # 41 - n rows before the chunk
        q = rng.standard_normal((n, n_kv, hd), dtype=np.float32)
        _check(kv.attn_batch(0, q.reshape(n, -1), 41 - n, n, n_kv, n_kv, hd).reshape(q.shape), attend(q, k, v, 41 - n, 1), n)
    kv.close()


@pytest.mark.parametrize("n_head,n_kv,hd,n", [(8, 2, 128, 40001), (4, 4, 64, 70000), (2, 2, 48, 9000)])
def test_long(ctx, n_head, n_kv, hd, n):
    """Past 16000 positions (and 2^16), several pages of scores a split, and a page table of its own layer."""
    rng = np.random.default_rng(n)
    kv, k, v = _case(ctx, rng, n_kv, hd, 128, n, layers=2)
    for pos in (n - 1, n // 2, 4097):
        q = rng.standard_normal((1, n_head, hd), dtype=np.float32) * np.float32(1.5)
        got = kv.attn_decode(1, q.reshape(-1), pos, n_head, n_kv, hd).reshape(1, n_head, hd)
        # weights spread over n rows leave sums of size 1 / sqrt(n) beside terms of size 1
        want = attend(q, k, v, pos, n_head // n_kv)
        assert np.linalg.norm(got - want) <= 2 * REL * np.linalg.norm(want), pos
    q = rng.standard_normal((5, n_head, hd), dtype=np.float32) * np.float32(1.5)
    got = kv.attn_batch(1, q.reshape(5, -1), n - 5, 5, n_head, n_kv, hd).reshape(5, n_head, hd)
    want = attend(q, k, v, n - 5, n_head // n_kv)
    assert np.linalg.norm(got - want) <= 2 * REL * np.linalg.norm(want)
    kv.close()


@pytest.mark.parametrize("scale_k,scale_v,scale_q", [(1e-3, 1.0, 1e3), (1.0, 1e-3, 1.0), (1.0, 2000.0, 1.0), (100.0, 1.0, 0.01),
                                                     (1.0, 1.0, 0.0), (1.0, 1.0, 1e-30), (30.0, 1.0, 1.0)])
def test_scales(ctx, scale_k, scale_v, scale_q):
    """Small and large keys, values and queries; q of zero weighs every row alike; one row that takes all the weight."""
    rng = np.random.default_rng(7)
    n_kv, hd, rows = 2, 64, 500
    k, v = (rng.standard_normal((rows, n_kv * hd), dtype=np.float32) * np.float32(s) for s in (scale_k, scale_v))
    kv = ctx.kv_cache(1, n_kv * hd, 128, rows, kv_type=capi.MVH_KV_Q4)
    kv.write(0, 0, k, v)
    k, v = (q4_values(a).reshape(rows, n_kv, hd) for a in (k, v))
    q = rng.standard_normal((1, 4, hd), dtype=np.float32) * np.float32(scale_q)
    got = kv.attn_decode(0, q.reshape(-1), rows - 1, 4, n_kv, hd).reshape(1, 4, hd)
    want = attend(q, k, v, rows - 1, 2)
    # scores thirty times as large carry thirty times the error
    assert np.linalg.norm(got - want) <= REL * max(1.0, scale_k * scale_q) * np.linalg.norm(want)
    kv.close()


@pytest.mark.parametrize("hd,page", [(128, 128), (64, 20), (48, 16)])
def test_rows_past_the_position_do_not_count(ctx, hd, page):
    """Rows after a token's position may hold anything, also NaN; the same for rows of other pages and unwritten slots."""
    rng = np.random.default_rng(hd)
    n_head, rows = 4, 90
    k, v = (rng.standard_normal((rows, n_head * hd), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((40, n_head * hd), dtype=np.float32)
    outs = []
    for far in (0.5, np.nan, np.inf):
        k[70:] = v[70:] = far
        kv = ctx.kv_cache(1, n_head * hd, page, 256, kv_type=capi.MVH_KV_Q4)
        kv.write(0, 0, np.full((256, n_head * hd), np.nan, np.float32), np.full((256, n_head * hd), np.nan, np.float32))
        kv.reset()  # the pages that follow hold NaN from here
        kv.write(0, 0, k, v)
        outs.append(kv.attn_batch(0, q, 50, 40, n_head, n_head, hd).copy())
        one = kv.attn_decode(0, q[0], 69, n_head, n_head, hd)
        outs.append(one)
        kv.close()
    for a, b in ((0, 2), (2, 4)):
        assert np.isfinite(outs[a][:20]).all()
        assert (outs[a][:20] == outs[b][:20]).all() and (outs[a + 1] == outs[b + 1]).all()
    assert np.isnan(outs[2][20:]).all()


@pytest.mark.parametrize("hd,page", [(128, 20), (64, 20), (128, 9), (64, 33)])
def test_slots_behind_a_page(ctx, hd, page):
    """Pages that end inside a group of 8: what the group's other slots hold (here memory that held NaN) does not count."""
    rng = np.random.default_rng(page)
    n_kv, rows = 2, 1800
    bad = ctx.kv_cache(1, n_kv * hd, 128, 4 * rows, kv_type=capi.MVH_KV_Q4)
    x = np.full((4 * rows, n_kv * hd), np.nan, np.float32)
    bad.write(0, 0, x, x)
    bad.close()
    kv, k, v = _case(ctx, rng, n_kv, hd, page, rows)
    for group, pos, n in ((1, rows - 1, 1), (4, rows - 5, 1), (8, 700, 3), (4, 1500, 200), (4, 1700, 100)):
        q = rng.standard_normal((n, group * n_kv, hd), dtype=np.float32) * np.float32(1.5)
        got = kv.attn_batch(0, q.reshape(n, -1), pos, n, group * n_kv, n_kv, hd).reshape(q.shape)
        _check(got, attend(q, k, v, pos, group), (group, pos, n))
    kv.close()


@pytest.mark.parametrize("hd", [128, 48])
def test_bad_rows_stay_with_their_head(ctx, hd):
    """A NaN in one kv head's row makes that head's outputs NaN from there on, and no other's (blocks of 32 at hd 48 hold
    elements of two heads: the neighbour shares the block)."""
    rng = np.random.default_rng(1)
    n_kv, rows = 4, 100
    k, v = (rng.standard_normal((rows, n_kv * hd), dtype=np.float32) for _ in range(2))
    k[30, 2 * hd + 40] = np.nan
    v[60, 0] = np.inf
    kv = ctx.kv_cache(1, n_kv * hd, 128, rows, kv_type=capi.MVH_KV_Q4)
    kv.write(0, 0, k, v)
    q = rng.standard_normal((rows, n_kv * 2 * hd), dtype=np.float32)
    out = kv.attn_batch(0, q, 0, rows, 2 * n_kv, n_kv, hd).reshape(rows, n_kv, 2, hd)
    assert np.isnan(out[30:, 2]).all() and np.isfinite(out[:30]).all()
    assert np.isnan(out[60:, 0, :, :32]).all() and np.isfinite(out[:, 0, :, 32:]).all()
    assert np.isfinite(out[:, 1]).all()
    if hd == 128:
        assert np.isfinite(out[:, 3]).all()
    q[50] = np.inf
    assert not np.isfinite(kv.attn_batch(0, q[50:51], 50, 1, 2 * n_kv, n_kv, hd)).any()
    kv.close()


def test_same_bits_every_time(ctx):
    """Split calls and repeated ones: no atomics, so the same bits; the same for q in device memory off any alignment."""
    rng = np.random.default_rng(11)
    kv, _, _ = _case(ctx, rng, 2, 128, 128, 3000)
    q = rng.standard_normal((7, 8 * 128), dtype=np.float32)
    first = kv.attn_batch(0, q, 2500, 7, 8, 2, 128)
    buf = torch.empty(7 * 8 * 128 + 1, device="cuda")
    buf[1:] = torch.from_numpy(q).cuda().reshape(-1)
    out = torch.empty(7 * 8 * 128 + 3, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        kv.attn_batch(0, buf[1:], 2500, 7, 8, 2, 128, out[3:])
        ctx.synchronize()
        assert (out[3:].cpu().numpy().reshape(first.shape) == first).all()
    kv.close()


def test_refusals(ctx):
    def refused(code, text, f, *a):
        with pytest.raises(capi.MvhError, match=text) as e:
            f(*a)
        assert e.value.code == code

    kv = ctx.kv_cache(1, 128, 16, 40, kv_type=capi.MVH_KV_Q4)
    assert kv.type() == 3 and capi.kv_parse_type("q4") == 3 and capi.kv_type_name(3) == "q4"
    q = np.zeros((2, 256), np.float32)
    refused(5, "missing", kv.attn_decode, 0, q[0], 0, 4, 2, 64)
    kv.write(0, 0, q[:, :128], q[:, :128])
    refused(5, "missing", kv.attn_batch, 0, q, 15, 2, 4, 2, 64)
    refused(5, "exhausted", kv.attn_decode, 0, q[0], 40, 4, 2, 64)
    refused(2, "head configuration", kv.attn_decode, 0, q[0], 0, 3, 2, 64)
    refused(2, "head_dim", kv.attn_decode, 0, q[0], 0, 4, 2, 60)
    refused(2, "head_dim", kv.attn_decode, 0, q[0], 0, 4, 2, 128)
    refused(5, "layer", kv.attn_decode, 1, q[0], 0, 4, 2, 64)
    for far in (2 ** 64 - 1, 2 ** 64 - 2, 2 ** 63):
        refused(5, "exhausted", kv.attn_batch, 0, q, far, 2, 4, 2, 64)
        refused(5, "exhausted", kv.write, 0, far, q[:, :128], q[:, :128])
    refused(5, "pages", ctx.kv_cache, 2 ** 60, 128, 16, 2 ** 20, capi.MVH_KV_Q4)
    assert (kv.attn_decode(0, q[0], 0, 4, 2, 64) == 0).all()
    kv.close()
