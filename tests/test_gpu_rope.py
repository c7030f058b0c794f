"""Rotary positions and rotated appends (mvh_rope_*, mvh_kv_append, mvh_kv_read) against plain restatements."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import angles, q4_values, rotate

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SCALED = {0: {}, 1: dict(factor=4.0), 2: dict(base=500000.0, factor=8.0, orig_ctx=8192.0, low=1.0, high=4.0),
          3: dict(factor=16.0, orig_ctx=4096.0, low=1.0, high=32.0, attn_scale=1.277)}


def _rope(ctx, hd, rot, layout, scaling):
    o = SCALED[scaling]
    r = ctx.rope(hd, rot_dim=rot, layout=layout, scaling=scaling, **o)
    o = dict(o)
    scale = o.pop("attn_scale", 1.0)
    return r, angles(rot, scaling=scaling, **o), scale


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
@pytest.mark.parametrize("rot", [2, 48, 64, 128])
def test_angles(ctx, rot, scaling):
    r, f, _ = _rope(ctx, 128, rot, 0, scaling)
    assert np.allclose(r.angles(), f, rtol=8 * 2.0 ** -53, atol=0)
    r.close()


# (tokens, heads, hd, rot): one token, more units than a workgroup, part of the head, odd sizes that are no vectors
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("n,heads,hd,rot,scaling", [(1, 40, 128, 128, 0), (3, 32, 64, 64, 2), (77, 6, 48, 24, 1),
                                                    (5, 3, 10, 6, 0), (2, 1, 2, 2, 3), (600, 2, 128, 64, 3),
                                                    (1, 1, 1024, 1024, 0), (9, 33, 80, 40, 2), (4, 2, 96, 36, 0)])
def test_apply(ctx, layout, n, heads, hd, rot, scaling):
    rng = np.random.default_rng(n + hd + rot)
    r, f, scale = _rope(ctx, hd, rot, layout, scaling)
    x = rng.standard_normal((n, heads * hd), dtype=np.float32)
    for positions, pos in ((None, 0), (None, 131000), (rng.integers(-50, 1 << 20, n).astype(np.int32), 0)):
        at = np.arange(pos, pos + n) if positions is None else positions
        want, err = rotate(x.reshape(n, heads, hd), at, f, rot, layout == 1, scale)
        got = r.apply(x, heads, pos=pos, positions=positions).reshape(n, heads, hd)
        assert (abs(got - want) <= err).all(), (abs(got - want) - err).max()
        assert (got[..., rot:] == x.reshape(n, heads, hd)[..., rot:]).all()
        # a strided view on the device, in place, gives the same bits and leaves its neighbours alone
        wide = torch.full((n, heads * hd + 6), 7.0, device="cuda")
        wide[:, 2:2 + heads * hd] = torch.from_numpy(x).cuda()
        view = wide[:, 2:2 + heads * hd]
        torch.cuda.synchronize()
        r.apply(view, heads, pos=pos, positions=None if positions is None else torch.from_numpy(positions).cuda(), out=view)
        ctx.synchronize()
        assert (view.cpu().numpy().reshape(got.shape) == got).all()
        assert (wide[:, :2] == 7).all() and (wide[:, -4:] == 7).all()
    r.close()


def test_far_positions_stay_exact(ctx):
    """The largest int32 positions: the angle's 31 bits and the reduction keep cos and sin to half a step."""
    r, f, _ = _rope(ctx, 128, 128, 0, 0)
    positions = np.array([2 ** 31 - 1, 2 ** 30 + 12345, -2 ** 31, 99_999_999], np.int32)
    x = np.zeros((4, 128), np.float32)
    x[:, :64] = 1
    want, err = rotate(x[:, None], positions, f, 128, False)
    got = r.apply(x, 1, positions=positions)[:, None]
    assert (abs(got - want) <= err + 1e-6 * (abs(want) < 1e-3)).all()
    r.close()


def _stored(kv_type, x, ctx):
    """Rows as a cache of the type holds them: written without rotation by mvh_kv_write."""
    kv = ctx.kv_cache(1, x.shape[1], 64, max(x.shape[0], 1), kv_type=kv_type)
    kv.write(0, 0, x, x)
    out = kv.read(0, 0, x.shape[0])[0]
    kv.close()
    return out


# pages of a row, of no whole group of 8 rows, of whole groups; one token, parts of groups, several pages
@pytest.mark.parametrize("kv_type", [0, 1, 2, 3])
@pytest.mark.parametrize("heads,kv_heads,hd,rot,page", [(4, 4, 128, 128, 128), (6, 6, 48, 24, 7), (8, 2, 64, 64, 16),
                                                        (3, 1, 32, 20, 1), (2, 2, 80, 40, 20)])
@pytest.mark.parametrize("layout", [0, 1])
def test_append(ctx, kv_type, heads, kv_heads, hd, rot, page, layout):
    rng = np.random.default_rng(hd + page + kv_type)
    r, _, _ = _rope(ctx, hd, rot, layout, 2)
    kv_dim = kv_heads * hd
    kv = ctx.kv_cache(2, kv_dim, page, 200, kv_type=kv_type)
    rows_k = np.full((200, kv_dim), np.nan, np.float32)
    rows_v = rows_k.copy()
    for pos, n in ((0, 1), (1, 1), (2, 13), (15, 1), (16, 8), (24, 40), (64, 3), (67, 100), (30, 5), (199, 1)):
        qkv = rng.standard_normal((n, heads * hd + 2 * kv_dim), dtype=np.float32) * 3
        q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:-kv_dim], qkv[:, -kv_dim:]
        fused = torch.from_numpy(qkv).cuda()
        q_out = torch.empty((n, heads * hd), device="cuda")
        dq, dk, dv = fused[:, :heads * hd], fused[:, heads * hd:-kv_dim], fused[:, -kv_dim:]
        torch.cuda.synchronize()
        if n % 2:  # q to rows of its own, else in place
            kv.append(1, pos, dk, dv, r, q=dq, q_out=q_out)
            ctx.synchronize()
        else:
            kv.append(1, pos, dk, dv, r, q=dq, q_out=dq)
            ctx.synchronize()
            q_out = dq
        want_q = r.apply(np.ascontiguousarray(q), heads, pos=pos)
        assert (q_out.cpu().numpy() == want_q).all()
        assert (dk.cpu().numpy() == k).all() and (dv.cpu().numpy() == v).all()
        rows_k[pos:pos + n] = _stored(kv_type, r.apply(np.ascontiguousarray(k), kv_heads, pos=pos), ctx)
        rows_v[pos:pos + n] = _stored(kv_type, np.ascontiguousarray(v), ctx)
        last = min(pos + n, 167) if pos < 199 else 167
        got_k, got_v = kv.read(1, 0, last)
        assert (got_k == rows_k[:last]).all() and (got_v == rows_v[:last]).all(), (pos, n)
    got_k, got_v = kv.read(1, 199, 1)
    assert (got_k == rows_k[199:]).all() and (got_v == rows_v[199:]).all()
    # host arrays, without q
    k = rng.standard_normal((9, kv_dim), dtype=np.float32)
    kv.append(1, 3, k, -k, r)
    got_k, got_v = kv.read(1, 3, 9)
    assert (got_k == _stored(kv_type, r.apply(k, kv_heads, pos=3), ctx)).all() and (got_v == _stored(kv_type, -k, ctx)).all()
    kv.close()
    r.close()


def test_q4_format(ctx):
    """mvh_kv_write to 4-bit pages: the values the format's definition gives, bit for bit, with its edges."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((40, 96), dtype=np.float32) * np.exp(rng.uniform(-12, 8, (40, 1))).astype(np.float32)
    x[0] = 0.0
    x[1] = -3.25
    x[2, :32] = np.linspace(-8, 7, 32)  # ties
    x[3, 5] = np.inf
    x[4, 40] = np.nan
    x[5, 70] = -np.inf
    x[6] = 3e38 * np.sign(x[6])
    x[7] = 1e-38
    x[8, :32] = np.arange(32) * np.float32(2.0 ** -24)
    x[9] = 1e6
    x[10] += np.float32(1000.0)
    x[11, :32] = np.linspace(0, 9000, 32)
    x[12] = -0.0
    for page in (128, 7, 1):
        kv = ctx.kv_cache(1, 96, page, 64, kv_type=capi.MVH_KV_Q4)
        kv.write(0, 3, x, x[::-1])
        k, v = kv.read(0, 3, 40)
        assert np.array_equal(k, q4_values(x), equal_nan=True)
        assert np.array_equal(v, q4_values(x[::-1]), equal_nan=True)
        row, scale = kv.read_row(0, 13, 1)
        assert scale == 1 and np.array_equal(row, v[10], equal_nan=True)
        touched = 42 // page - 3 // page + 1
        assert kv.bytes_allocated() == touched * page * 2 * 96 * 5 // 8
        kv.close()


@pytest.mark.parametrize("kind", ["normal", "steps", "halves", "wide", "tiny", "huge"])
def test_q4_codes(ctx, kind):
    """Every code of half a million elements, also values on and next to the borders between two codes; by a write, and by a
    rotated append at position 0, which leaves finite rows as they are."""
    rng = np.random.default_rng(len(kind))
    n, f = 1024, np.float32
    x = rng.standard_normal((n, 512), dtype=f)
    if kind in ("steps", "halves"):  # lo + s (i or i + 1/2), exact, and their neighbours
        s = np.exp2(rng.integers(-14, 9, (n, 16, 1))).astype(f) * rng.integers(1, 1024, (n, 16, 1)).astype(f) / f(512)
        i = rng.integers(0, 16, (n, 16, 32)).astype(f)
        i[:, :, 0], i[:, :, 1] = 0, 15
        half = np.where((i > 0) & (i < 15), f(0.5) if kind == "halves" else f(0), f(0))
        x = (rng.integers(-20, 4, (n, 16, 1)).astype(f) * s + s * (i + half)).reshape(n, 512)
        off = rng.integers(-1, 2, x.shape)
        x = np.where(off > 0, np.nextafter(x, f(np.inf)), np.where(off < 0, np.nextafter(x, f(-np.inf)), x))
    elif kind == "wide":
        x *= np.exp(rng.uniform(-30, 30, (n, 1))).astype(f)
    elif kind == "tiny":
        x *= f(2.0 ** -22) * np.exp2(rng.integers(-20, 4, (n, 1))).astype(f)
    elif kind == "huge":
        x *= f(3e37)
    want = q4_values(x)
    kv = ctx.kv_cache(1, 512, 128, n, kv_type=capi.MVH_KV_Q4)
    kv.write(0, 0, x, x[::-1])
    k, v = kv.read(0, 0, n)
    assert (k == want).all() and (v == want[::-1]).all()
    r = ctx.rope(64)
    for row in range(0, 64):
        kv.append(0, 0, x[row:row + 1], x[row + 1:row + 2], r)
        k, v = kv.read(0, 0, 1)
        assert (k == want[row]).all() and (v == want[row + 1]).all(), row
    r.close()
    kv.close()


def test_refusals(ctx):
    def refused(code, text, f, *a, **k):
        with pytest.raises(capi.MvhError, match=text) as e:
            f(*a, **k)
        assert e.value.code == code

    refused(2, "head_dim", ctx.rope, 7)
    refused(2, "head_dim", ctx.rope, 1026)
    refused(2, "rot_dim", ctx.rope, 64, rot_dim=66)
    refused(2, "rot_dim", ctx.rope, 64, rot_dim=33)
    refused(1, "layout", ctx.rope, 64, layout=2)
    refused(1, "scaling", ctx.rope, 64, scaling=4)
    refused(1, "base", ctx.rope, 64, base=1.0)
    refused(1, "base", ctx.rope, 64, base=float("nan"))
    refused(1, "factor", ctx.rope, 64, scaling=1, factor=0.0)
    refused(1, "low < high", ctx.rope, 64, scaling=2, factor=2.0, orig_ctx=10.0, low=4.0, high=4.0)
    refused(1, "attn_scale", ctx.rope, 64, attn_scale=-1.0)
    r = ctx.rope(64)
    x = np.zeros((2, 128), np.float32)
    lib = ctx.lib

    def call(f, *a):
        rc = f(*a)
        return rc, lib.mvh_last_error().decode()

    p = x.ctypes.data
    assert call(lib.mvh_rope_apply, ctx.h, None, p, 128, 2, 2, None, 0, p, 128, 0) == (1, "null rope")
    assert call(lib.mvh_rope_apply, ctx.h, r.h, p, 127, 2, 2, None, 0, p, 128, 0)[0] == 2
    assert call(lib.mvh_rope_apply, ctx.h, r.h, p, 128, 2, 2, None, 0, p, 129, 0)[0] == 1  # in place, another pitch
    assert call(lib.mvh_rope_apply, ctx.h, r.h, None, 128, 2, 2, None, 0, p, 128, 0)[0] == 1
    assert call(lib.mvh_rope_apply, ctx.h, r.h, p, 128, 2, 2, None, 2 ** 31 - 2, p, 128, 0)[0] == 5
    assert call(lib.mvh_rope_apply, ctx.h, r.h, p, 128, 2, 2, None, 0, p, 128, 2)[0] == 1
    assert call(lib.mvh_rope_apply, ctx.h, r.h, None, 128, 0, 2, None, 0, None, 128, 0)[0] == 0  # no rows
    kv = ctx.kv_cache(1, 128, 16, 20)
    refused(5, "exhausted", kv.append, 0, 19, x, x, r)
    refused(5, "exhausted", kv.append, 0, 2 ** 64 - 1, x, x, r)
    refused(5, "layer", kv.append, 1, 0, x, x, r)
    refused(5, "missing", kv.read, 0, 0, 1)
    kv.append(0, 0, x, x, r)
    refused(5, "out of range", kv.read, 0, 19, 2)
    refused(5, "missing", kv.read, 0, 0, 17)
    r48 = ctx.rope(48)
    refused(2, "whole heads", kv.append, 0, 0, x, x, r48)
    r2 = ctx.rope(2)
    refused(2, "whole heads", kv.append, 0, 0, x, x, r2)
    with pytest.raises(ValueError):
        kv.append(0, 0, x, x[:, :64], r)
    refused(2, "multiple of 32", ctx.kv_cache, 1, 40, 16, 16, kv_type=capi.MVH_KV_Q4)
    refused(5, "max_tokens", ctx.kv_cache, 1, 32, 16, 2 ** 20 + 1, kv_type=capi.MVH_KV_Q4)
    refused(5, "16000", ctx.kv_cache, 1, 32, 16, 16001)
    refused(1, "type id 4", ctx.kv_cache, 1, 32, 16, 16, kv_type=4)
    for o in (kv, r, r48, r2):
        o.close()
