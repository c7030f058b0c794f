"""The largest calls that the rotary and cache entry points take, and what they refuse beyond."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import q4_values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def test_rotate_2_24_tokens(ctx):
    """A workgroup of 256 threads a token would be 2^32 of them in one launch: 17 GB rotated in place."""
    n, hd = 2 ** 24, 258  # of no whole vectors, 129 units: one token a workgroup
    r = ctx.rope(hd)
    x = torch.ones((n, hd), device="cuda")
    torch.cuda.synchronize()
    r.apply(x, 1, pos=5, out=x)
    ctx.synchronize()
    at = np.array([0, 1, 2 ** 22 - 1, 2 ** 22, 2 ** 23 + 12345, n - 2, n - 1])
    want = r.apply(np.ones((len(at), hd), np.float32), 1, positions=(at + 5).astype(np.int32))
    assert (x[torch.from_numpy(at).cuda()].cpu().numpy() == want).all()
    # the same by a list of positions
    x.fill_(1.0)
    positions = torch.arange(5, n + 5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    r.apply(x, 1, positions=positions, out=x)
    ctx.synchronize()
    assert (x[torch.from_numpy(at).cuda()].cpu().numpy() == want).all()
    r.close()


def test_read_2_34_elements(ctx):
    """2^20 rows of 16384 channels in one call: 2^32 quads, 64 GiB."""
    n, dim = 2 ** 20, 16384
    kv = ctx.kv_cache(1, dim, n, n, kv_type=capi.MVH_KV_Q4)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, dim), dtype=np.float32)
    at = (0, 2 ** 19 - 1, n - 3)
    for pos in at:
        kv.write(0, pos, x, x)
    out = torch.empty((n, dim), device="cuda")
    torch.cuda.synchronize()
    kv.read(0, 0, n, k=out)
    ctx.synchronize()
    for pos in at:
        assert (out[pos:pos + 3].cpu().numpy() == q4_values(x)).all(), pos
    kv.close()


@pytest.mark.parametrize("off", [0, 1])
def test_append_rows_of_2_24(ctx, off):
    """The widest rows an append takes, as vectors and (one float off) pair by pair."""
    hd, dim = 128, 2 ** 24
    r = ctx.rope(hd)
    kv = ctx.kv_cache(1, dim, 2, 2, kv_type=capi.MVH_KV_F16)
    buf = torch.randn(3 * dim + off, device="cuda")
    q, k, v = (buf[off + i * dim: off + (i + 1) * dim].view(1, dim) for i in range(3))
    q_out = torch.empty((1, dim), device="cuda")
    torch.cuda.synchronize()
    kv.append(0, 1, k, v, r, q=q, q_out=q_out)
    ctx.synchronize()
    some = np.concatenate([np.arange(0, 4), np.arange(2 ** 16, 2 ** 16 + 4), np.arange(dim // hd - 4, dim // hd)])  # heads
    rows = [np.ascontiguousarray(x.cpu().numpy().reshape(-1, hd)[some].reshape(1, -1)) for x in (q, k, v)]
    assert (q_out.cpu().numpy().reshape(-1, hd)[some].reshape(1, -1) == r.apply(rows[0], len(some), pos=1)).all()
    half = lambda x: ctx.fp16_to_fp32(ctx.fp32_to_fp16(x)).reshape(x.shape)
    got_k, got_v = kv.read(0, 1, 1)
    assert (got_k.reshape(-1, hd)[some].reshape(1, -1) == half(r.apply(rows[1], len(some), pos=1))).all()
    assert (got_v.reshape(-1, hd)[some].reshape(1, -1) == half(rows[2])).all()
    kv.close()
    r.close()


def test_sizes_beyond_int(ctx):
    """Page and row sizes that the kernels' 32-bit arithmetic cannot hold are refused before a page is made."""
    for dim, page in ((8, 2 ** 31), (8, 2 ** 32), (2 ** 31, 1), (2 ** 32 + 8, 1)):
        for kv_type in (capi.MVH_KV_F32, capi.MVH_KV_F16, capi.MVH_KV_Q8):
            with pytest.raises(capi.MvhError, match="2147483647") as e:
                ctx.kv_cache(1, dim, page, 4, kv_type=kv_type)
            assert e.value.code == 5
    kv = ctx.kv_cache(1, 2 ** 24 + 128, 1, 1, kv_type=capi.MVH_KV_F16)
    r = ctx.rope(128)
    x = torch.empty((1, 2 ** 24 + 128), device="cuda")
    with pytest.raises(capi.MvhError, match="16777216") as e:
        kv.append(0, 0, x, x, r)
    assert e.value.code == 5
    kv.close()
    r.close()
