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
