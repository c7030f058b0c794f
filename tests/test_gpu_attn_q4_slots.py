"""Slots of a 4-bit page that no row has been written to, or that lie behind the page's last row in its group of 8, hold NaN
here for certain: the library's own launchers on pages and tables of the test's making."""
import ctypes
import math

import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import attend, q4_values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

REL = 4e-6  # as in test_gpu_attn_q4.py


def _launchers():
    lib = ctypes.CDLL(capi.load_library()._name)
    p, n = ctypes.c_void_p, ctypes.c_size_t
    write = lib["_ZN3mvh16launch_kv4_writeEPKPvS2_PKfS4_mPKimmmmP12ihipStream_t"]
    write.argtypes = [p, p, p, p, n, p, n, n, n, n, p]
    scratch = lib["_ZN3mvh15attn_q4_scratchEmmmmmmm"]
    scratch.argtypes, scratch.restype = [n] * 7, n
    attn = lib["_ZN3mvh14launch_attn_q4EPKPKvS3_PKfmPfS6_PKimmmmmmmmmP12ihipStream_t"]
    attn.argtypes = [p, p, p, n, p, p, p] + [n] * 9 + [p]
    return write, scratch, attn


@pytest.mark.parametrize("hd,n_kv,page", [(128, 2, 20), (64, 2, 20), (128, 1, 9), (64, 2, 33), (48, 2, 20), (288, 1, 13), (128, 2, 64)])
def test_slots_that_hold_nan(hd, n_kv, page):
    write, scratch, attn = _launchers()
    rng = np.random.default_rng(hd + page)
    rows, kv_dim = 1790, n_kv * hd
    groups, blocks, pages = (page + 7) // 8, kv_dim // 32, math.ceil(1800 / page)
    size = blocks * groups * 160
    slab = torch.full((2, pages, size), 0xff, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[slab[w, i].data_ptr() for i in range(pages)] for w in range(2)], dtype=torch.int64, device="cuda")
    k, v = (rng.standard_normal((rows, kv_dim), dtype=np.float32) for _ in range(2))
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    stream = torch.cuda.current_stream().cuda_stream
    at = [table[w].data_ptr() for w in range(2)]
    for pos in range(0, rows, 179):  # 10 calls, whose ends lie inside groups
        assert write(*at, dk[pos:].data_ptr(), dv[pos:].data_ptr(), kv_dim, None, pos, 179, kv_dim, page, stream) == 0
    # the steps and middles of slots that no row is in are NaN still, those of rows are not
    scales = slab[:, :, blocks * groups * 128:].cpu().numpy().view(np.float16).reshape(2, pages, blocks, groups, 2, 8)
    place = [(r & 3) * 2 + ((r >> 2) ^ (1 if r & 3 == 3 else 0)) for r in range(8)]
    scales = scales[..., place].transpose(0, 1, 3, 5, 4, 2).reshape(2, pages, groups * 8, 2, blocks)
    used = (np.arange(groups * 8) < page) & (np.arange(pages)[:, None] * page + np.arange(groups * 8) < rows)
    assert np.isnan(scales[:, ~used]).all() and np.isfinite(scales[:, used]).all()
    assert page % 8 == 0 or (~used[: pages - 1]).any()
    k, v = (q4_values(x).reshape(rows, n_kv, hd) for x in (k, v))
    for group, pos, n in ((1, rows - 1, 1), (4, rows - 5, 1), (2, 1000, 2), (8, 700, 3), (4, 1500, 200), (4, 1700, 90), (1, 3, 1), (3, 0, 40)):
        q = rng.standard_normal((n, group * n_kv, hd), dtype=np.float32) * np.float32(1.5)
        dq = torch.from_numpy(q).cuda()
        want = attend(q, k, v, pos, group)
        for chunk in (0, 16):
            part = torch.full((max(1, scratch(pos + n, n, group * n_kv, n_kv, hd, page, chunk)),), math.nan, device="cuda")
            out = torch.full(q.shape, math.nan, device="cuda")
            assert attn(*at, dq.data_ptr(), group * n_kv * hd, part.data_ptr(), out.data_ptr(), None, pos, pos + n, n, group * n_kv,
                        n_kv, hd, kv_dim, page, chunk, stream) == 0
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            assert np.linalg.norm(got - want) <= REL * np.linalg.norm(want), (group, pos, n, chunk)
