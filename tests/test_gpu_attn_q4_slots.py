"""The library's own launchers on pages and tables of the test's making: slots that no row has been written to, or that lie
behind the page's last row in its group of 8, hold NaN for certain; splits of a fixed number of steps give a token the bits it
has in any other chunk."""
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


class _Pages:
    """Pages of one layer, all bytes 0xff, with tables for K and V."""

    def __init__(self, kv_dim, page, tokens):
        self.kv_dim, self.page = kv_dim, page
        self.groups, self.blocks, self.pages = (page + 7) // 8, kv_dim // 32, math.ceil(tokens / page)
        self.slab = torch.full((2, self.pages, self.blocks * self.groups * 160), 0xff, dtype=torch.uint8, device="cuda")
        self.table = torch.tensor([[self.slab[w, i].data_ptr() for i in range(self.pages)] for w in range(2)], dtype=torch.int64,
                                  device="cuda")
        self.at = [self.table[w].data_ptr() for w in range(2)]
        self.write_, self.scratch, self.attn = _launchers()
        self.stream = torch.cuda.current_stream().cuda_stream

    def write(self, k, v, per):
        dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
        for pos in range(0, len(k), per):
            n = min(per, len(k) - pos)
            assert self.write_(*self.at, dk[pos:].data_ptr(), dv[pos:].data_ptr(), self.kv_dim, None, pos, n, self.kv_dim, self.page,
                               self.stream) == 0

    def attend(self, q, pos, n_kv, chunk):
        n, heads, hd = q.shape
        dq = torch.from_numpy(np.ascontiguousarray(q)).cuda()
        part = torch.full((max(1, self.scratch(pos + n, n, heads, n_kv, hd, self.page, chunk)),), math.nan, device="cuda")
        out = torch.full(q.shape, math.nan, device="cuda")
        assert self.attn(*self.at, dq.data_ptr(), heads * hd, part.data_ptr(), out.data_ptr(), None, pos, pos + n, n, heads, n_kv, hd,
                         self.kv_dim, self.page, chunk, self.stream) == 0
        torch.cuda.synchronize()
        return out.cpu().numpy()


@pytest.mark.parametrize("hd,n_kv,page", [(128, 2, 20), (64, 2, 20), (128, 1, 9), (64, 2, 33), (48, 2, 20), (288, 1, 13), (128, 2, 64)])
def test_slots_that_hold_nan(hd, n_kv, page):
    rng = np.random.default_rng(hd + page)
    rows, kv_dim = 1790, n_kv * hd
    p = _Pages(kv_dim, page, 1800)
    k, v = (rng.standard_normal((rows, kv_dim), dtype=np.float32) for _ in range(2))
    p.write(k, v, 179)  # 10 calls, whose ends lie inside groups
    # the steps and middles of slots that no row is in are NaN still, those of rows are not
    scales = p.slab[:, :, p.blocks * p.groups * 128:].cpu().numpy().view(np.float16).reshape(2, p.pages, p.blocks, p.groups, 2, 8)
    place = [(r & 3) * 2 + ((r >> 2) ^ (1 if r & 3 == 3 else 0)) for r in range(8)]
    scales = scales[..., place].transpose(0, 1, 3, 5, 4, 2).reshape(2, p.pages, p.groups * 8, 2, p.blocks)
    slot = np.arange(p.groups * 8)
    used = (slot < page) & (np.arange(p.pages)[:, None] * page + slot < rows)
    assert np.isnan(scales[:, ~used]).all() and np.isfinite(scales[:, used]).all()
    assert page % 8 == 0 or (~used[: p.pages - 1]).any()
    k, v = (q4_values(x).reshape(rows, n_kv, hd) for x in (k, v))
    for group, pos, n in ((1, rows - 1, 1), (4, rows - 5, 1), (2, 1000, 2), (8, 700, 3), (4, 1500, 200), (4, 1700, 90), (1, 3, 1), (3, 0, 40)):
        q = rng.standard_normal((n, group * n_kv, hd), dtype=np.float32) * np.float32(1.5)
        want = attend(q, k, v, pos, group)
        for chunk in (0, 16):
            got = p.attend(q, pos, n_kv, chunk)
            assert np.linalg.norm(got - want) <= REL * np.linalg.norm(want), (group, pos, n, chunk)


@pytest.mark.parametrize("hd,n_kv,page", [(128, 2, 128), (64, 4, 20), (64, 2, 32), (128, 1, 9), (96, 2, 64), (48, 4, 20), (256, 1, 128), (288, 1, 16)])
@pytest.mark.parametrize("size", ["even", "rows", "later"])
def test_a_tokens_bits_are_its_own(hd, n_kv, page, size):
    """Values of one size; of sizes that differ by row and block, so that the blocks' units fall again and again; of rows after
    the first tokens that are far wider, or NaN.  Each token of a chunk has the bits of smaller chunks and of a call of its own,
    with the later rows there or not."""
    rng = np.random.default_rng(hd + page)
    rows, kv_dim, group, pos = 1300, n_kv * hd, 3, 1130
    k, v = (rng.standard_normal((rows, kv_dim), dtype=np.float32) for _ in range(2))
    blocks = np.arange(kv_dim) // 32
    if size == "rows":
        v *= np.exp(rng.uniform(-11, 6, (rows, kv_dim // 32))).astype(np.float32)[:, blocks]
    elif size == "later":
        v *= np.float32(1e-3)
        v[1180:, blocks % 2 == 0] *= np.float32(1e6)
        v[1250, blocks % 3 == 1] = np.nan
    p = _Pages(kv_dim, page, rows + 50)
    q = rng.standard_normal((170, group * n_kv, hd), dtype=np.float32) * np.float32(1.5)
    q[100:120] *= np.float32(1e9)  # scores that have their maximum taken off first
    p.write(k[:1180], v[:1180], 300)
    early = p.attend(q[:50], pos, n_kv, 16)
    p.write(k, v, 300)
    whole = p.attend(q, pos, n_kv, 16)
    assert np.isfinite(whole[:120]).all()
    bits = lambda a: np.ascontiguousarray(a).view(np.uint32)
    nan = np.isnan(whole)
    assert (bits(early) == bits(whole[:50])).all()
    for at, n in ((0, 7), (7, 64), (71, 1), (72, 33), (105, 65), (49, 1), (169, 1), (3, 1)):
        got = p.attend(q[at:at + n], pos + at, n_kv, 16)
        w = nan[at:at + n]
        assert (np.isnan(got) == w).all() and (bits(got)[~w] == bits(whole[at:at + n])[~w]).all(), (at, n)
    kq, vq = (q4_values(x).reshape(rows, n_kv, hd) for x in (k, v))
    plain = np.r_[0:100]
    want = attend(q[plain], kq, vq, pos, group)
    if size != "later":
        assert np.linalg.norm(whole[plain] - want) <= REL * np.linalg.norm(want)
