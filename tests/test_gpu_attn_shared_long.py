"""Attention behind a shared prefix in parts of many rows: a part of more than 128 rows goes round its loop of tiles again, one of
more than 256 takes row addresses and scales from the next turn of their ring, against 64 bits over the stored rows.

A part has about len / ceil(256 / (tiles of query rows * kv heads)) rows of the prefix for tokens one by one, len / (512 / that)
for chunks, rounded up to 128s; of own rows all where the batch has 512 or more (sequence, kv head, tile).  What the cases' parts
hold is noted with them."""
import numpy as np
import pytest

from memvanta_amd import capi
from test_gpu_attn_shared import F16, Q8, _Batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _attend(b):
    """attend_shared of all tokens of a head at once: outputs and the sums of magnitudes, [token][head][hd]."""
    group, n = b.heads // b.kv_heads, len(b.q)
    cut = lambda x: np.ascontiguousarray(x.astype(np.float64).reshape(len(x), b.kv_heads, b.hd).transpose(1, 0, 2))
    q = b.q.astype(np.float64).reshape(n, b.kv_heads, group, b.hd).transpose(1, 0, 2, 3) / np.sqrt(b.hd)
    pk, pv = map(cut, b.held)
    own = [tuple(map(cut, kv)) for kv in b.own]
    out, size = np.empty((n, b.kv_heads, group, b.hd)), np.empty((n, b.kv_heads, group, b.hd))
    for g in range(b.kv_heads):
        first = q[g].reshape(n * group, b.hd) @ pk[g].T
        at = 0
        for (k, v), count in zip(own, b.n):
            rows = slice(at * group, (at + count) * group)
            s = q[g].reshape(n * group, b.hd)[rows] @ k[g].T
            last = s.shape[1] - count + np.arange(count).repeat(group)
            s[np.arange(s.shape[1])[None] > last[:, None]] = -np.inf
            s = np.concatenate([first[rows], s], 1)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            both = np.concatenate([pv[g], v[g]])
            out[at:at + count, g] = (w @ both).reshape(count, group, b.hd)
            size[at:at + count, g] = (w @ np.abs(both)).reshape(count, group, b.hd)
            at += count
    return out, size


def _check(b, longest):
    """q and weights keep 22 bits: a score up to 16 of four times that in magnitudes is off by 2^-22 of those, its weight by as much,
    once in a sum and once in its divisor, and by 4 * 2^-22 for its own bits; sums of a part of `longest` rows add longest / 4
    weights a lane, and longest / 16 products, rounded or cut, then a handful of parts."""
    got = b.run().reshape(len(b.q), b.kv_heads, b.heads // b.kv_heads, b.hd)
    want, size = _attend(b)
    bound = ((2 * 4 * 16 + 4) * 2.0 ** -22 + (longest / 4 + longest / 8 + 128) * 2.0 ** -24) * size
    off = np.abs(got - want) / bound
    assert off.max() <= 1, (float(off.max()), np.unravel_index(off.argmax(), off.shape))


# own rows of 64 sequences: parts that end at, before and just behind a turn of the ring
OWN = [1, 255, 256, 257, 384, 511, 512, 513, 700, 767, 768, 769, 900, 64, 129, 320]


# 64 tokens of 32 heads on 8: 16 parts of the prefix, of 128s; the last one ends just behind 256, 512 and 768
@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("prefix,chunk", [(15 * 384 + 257, 384), (15 * 640 + 513, 640), (15 * 896 + 769, 896)])
def test_many_tokens(ctx, kv_type, prefix, chunk):
    rng = np.random.default_rng(prefix)
    b = _Batch(ctx, rng, kv_type, prefix, [prefix + OWN[i % 16] - 1 for i in range(64)], [1] * 64, 32, 8, 64, page=(16, 20)[prefix % 2],
               p_page=128)
    _check(b, max(chunk, 900))
    b.close()


# the other sizes of heads, among them one whose last channels a tile only pads
@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("hd", [72, 128, 256])
def test_many_tokens_of_wide_heads(ctx, kv_type, hd):
    rng = np.random.default_rng(hd)
    prefix = 6017  # 16 parts of 384 rows, of heads of 256, whose tiles are of 64 query rows, 8 of 768
    b = _Batch(ctx, rng, kv_type, prefix, [prefix + OWN[i % 16] - 1 for i in range(64)], [1] * 64, 32, 8, hd, page=16, p_page=128)
    _check(b, 900)
    b.close()


# 32 tokens of a kv head a head: tiles of 32 query rows, 8 parts of the prefix of 640 and 1280 rows
@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("hd,prefix", [(64, 7 * 1280 + 257), (128, 7 * 640 + 513)])
def test_tiles_of_32_rows(ctx, kv_type, hd, prefix):
    rng = np.random.default_rng(hd)
    b = _Batch(ctx, rng, kv_type, prefix, [prefix + OWN[i % 16] - 1 for i in range(32)], [1] * 32, 32, 32, hd, page=16, p_page=20)
    _check(b, 1280)
    b.close()


# one and four tokens: tiles of 16 query rows, 29 parts of 512 rows, whose steps are of 128; few own parts of up to 128 rows
@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("seqs", [1, 4])
def test_tiles_of_16_rows(ctx, kv_type, seqs):
    rng = np.random.default_rng(seqs)
    b = _Batch(ctx, rng, kv_type, 14593, [14593 + 300 + i for i in range(seqs)], [1] * seqs, 32, 8, 64, page=128)
    _check(b, 512)
    b.close()


# chunks: 2280 query rows of a kv head in 18 or 36 tiles, the prefix in three parts of 1024 or, of heads of 256,
# in one; own rows in parts of 512
@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("hd", [64, 72, 128, 256])
def test_chunks(ctx, kv_type, hd):
    rng = np.random.default_rng(hd)
    n = [75 - 5 * i for i in range(12)]
    own = [0, 900, 257, 512 - 65, 60, 513 - 55, 1, 769, 300, 256, 20, 511]
    b = _Batch(ctx, rng, kv_type, 3001, [3001 + o for o in own], n, 32, 8, hd, page=16, p_page=128)
    _check(b, 3001)
    b.close()


def test_again(ctx):
    """The same batch again gives the same bits."""
    rng = np.random.default_rng(3)
    for n in ([1] * 64, [40] * 12):
        b = _Batch(ctx, rng, F16, 9000, [9000 + OWN[i % 16] - 1 for i in range(len(n))], n, 32, 8, 128, page=16, p_page=128)
        q, out = torch.from_numpy(b.q).cuda(), torch.empty(b.q.shape, device="cuda")
        torch.cuda.synchronize()
        b.run(q, out=out)
        ctx.synchronize()
        first = out.clone()
        torch.cuda.synchronize()
        for i in range(8):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            b.run(q, out=out)
            ctx.synchronize()
            assert torch.equal(out, first), i
        b.close()
