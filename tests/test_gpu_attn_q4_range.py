"""Attention over a 4-bit cache where its numbers are far apart: blocks of values of different size, small query elements on
wide key channels, large queries; against attention in 64 bits over the values that the cache holds, block by block."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import attend, q4_values

pytestmark = pytest.mark.gpu

# As in test_gpu_attn_q4.py: 20 * (2^-22 + 4 * 2^-24) in a score in powers of two, times ln 2 and a fourth of it in the rms,
# and some 2^-22 for the weights' two fp16.  Nothing of it depends on how large a block's values are beside another's.
REL = 4e-6

# (heads, kv heads, hd, position, tokens): the 4 x 4 products, 16-row tiles (whole blocks, parts of blocks, eight blocks),
# 32-row tiles, heads beyond eight blocks; a token and a chunk; one split and several
CALLS = [(4, 1, 128, 1400, 1), (2, 2, 64, 1600, 1), (3, 1, 128, 1100, 1), (8, 1, 64, 1400, 1), (8, 2, 128, 300, 9), (6, 6, 48, 700, 1),
         (4, 2, 96, 500, 20), (2, 1, 256, 900, 1), (8, 2, 128, 1300, 100), (8, 2, 64, 1500, 150), (2, 1, 288, 200, 3)]


def _by_block(got, want, hd, rel, what):
    """The error of each block of 32 channels against that block's size."""
    n_kv = want.shape[1]
    block = (np.arange(n_kv)[:, None] * hd + np.arange(hd)) // 32
    for b in range(block.max() + 1):
        at = [(h, block[h] == b) for h in range(n_kv) if (block[h] == b).any()]
        g, w = (np.concatenate([a[:, h][:, :, m].ravel() for h, m in at]) for a in (got, want))
        err = np.linalg.norm(g - w) / np.linalg.norm(w)
        assert err <= rel, (what, b, err)


def _run(ctx, q, k, v, heads, n_kv, hd, pos, n, page=128):
    kv = ctx.kv_cache(1, n_kv * hd, page, pos + n, kv_type=capi.MVH_KV_Q4)
    kv.write(0, 0, k, v)
    got = kv.attn_batch(0, q.reshape(n, -1), pos, n, heads, n_kv, hd).reshape(n, n_kv, heads // n_kv, hd)
    kv.close()
    k, v = (q4_values(x).reshape(pos + n, n_kv, hd) for x in (k, v))
    return got, attend(q, k, v, pos, heads // n_kv).reshape(got.shape), k


@pytest.mark.parametrize("page", [128, 20])
@pytest.mark.parametrize("heads,n_kv,hd,pos,n", CALLS)
@pytest.mark.parametrize("sizes", [(1e-4,), (1e-5,), (30.0, 1e-3), (2000.0, 1e-2, 1.0), (1.0, 1e-5, 100.0, 1e-3)])
def test_blocks_of_different_size(ctx, heads, n_kv, hd, pos, n, page, sizes):
    rng = np.random.default_rng(hd + pos)
    k, v = (rng.standard_normal((pos + n, n_kv * hd), dtype=np.float32) for _ in range(2))
    v *= np.float32(sizes)[np.arange(n_kv * hd) // 32 % len(sizes)]
    q = rng.standard_normal((n, heads, hd), dtype=np.float32) * np.float32(1.5)
    got, want, _ = _run(ctx, q, k, v, heads, n_kv, hd, pos, n, page)
    _by_block(got, want, hd, REL, sizes)


@pytest.mark.parametrize("heads,n_kv,hd,pos,n", CALLS)
@pytest.mark.parametrize("at", [0, 100, -1])
def test_one_row_with_a_wide_block(ctx, heads, n_kv, hd, pos, n, at):
    """One seen row whose steps in every other block are above 2: the other blocks, small ones, keep their bits."""
    rng = np.random.default_rng(hd + pos + 1)
    k, v = (rng.standard_normal((pos + n, n_kv * hd), dtype=np.float32) for _ in range(2))
    v *= np.float32(0.01)
    v[at if at >= 0 else pos, np.arange(n_kv * hd) // 32 % 2 == 0] *= np.float32(1e5)
    q = rng.standard_normal((n, heads, hd), dtype=np.float32) * np.float32(1.5)
    got, want, _ = _run(ctx, q, k, v, heads, n_kv, hd, pos, n)
    _by_block(got, want, hd, REL, at)


@pytest.mark.parametrize("heads,n_kv,hd,pos,n", CALLS)
def test_first_row_takes_the_weight(ctx, heads, n_kv, hd, pos, n):
    """A first row that takes most of the weight and has next to no values, beside rows of e^-8 of its weight: the output is
    theirs.  A weight keeps 2^-35 of the largest one's, so these keep 2^-35 e^8 = 9e-8, with every other block's steps above 2
    all the same.  The first row's score (up to 16 in powers of two) is off by up to 16 (2^-22 + 4 * 2^-24), and ln 2 of that
    is a factor of the whole output: 5.3e-6 beside REL."""
    rng = np.random.default_rng(hd + pos + 2)
    k, v = (rng.standard_normal((pos + n, n_kv * hd), dtype=np.float32) for _ in range(2))
    k *= np.float32(0.25)
    v[:, np.arange(n_kv * hd) // 32 % 2 == 0] *= np.float32(40.0)
    v[0] *= np.float32(1e-7)
    q = rng.standard_normal((n, heads, hd), dtype=np.float32)
    # the first row's score is some 8 above the others' for every head: q has an even part that meets an even key
    q += np.float32(1.0)
    k[0] = np.float32(8.0 / np.sqrt(hd))
    got, want, _ = _run(ctx, q, k, v, heads, n_kv, hd, pos, n)
    _by_block(got, want, hd, REL + 5.3e-6, "")


@pytest.mark.parametrize("heads,n_kv,hd,pos,n", CALLS)
def test_small_queries_on_wide_keys(ctx, heads, n_kv, hd, pos, n):
    """Blocks of q a thousand times smaller than others, on keys as much wider: each block gives its share of the score."""
    rng = np.random.default_rng(hd + pos + 3)
    k, v = (rng.standard_normal((pos + n, n_kv * hd), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((n, heads, hd), dtype=np.float32) * np.float32(1.5)
    if hd % 32:  # blocks that heads share: a size per head's middle
        width = np.where(np.arange(n_kv * hd) // 32 % 2 == 0, np.float32(1000.0), np.float32(1.0))
    else:
        width = np.tile(np.float32([1000.0, 1.0, 30.0, 1.0, 200.0, 1.0, 1.0, 1000.0, 5.0])[: hd // 32].repeat(32), n_kv)
    k *= width
    q /= width.reshape(n_kv, hd).repeat(heads // n_kv, axis=0)
    got, want, _ = _run(ctx, q, k, v, heads, n_kv, hd, pos, n)
    _by_block(got, want, hd, REL, "")


@pytest.mark.parametrize("heads,n_kv,hd,pos,n", CALLS + [(1, 1, 128, 1022, 4), (1, 1, 64, 1021, 4), (8, 2, 128, 20, 40), (4, 2, 128, 0, 300)])
@pytest.mark.parametrize("size,low", [(1e9, False), (1e28, False), (1e34, False), (1e14, True), (1e20, True)])
def test_large_queries(ctx, heads, n_kv, hd, pos, n, size, low):
    """Queries whose scores are far from 0 (from 1e9 on, all of them below -1e12 or not) and finite: one row takes all the
    weight."""
    rng = np.random.default_rng(hd + pos + 4)
    k, v = (rng.standard_normal((pos + n, n_kv * hd), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((n, heads, hd), dtype=np.float32)
    if low:
        k -= np.float32(3.0)
        q = abs(q) + np.float32(0.5)
    q *= np.float32(size)
    got, want, k = _run(ctx, q, k, v, heads, n_kv, hd, pos, n)
    assert np.isfinite(got).all()
    # where the two best scores are clear of each other (2^-20 of the score's terms), the output is the best row's values
    clear = 0
    for t in range(n):
        for h in range(heads):
            s = np.sort((k[: pos + t + 1, h // (heads // n_kv)].astype(np.float64) @ q[t, h].astype(np.float64)))
            if len(s) > 1 and s[-1] - s[-2] < 2.0 ** -20 * hd * 6 * size:
                continue
            g, w = got[t].reshape(heads, hd)[h], want[t].reshape(heads, hd)[h]
            assert abs(g - w).max() <= 2.0 ** -20 * abs(w).max(), (t, h)
            clear += 1
    assert clear >= n * heads // 2
