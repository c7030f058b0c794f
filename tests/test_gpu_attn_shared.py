"""Attention of a batch of sequences behind a shared prefix, against 64 bits over the stored rows."""
import numpy as np
import pytest

from batch_ops import attend_shared
from memvanta_amd import capi

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F = np.float32
F16, Q8 = capi.MVH_KV_F16, capi.MVH_KV_Q8


class _Batch:
    """A prefix cache and a cache per sequence, filled with random rows, and what they hold."""

    def __init__(self, ctx, rng, kv_type, prefix, pos, n_tokens, heads, kv_heads, hd, page=16, p_page=None, layers=1,
                 spare=0, value=None):
        self.ctx, self.heads, self.kv_heads, self.hd = ctx, heads, kv_heads, hd
        self.prefix_len, self.pos, self.n = prefix, list(pos), list(n_tokens)
        self.layer = layers - 1
        kv_dim = kv_heads * hd + spare
        rows = lambda n: [(rng.standard_normal((n, kv_dim)) + rng.standard_normal(kv_dim)).astype(F) for _ in range(2)]
        self.prefix, self.held = None, (np.zeros((0, kv_heads * hd)),) * 2
        if prefix:
            self.prefix = ctx.kv_cache(layers, kv_dim, p_page or page, prefix + 3, kv_type)
            self.held = self.fill(self.prefix, 0, *(value(*rows(prefix)) if value else rows(prefix)))
        self.kvs, self.own = [], []
        for p, n in zip(pos, n_tokens):
            kv = ctx.kv_cache(layers, kv_dim, page, max(1, p + n), kv_type)
            end = p + n if n else prefix
            self.kvs.append(kv)
            r = rows(end - prefix)
            self.own.append(self.fill(kv, prefix, *(value(*r) if value else r)))
        self.q = (1.5 * rng.standard_normal((sum(n_tokens), heads * hd))).astype(F)

    def fill(self, kv, pos, k, v):
        if not len(k):
            return (np.zeros((0, self.kv_heads * self.hd)),) * 2
        kv.write(self.layer, pos, k, v)
        return [x[:, : self.kv_heads * self.hd] for x in kv.read(self.layer, pos, len(k))]

    def run(self, q=None, **more):
        n = None if all(n == 1 for n in self.n) else self.n
        return self.ctx.attn_shared(self.kvs, self.layer, self.q if q is None else q, self.pos, self.heads, self.kv_heads,
                                    self.hd, prefix=self.prefix, prefix_len=self.prefix_len, n_tokens=n, **more)

    def want(self, q=None):
        return attend_shared(self.q if q is None else q, self.held, self.own, self.pos, self.n, self.heads, self.kv_heads)

    def check(self, q=None):
        off = _off(self.run(q), *self.want(q))
        assert off <= 1

    def close(self):
        for kv in self.kvs + ([self.prefix] if self.prefix else []):
            kv.close()


def _off(got, want, size, scores=16.0):
    """The largest error over its bound.  q and weights keep 22 bits, products and sums round 24: a score of `scores` (in
    units of 1, its sum of magnitudes four times that) is off by 4 * 2^-22 of it and its weight by as much, the weighted sum
    by that and 2^-22 for the weight's own bits, 8 * 2^-24 for its sums, exponent and quotient."""
    bound = (2 * 4 * scores * 2.0 ** -22 + 4 * 2.0 ** -22) * size
    fine = np.isfinite(want)  # a stored infinity, of a value beyond fp16, leaves no number
    assert (np.isfinite(got) == fine).all()
    return float((abs(got.astype(np.float64) - want)[fine] / (bound[fine] + 1e-300)).max())


SHAPES = [(4, 2, 64), (6, 6, 48), (8, 1, 128), (32, 4, 64), (2, 2, 256), (3, 3, 8), (4, 4, 200), (5, 1, 72)]


@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("prefix,seqs", [(0, 3), (1, 1), (37, 2), (300, 5), (129, 40)])
def test_tokens(ctx, kv_type, heads, kv_heads, hd, prefix, seqs):
    rng = np.random.default_rng(prefix + hd)
    pos = [prefix + int(x) for x in rng.integers(0, 200, seqs)]
    pos[0] = prefix
    b = _Batch(ctx, rng, kv_type, prefix, pos, [1] * seqs, heads, kv_heads, hd)
    b.check()
    b.close()


@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("prefix,n_tokens", [(0, [3, 1]), (70, [2, 0, 5, 1]), (33, [65, 1, 40]), (5, [150])])
def test_chunks(ctx, kv_type, heads, kv_heads, hd, prefix, n_tokens):
    rng = np.random.default_rng(prefix + hd)
    pos = [prefix + int(x) for x in rng.integers(0, 60, len(n_tokens))]
    pos[-1] = prefix
    b = _Batch(ctx, rng, kv_type, prefix, pos, n_tokens, heads, kv_heads, hd)
    b.check()
    b.close()


@pytest.mark.parametrize("page,p_page", [(1, 1), (1, 128), (3, 20), (20, 7), (128, 16), (20000, 20000), (1000, 3)])
def test_pages(ctx, page, p_page):
    rng = np.random.default_rng(page)
    b = _Batch(ctx, rng, F16, 777, [777 + 600, 777, 777 + 33], [1, 1, 3], 4, 2, 64, page=page, p_page=p_page, layers=2)
    b.check()
    b.close()


@pytest.mark.parametrize("kv_type", [F16, Q8])
def test_long(ctx, kv_type):
    """A prefix near the caches' end, many parts; and a long cache of its own behind a short prefix."""
    rng = np.random.default_rng(5)
    b = _Batch(ctx, rng, kv_type, 15000, [15000 + i * 7 for i in range(9)], [1] * 9, 8, 2, 64, page=128)
    b.check()
    b.close()
    b = _Batch(ctx, rng, kv_type, 3, [15900, 40], [1, 1], 8, 2, 64, page=16)
    b.check()
    b.close()


def test_many_sequences(ctx):
    """More sequences than one launch takes, some without a token, some sharing a cache."""
    rng = np.random.default_rng(6)
    n = [int(x) for x in rng.integers(0, 3, 300)]
    b = _Batch(ctx, rng, F16, 50, [50 + int(x) for x in rng.integers(0, 30, 300)], n, 2, 1, 64)
    b.check()
    same = b.kvs[n.index(2)]
    at = b.pos[n.index(2)]
    q = np.repeat(b.q[:1], 4, 0)
    got = ctx.attn_shared([same] * 4, 0, q, [at, at + 1, at, at + 1], 2, 1, 64, prefix=b.prefix, prefix_len=50)
    assert (got[0] == got[2]).all() and (got[1] == got[3]).all() and (got[0] != got[1]).any()
    b.close()


def test_row_wider_than_the_heads(ctx):
    rng = np.random.default_rng(7)
    for kv_type in (F16, Q8):
        b = _Batch(ctx, rng, kv_type, 40, [45, 60], [1, 2], 4, 2, 64, spare=24)
        b.check()
        b.close()


def test_same_as_one_sequence(ctx):
    """A prefix and a sequence's own rows against the attention over one cache that holds both."""
    rng = np.random.default_rng(8)
    b = _Batch(ctx, rng, F16, 100, [160], [1], 8, 2, 64)
    whole = ctx.kv_cache(1, 128, 16, 200, F16)
    whole.write(0, 0, b.held[0], b.held[1])
    whole.write(0, 100, b.own[0][0], b.own[0][1])
    one = whole.attn_decode(0, b.q[0], 160, 8, 2, 64)
    assert abs(b.run()[0] - one).max() <= 1e-5 * abs(one).max()
    # the cache of both as prefix and as the sequence's
    both = ctx.attn_shared([whole], 0, b.q, [160], 8, 2, 64, prefix=whole, prefix_len=100)
    assert (both == b.run()).all()
    whole.close()
    b.close()


@pytest.mark.parametrize("size", [1e-3, 1.0, 300.0, 1e4])
def test_sizes(ctx, size):
    """Queries, keys and values of very different sizes; the peak of the softmax may be one row."""
    rng = np.random.default_rng(9)
    for kv_type in (F16, Q8):
        b = _Batch(ctx, rng, kv_type, 90, [130, 95], [1, 4], 4, 2, 64, value=lambda k, v: (k / F(size), v * F(size)))
        q = (b.q * F(size)).astype(F)
        b.check(q)
        b.close()


def test_large_scores(ctx):
    """One query element that outweighs the others of its head by 2^60: scores beyond 2^58, one row takes all; the other head
    as ever."""
    rng = np.random.default_rng(10)
    for kv_type in (F16, Q8):
        b = _Batch(ctx, rng, kv_type, 64, [99], [1], 2, 2, 64)
        q = b.q.copy()
        q[:, 3] *= F(2.0 ** 60)
        got, (want, size) = b.run(q), b.want(q)
        k, v = (np.concatenate([b.held[i], b.own[0][i]]).reshape(-1, 2, 64)[:, 0] for i in range(2))
        best = (k[:, 3].astype(np.float64) * q[0, 3]).argmax()
        assert abs(got[0, :64] - v[best]).max() <= 2.0 ** -20 * abs(v[best]).max()
        assert _off(got[:, 64:], want[:, 64:], size[:, 64:]) <= 1
        b.close()


@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("power", range(20, 34, 2))
def test_scores_coarser_than_weights(ctx, kv_type, power):
    """Scores whose last bit stands for a factor of 2^-2 to 2^12 of a weight: still one row that takes all."""
    rng = np.random.default_rng(17)
    for seed in range(4):
        b = _Batch(ctx, rng, kv_type, 64, [99], [1], 2, 2, 64)
        q = b.q.copy()
        q[:, 3] = F(2.0 ** power * rng.uniform(1, 2))
        got = b.run(q)
        k, v = (np.concatenate([b.held[i], b.own[0][i]]).reshape(-1, 2, 64)[:, 0] for i in range(2))
        s = (k.astype(np.float64) * q[0, :64]).sum(1) / 8
        best = s.argmax()
        if s[best] - np.sort(s)[-2] > 2.0 ** -20 * s[best] + 50:  # beyond what fp32 sums leave in doubt
            assert abs(got[0, :64] - v[best]).max() <= 2.0 ** -20 * abs(v[best]).max()
        b.close()


def test_rows_of_different_sizes_q8(ctx):
    """Rows whose scales differ by powers of ten, the wide ones late."""
    rng = np.random.default_rng(11)
    def value(k, v):
        s = (10.0 ** rng.uniform(-4, 0, (len(v), 1))).astype(F)
        s[len(v) // 2:] *= 100
        return k, v * s
    b = _Batch(ctx, rng, Q8, 150, [200, 170], [1, 3], 4, 2, 64, value=value)
    b.check()
    b.close()


@pytest.mark.parametrize("kv_type", [F16, Q8])
@pytest.mark.parametrize("n_tokens", [[1, 1], [6, 3], [40, 9]])
def test_slots_that_hold_nan(ctx, kv_type, n_tokens):
    """What a token does not see may be NaN or an infinity: rows behind it in its cache, a later token's row, the pages'
    rows below the prefix's end, the prefix's rows behind its end."""
    rng = np.random.default_rng(12)
    b = _Batch(ctx, rng, kv_type, 21, [30, 23], n_tokens, 8, 2, 64, page=16)
    for bad in (np.nan, np.inf):
        for kv, p, n in zip(b.kvs, b.pos, b.n):
            rows = np.full((2, 128), bad, F)
            kv.write(0, 16, np.repeat(rows, 3, 0)[:5], np.repeat(rows, 3, 0)[:5])
        b.prefix.write(0, 21, np.full((3, 128), bad, F), np.full((3, 128), bad, F))
        b.check()
    # the last token's row of sequence 0: that token alone
    if n_tokens[0] > 1:
        k, v = np.zeros((1, 128), F), np.zeros((1, 128), F)
        v[0, 5], v[0, 70] = np.nan, np.inf
        b.kvs[0].write(0, b.pos[0] + b.n[0] - 1, k, v)
        got, (want, size) = b.run(), b.want()
        last = b.n[0] - 1
        keep = np.arange(len(got)) != last
        assert _off(got[keep], want[keep], size[keep]) <= 1
        head = got[last].reshape(8, 64)
        assert not np.isfinite(head[:4, 5]).any() and not np.isfinite(head[4:, 6]).any()
    b.close()


def test_nan_that_is_seen(ctx):
    """A NaN in a row (an infinity, once stored as fp16) leaves its sequence no number in that channel, and others theirs."""
    rng = np.random.default_rng(13)
    b = _Batch(ctx, rng, F16, 40, [60, 50, 44], [1, 1, 1], 4, 2, 64)
    k, v = (x[:1].astype(F).copy() for x in b.own[1])
    v[0, 9] = np.nan
    b.kvs[1].write(0, 40, k, v)
    got = b.run().reshape(3, 4, 64)
    bad = np.zeros_like(got, bool)
    bad[1, :2, 9] = True
    assert (np.isfinite(got) == ~bad).all()
    b.close()


def test_what_lies_around(ctx):
    rng = np.random.default_rng(14)
    for n in ([1, 1, 1], [3, 0, 40]):
        b = _Batch(ctx, rng, F16, 30, [33, 30, 50], n, 6, 6, 48)
        rows = sum(n)
        out = torch.full((rows + 2, 288), 7.0, device="cuda")
        q = torch.full((rows + 2, 288), float("nan"), device="cuda")
        q[1:-1] = torch.from_numpy(b.q).cuda()
        torch.cuda.synchronize()
        b.run(q[1:-1], out=out[1:-1])
        ctx.synchronize()
        y = out.cpu().numpy()
        assert (y[[0, -1]] == 7).all() and (y[1:-1] == b.run()).all()
        b.close()


def test_captured(ctx):
    """Captured after a call of its size, replayed with new queries and eager calls of other sizes between the replays."""
    rng = np.random.default_rng(15)
    own = capi.Context(0)
    stream = torch.cuda.ExternalStream(own.stream)
    b = _Batch(own, rng, F16, 300, [310, 420, 300], [1, 1, 1], 8, 2, 64)
    big = _Batch(own, rng, F16, 900, [1000 + i for i in range(30)], [1] * 30, 8, 2, 64)
    q, out = torch.zeros((3, 512), device="cuda"), torch.zeros((3, 512), device="cuda")
    torch.cuda.synchronize()
    fresh = capi.Context(0)
    with pytest.raises(capi.MvhError, match="before capturing"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(fresh.stream)):
            fresh.attn_shared(b.kvs, 0, q, b.pos, 8, 2, 64, out=out, prefix=b.prefix, prefix_len=300)
    b.run(q, out=out)
    own.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        b.run(q, out=out)
    for i in range(4):
        rows = rng.standard_normal((3, 512)).astype(F)
        q.copy_(torch.from_numpy(rows))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert (out.cpu().numpy() == b.run(rows)).all(), i
        big.run()
    for x in (b, big, fresh, own):
        x.close()


def test_refusals(ctx):
    rng = np.random.default_rng(16)
    b = _Batch(ctx, rng, F16, 20, [25, 30], [1, 1], 4, 2, 64)
    q, go = b.q, lambda **k: ctx.attn_shared(**{**dict(kvs=b.kvs, layer=0, q=b.q, pos=b.pos, n_head=4, n_head_kv=2,
                                                       head_dim=64, prefix=b.prefix, prefix_len=20), **k})
    assert (go() == b.run()).all()
    other = {"page": ctx.kv_cache(1, 128, 8, 64), "dim": ctx.kv_cache(1, 256, 16, 64), "type": ctx.kv_cache(1, 128, 16, 64, Q8),
             "f32": ctx.kv_cache(1, 128, 16, 64, capi.MVH_KV_F32), "q4": ctx.kv_cache(1, 128, 16, 64, capi.MVH_KV_Q4)}
    for kv in other.values():
        kv.write(0, 0, np.zeros((40, kv.kv_dim), F), np.zeros((40, kv.kv_dim), F))
    for name, match in (("page", "page sizes"), ("dim", "different types or kv_dim"), ("type", "different types or kv_dim"),
                        ("f32", "F16 and Q8"), ("q4", "F16 and Q8")):
        with pytest.raises(capi.MvhError, match=match):
            go(kvs=[b.kvs[0], other[name]])
    for more, match in ((dict(pos=[25, 19]), "lies in the prefix"), (dict(pos=[25, 99]), "context exhausted"),
                        (dict(layer=1), "layer 1"), (dict(prefix=None), "null KV cache"), (dict(prefix_len=24), "context exhausted|page missing|lies"),
                        (dict(n_head_kv=3), "head configuration"), (dict(head_dim=60), "multiple of 8"),
                        (dict(head_dim=264, q=np.zeros((2, 4 * 264), F)), "multiple of 8 up to 256"),
                        (dict(head_dim=128, q=np.zeros((2, 512), F)), "<= kv_dim"), (dict(prefix_len=2 ** 40), "exhausted|lies")):
        with pytest.raises(capi.MvhError, match=match):
            go(**more)
    empty = ctx.kv_cache(1, 128, 16, 64)
    with pytest.raises(capi.MvhError, match="page missing"):
        go(kvs=[b.kvs[0], empty])
    with pytest.raises(capi.MvhError, match="page missing"):
        go(prefix=empty)
    for bad in (dict(pos=[25]), dict(n_tokens=[1]), dict(pos=[25, -1]), dict(q=q[:1]), dict(out=torch.zeros((2, 256), device="cuda"))):
        with pytest.raises(ValueError):
            go(**bad)
    assert go(n_tokens=[0, 0], q=np.zeros((0, 256), F)).size == 0
    flat = torch.zeros(2 * 256 + 1, device="cuda")
    with pytest.raises(capi.MvhError, match="16-byte aligned"):
        go(q=flat[1:].reshape(2, 256), out=torch.zeros((2, 256), device="cuda"))
    flat = torch.zeros(1024, device="cuda")
    with pytest.raises(capi.MvhError, match="must not overlap"):
        go(q=flat[:512].reshape(2, 256), out=flat[508:1020].reshape(2, 256))
    for kv in (*other.values(), empty):
        kv.close()
    b.close()
