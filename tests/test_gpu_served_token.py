"""The served token's operators together, as a program calls them: projections, rotated append, attention, log
probabilities; captured into graphs and replayed; side by side on two contexts; and whole models on a 4-bit cache."""
import numpy as np
import pytest

from memvanta_amd import capi, synth
from served_ops import angles, attend, log_softmax, rotate

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HEADS, KV_HEADS, HD, DIM, VOCAB = 8, 2, 64, 256, 700
KV_DIM = KV_HEADS * HD


class _Net:
    """Two layers of attention alone (F32 weights) and an output head, on the calls of one context."""

    def __init__(self, ctx, rng, kv_type, scaling):
        self.ctx, f = ctx, np.float32
        w = lambda rows, cols: (rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(f)
        self.wqkv = [w(HEADS * HD + 2 * KV_DIM, DIM) for _ in range(2)]
        self.wo = [w(DIM, HEADS * HD) for _ in range(2)]
        self.head = w(VOCAB, DIM)
        up = lambda m: ctx.upload("w", synth.F32, m.shape[1], m.shape[0], m.view(np.uint8))
        self.tqkv, self.to, self.thead = [up(m) for m in self.wqkv], [up(m) for m in self.wo], up(self.head)
        self.options = dict(scaling=scaling, base=500000.0, factor=8.0, orig_ctx=64.0, low=1.0, high=4.0)
        self.rope = ctx.rope(HD, rot_dim=48, layout=1, **self.options)
        self.kv = ctx.kv_cache(2, KV_DIM, 16, 128, kv_type=kv_type)

    def buffers(self, n):
        e = lambda *s: torch.zeros(s, device="cuda")
        return {"x": e(n, DIM), "qkv": [e(n, HEADS * HD + 2 * KV_DIM) for _ in range(2)], "q": e(n, HEADS * HD),
                "att": [e(n, HEADS * HD) for _ in range(2)], "y": [e(n, DIM) for _ in range(2)], "logits": e(n, VOCAB),
                "lp": e(n), "entropy": e(n), "ids": torch.zeros((n, 4), dtype=torch.int32, device="cuda"), "top": e(n, 4),
                "targets": torch.zeros(n, dtype=torch.int32, device="cuda")}

    def step(self, b, pos):
        """The step's calls, on device buffers."""
        x, n = b["x"], b["x"].shape[0]
        for layer in range(2):
            self.ctx.matmul_batch(self.tqkv[layer], x, b["qkv"][layer])
            qkv = b["qkv"][layer]
            self.kv.append(layer, pos, qkv[:, HEADS * HD:-KV_DIM], qkv[:, -KV_DIM:], self.rope, q=qkv[:, :HEADS * HD],
                           q_out=b["q"])
            if n == 1:
                self.kv.attn_decode(layer, b["q"], pos, HEADS, KV_HEADS, HD, b["att"][layer])
            else:
                self.kv.attn_batch(layer, b["q"], pos, n, HEADS, KV_HEADS, HD, b["att"][layer])
            self.ctx.matmul_batch(self.to[layer], b["att"][layer], b["y"][layer])
            x = b["y"][layer]
        self.ctx.matmul_batch(self.thead, x, b["logits"])
        self.ctx.logprobs(b["logits"], b["targets"], 4, b["lp"], b["entropy"], b["ids"], b["top"])

    def check(self, b, pos):
        """Each operator's output against 64 bits from its own input."""
        n = b["x"].shape[0]
        o = dict(self.options)
        if not o["scaling"]:
            o.update(factor=1.0)
        f = angles(48, **o)
        at = np.arange(pos, pos + n)
        x = b["x"].cpu().numpy()
        for layer in range(2):
            qkv = b["qkv"][layer].cpu().numpy()
            want = x.astype(np.float64) @ self.wqkv[layer].T
            assert np.linalg.norm(qkv - want) <= 1e-5 * np.linalg.norm(want)
            q, _ = rotate(qkv[:, :HEADS * HD].reshape(n, HEADS, HD), at, f, 48, True)
            k, _ = rotate(qkv[:, HEADS * HD:-KV_DIM].reshape(n, KV_HEADS, HD), at, f, 48, True)
            rk, rv = self.kv.read(layer, 0, pos + n)
            v = qkv[:, -KV_DIM:]
            if self.kv.kv_type == capi.MVH_KV_F16:
                # a mantissa that rounds up to the next power of two is OR-ed into the exponent (1.9999 is stored as 1),
                # so the distance has no useful bound: the stored rows are the conversion's, bit for bit
                turned = self.rope.apply(np.ascontiguousarray(qkv[:, HEADS * HD:-KV_DIM]), KV_HEADS, pos=pos)
                for rows, x32 in ((rk, turned), (rv, v)):
                    half = self.ctx.fp16_to_fp32(self.ctx.fp32_to_fp16(np.ascontiguousarray(x32)))
                    assert (rows[pos:].reshape(-1) == half).all()
            else:
                step = {0: 1e-6, 2: 1 / 100, 3: 1 / 6}[self.kv.kv_type]  # half a step of the widest block
                assert abs(rk[pos:].reshape(k.shape) - k).max() <= step * abs(k).max()
                assert abs(rv[pos:] - v).max() <= step * abs(v).max()
            got = b["att"][layer].cpu().numpy().reshape(n, HEADS, HD)
            want = attend(q, rk.reshape(-1, KV_HEADS, HD), rv.reshape(-1, KV_HEADS, HD), pos, HEADS // KV_HEADS)
            assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want), layer
            x = b["y"][layer].cpu().numpy()
        logits = b["logits"].cpu().numpy()
        lp = log_softmax(logits)
        assert abs(b["lp"].cpu().numpy() - lp[np.arange(n), b["targets"].cpu().numpy()]).max() <= 5e-6
        assert (b["ids"].cpu().numpy() == np.argsort(-logits, axis=1, kind="stable")[:, :4]).all()
        assert (b["ids"].cpu().numpy()[:, 0] == self.ctx.argmax(logits)).all()

    def close(self):
        for t in (*self.tqkv, *self.to, self.thead):
            t.free()
        self.kv.close()
        self.rope.close()


def _fill(b, rng):
    b["x"].copy_(torch.from_numpy(rng.standard_normal(tuple(b["x"].shape)).astype(np.float32)))
    b["targets"].copy_(torch.from_numpy(rng.integers(0, VOCAB, len(b["targets"])).astype(np.int32)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("kv_type", [0, 1, 2, 3])
@pytest.mark.parametrize("scaling", [0, 2])
def test_prompt_then_tokens(ctx, kv_type, scaling):
    rng = np.random.default_rng(kv_type)
    net = _Net(ctx, rng, kv_type, scaling)
    pos = 0
    for n in (37, 1, 1, 20, 1, 3):
        b = net.buffers(n)
        _fill(b, rng)
        net.step(b, pos)
        ctx.synchronize()
        net.check(b, pos)
        pos += n
    net.close()


def test_captured_step(ctx):
    """A step captured into a graph and replayed with other inputs, eager calls of another size between the replays; a call
    whose workspace is not there yet is refused under capture and leaves the context usable."""
    rng = np.random.default_rng(3)
    c = capi.Context(0)
    net = _Net(c, rng, capi.MVH_KV_Q4, 2)
    prompt, one = net.buffers(90), net.buffers(1)
    _fill(prompt, rng)
    net.step(prompt, 0)
    _fill(one, rng)
    net.step(one, 90)  # once before the capture: the page of position 90 and the workspace are there
    c.synchronize()
    stream = torch.cuda.ExternalStream(c.stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        net.step(one, 90)
    for _ in range(3):
        _fill(one, rng)
        with torch.cuda.stream(stream):
            g.replay()
        c.synchronize()
        net.check(one, 90)
        got = one["lp"].clone()
        net.step(one, 90)
        c.synchronize()
        assert torch.equal(got, one["lp"])
        wide = torch.randn(3, 200000, device="cuda")  # a larger workspace: the graph's stays where it is
        out = torch.empty(3, device="cuda")
        torch.cuda.synchronize()
        c.logprobs(wide, None, 64, None, out, torch.empty((3, 64), dtype=torch.int32, device="cuda"), None)
        c.synchronize()
    del g
    net.close()
    c.close()


def test_no_workspace_under_capture():
    c = capi.Context(0)
    x = torch.randn(1, 200000, device="cuda")  # long enough for parts, which take a workspace
    out, y = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.ExternalStream(c.stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        with pytest.raises(capi.MvhError, match="before capturing") as e:
            c.logprobs(x, None, 0, None, out)
        assert e.value.code == 6
    del g
    c.logprobs(x, None, 0, None, out)
    c.synchronize()
    want = -(torch.softmax(x.double(), 1) * torch.log_softmax(x.double(), 1)).sum()
    assert abs(out.item() - want.item()) < 1e-4
    c.close()


def test_no_page_under_capture():
    """A position whose page is not there cannot be captured, also where freed pages wait; it is missing afterwards too."""
    c = capi.Context(0)
    kv = c.kv_cache(1, 64, 8, 64, kv_type=capi.MVH_KV_Q4)
    rope = c.rope(64)
    rows = torch.randn(16, 64, device="cuda")
    out = torch.empty(64, device="cuda")
    torch.cuda.synchronize()
    kv.append(0, 0, rows, rows, rope)
    c.synchronize()
    kv.reset()  # the pages of positions 0..15 are free ones now
    kv.append(0, 0, rows[:8], rows[:8], rope)
    stream = torch.cuda.ExternalStream(c.stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        with pytest.raises(capi.MvhError, match="before capturing") as e:
            kv.append(0, 8, rows[8:], rows[8:], rope)
        assert e.value.code == 6
        kv.attn_decode(0, rows[0], 7, 1, 1, 64, out)
    with pytest.raises(capi.MvhError, match="missing"):
        kv.attn_decode(0, rows[0], 8, 1, 1, 64, out)
    with torch.cuda.stream(stream):
        g.replay()
    c.synchronize()
    captured = out.clone()
    kv.append(0, 8, rows[8:], rows[8:], rope)
    kv.attn_decode(0, rows[0], 7, 1, 1, 64, out)
    c.synchronize()
    assert torch.equal(out, captured)
    del g
    kv.close()
    rope.close()
    c.close()


def test_two_contexts(ctx):
    """Two contexts' steps in flight together give the bits of each alone."""
    other = capi.Context(0)
    rng = np.random.default_rng(8)
    nets = [_Net(c, np.random.default_rng(5), capi.MVH_KV_Q4, 0) for c in (ctx, other)]
    bufs = [n.buffers(60) for n in nets]
    for b in bufs:
        _fill(b, rng)
    alone = []
    for n, b in zip(nets, bufs):
        n.step(b, 0)
        n.ctx.synchronize()
        alone.append({k: b[k].clone() for k in ("lp", "entropy", "ids", "top", "logits")})
    for _ in range(10):
        for n, b in zip(nets, bufs):
            n.step(b, 0)
    for n, b, a in zip(nets, bufs, alone):
        n.ctx.synchronize()
        for k, v in a.items():
            assert torch.equal(b[k], v), k
        n.close()
    other.close()


# ---- whole models ----

_SHAPES = [synth.ModelConfig("q4kv-128", 1024, 2816, 2, 8, 2, 512, 384, synth.Q4_0, synth.Q4_0, synth.Q4_0),
           synth.ModelConfig("q4kv-64", 1024, 2816, 2, 16, 4, 512, 1100, synth.Q8_0, synth.Q8_0, synth.Q6_K, synth.Q6_K),
           synth.ModelConfig("q4kv-48", 288, 768, 2, 6, 6, 512, 256, synth.Q4_0, synth.Q4_0, synth.Q4_0)]


@pytest.fixture(scope="module", params=_SHAPES, ids=lambda c: c.name)
def model_path(request, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("q4kv") / "m.gguf")
    synth.write_model(request.param, path, seed=5, device="cuda", digest=False)
    return path


@pytest.mark.parametrize("mode,batch", [(1, 32), (0, 8), (0, 64), (1, 5)])
def test_model_chunks_join(model_path, mode, batch):
    """Prefill in joined chunks gives the bits of chunk by chunk, and close to an F16 cache's logits."""
    n = 200
    prompt = np.random.default_rng(n).integers(0, 512, n).astype(np.int32)
    m = capi.Model(model_path, act_mode=mode, max_batch=64, kv_type=capi.MVH_KV_Q4, page_tokens=20 if batch == 5 else 128)
    assert m.kv_type() == capi.MVH_KV_Q4
    got = m.prefill(prompt, batch).copy()
    used = m.kv_bytes()
    m.reset()
    for i in range(0, n, batch):
        want = m.prefill(prompt[i:i + batch], batch)
    assert np.isfinite(got).all() and (got.view(np.uint32) == want.view(np.uint32)).all()
    m.close()
    f = capi.Model(model_path, act_mode=mode, max_batch=64, kv_type=capi.MVH_KV_F16, page_tokens=20 if batch == 5 else 128)
    near = f.prefill(prompt, batch)
    assert used * 16 == f.kv_bytes() * 5
    # a block of 32 keeps 8 % rms of its rows (0.077 for normal rows); softmax weights and two layers pass on part of it
    assert np.linalg.norm(got - near) <= 0.25 * np.linalg.norm(near)
    f.close()


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (16, 4, 64), (4, 4, 96)])
def test_model_long_chunks_join(tmp_path, heads, kv_heads, hd):
    """The same past 512 positions, where the attention is split: a token's rows are those of any other chunk."""
    cfg = synth.ModelConfig("q4kv-long", heads * hd, 2 * heads * hd, 2, heads, kv_heads, 512, 1400, synth.Q4_0, synth.Q4_0, synth.Q4_0)
    path = str(tmp_path / "m.gguf")
    synth.write_model(cfg, path, seed=6, device="cuda", digest=False)
    m = capi.Model(path, act_mode=1, max_batch=256, kv_type=capi.MVH_KV_Q4)
    for n, batch in ((530, 64), (1050, 64), (1300, 96)):
        prompt = np.random.default_rng(n).integers(0, 512, n).astype(np.int32)
        got = m.prefill(prompt, batch).copy()
        m.reset()
        for i in range(0, n, batch):
            want = m.prefill(prompt[i:i + batch], batch)
        assert np.isfinite(got).all() and (got.view(np.uint32) == want.view(np.uint32)).all(), n
        m.reset()
    m.close()


@pytest.mark.parametrize("mode", [0, 1])
def test_model_greedy(model_path, mode):
    """Greedy decoding from captured graphs gives the tokens and logits of single steps."""
    prompt = np.random.default_rng(2).integers(0, 512, 70).astype(np.int32)
    m = capi.Model(model_path, act_mode=mode, max_batch=32, kv_type=capi.MVH_KV_Q4)
    first = int(np.argmax(m.prefill(prompt, 32)))
    ids, last = m.generate_greedy(first, 40, logits=True)
    m.reset()
    tok = int(np.argmax(m.prefill(prompt, 32)))
    assert tok == first
    for i in range(40):
        logits = m.forward(tok)
        tok = int(np.argmax(logits))
        assert tok == ids[i], i
    assert (logits.view(np.uint32) == last.view(np.uint32)).all()
    m.close()
