"""A batch served behind a shared prefix, as a program calls it: 8-bit floating point projections, rotated appends to each
sequence's cache, attention behind the prefix, the gated feed-forward block, log probabilities; captured into a graph and
replayed; side by side on two contexts."""
import threading

import numpy as np
import pytest

from batch_ops import attend_shared, gated, product
from memvanta_amd import capi
from served_ops import log_softmax

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HEADS, KV_HEADS, HD, DIM, FFN, VOCAB, LAYERS, PREFIX = 8, 2, 64, 256, 656, 700, 2, 150
KV_DIM, Q_DIM = KV_HEADS * HD, HEADS * HD


class _Net:
    """Two layers and an output head on the calls of one context; a prefix cache and one per sequence."""

    def __init__(self, ctx, rng, kv_type, seqs):
        self.ctx = ctx
        shapes = {"qkv": (Q_DIM + 2 * KV_DIM, DIM), "o": (DIM, Q_DIM), "gate": (FFN, DIM), "up": (FFN, DIM), "down": (DIM, FFN)}
        self.w, self.t = {}, {}
        for name, (rows, cols) in [("head", (VOCAB, DIM))] + [((n, l), s) for n, s in shapes.items() for l in range(LAYERS)]:
            w = (rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32)
            self.w[name] = ctx.quantize_fp8(w, 128)
            self.t[name] = ctx.upload_fp8(str(name), w)
        self.rope = ctx.rope(HD)
        self.prefix = ctx.kv_cache(LAYERS, KV_DIM, 128, PREFIX, kv_type)
        self.kvs = [ctx.kv_cache(LAYERS, KV_DIM, 16, 256, kv_type) for _ in range(seqs)]
        b = self.buffers(PREFIX)
        fill(b, rng)
        self.step(b, [self.prefix], [0], [PREFIX], 0)
        ctx.synchronize()
        self.check(b, [self.prefix], [0], [PREFIX], 0)

    def buffers(self, n):
        e = lambda width: torch.zeros((n, width), device="cuda")
        return {"x": e(DIM), "logits": e(VOCAB), "lp": torch.zeros(n, device="cuda"), "entropy": torch.zeros(n, device="cuda"),
                "targets": torch.zeros(n, dtype=torch.int32, device="cuda"),
                **{(name, l): e(w) for l in range(LAYERS)
                   for name, w in (("qkv", Q_DIM + 2 * KV_DIM), ("q", Q_DIM), ("att", Q_DIM), ("o", DIM), ("ffn", FFN), ("y", DIM))}}

    def step(self, b, kvs, pos, n_tokens, prefix_len=PREFIX):
        ctx, t, x = self.ctx, self.t, b["x"]
        for l in range(LAYERS):
            qkv, q = b["qkv", l], b["q", l]
            ctx.matmul_fp8(t["qkv", l], x, qkv)
            at = 0
            for kv, p, n in zip(kvs, pos, n_tokens):
                r = slice(at, at + n)
                kv.append(l, p, qkv[r, Q_DIM:-KV_DIM], qkv[r, -KV_DIM:], self.rope, q=qkv[r, :Q_DIM], q_out=q[r])
                at += n
            ctx.attn_shared(kvs, l, q, pos, HEADS, KV_HEADS, HD, out=b["att", l], prefix=self.prefix if prefix_len else None,
                            prefix_len=prefix_len, n_tokens=n_tokens)
            ctx.matmul_fp8(t["o", l], b["att", l], b["o", l])
            ctx.gated_ffn_fp8(t["gate", l], t["up", l], b["o", l], capi.MVH_GATE_SILU, b["ffn", l])
            ctx.matmul_fp8(t["down", l], b["ffn", l], b["y", l])
            x = b["y", l]
        ctx.matmul_fp8(t["head"], x, b["logits"])
        ctx.logprobs(b["logits"], b["targets"], 0, b["lp"], b["entropy"])

    def check(self, b, kvs, pos, n_tokens, prefix_len=PREFIX):
        """Each operator's output against 64 bits from its own input."""
        h = {k: v.cpu().numpy() for k, v in b.items()}
        x = h["x"]

        def close(got, want, bound):
            assert (abs(got - want) <= bound + 1e-30).all()

        for l in range(LAYERS):
            close(h["qkv", l], *product(x, *self.w["qkv", l]))
            held = self.prefix.read(l, 0, prefix_len) if prefix_len else (np.zeros((0, KV_DIM)),) * 2
            own = [kv.read(l, prefix_len, p + n - prefix_len) for kv, p, n in zip(kvs, pos, n_tokens)]
            at = 0
            for (k, _), p, n in zip(own, pos, n_tokens):  # the rows appended, as the cache holds them
                turned = self.rope.apply(np.ascontiguousarray(h["qkv", l][at:at + n, Q_DIM:-KV_DIM]), KV_HEADS, pos=p)
                half = self.ctx.fp16_to_fp32(self.ctx.fp32_to_fp16(turned)).reshape(turned.shape)
                step = 0 if kvs[0].kv_type == capi.MVH_KV_F16 else 1 / 100  # half a step of a row's widest channel
                assert (abs(k[p - prefix_len:] - (turned if step else half)) <= step * abs(turned).max(1, keepdims=True)).all()
                q = self.rope.apply(np.ascontiguousarray(h["qkv", l][at:at + n, :Q_DIM]), HEADS, pos=p)
                assert (h["q", l][at:at + n] == q).all()
                at += n
            want, size = attend_shared(h["q", l], held, own, pos, n_tokens, HEADS, KV_HEADS)
            # scores up to 16, of four times that in magnitudes, in 22 bits each; so are the weights
            close(h["att", l], want, (2 * 4 * 16 + 4) * 2.0 ** -22 * size)
            close(h["o", l], *product(h["att", l], *self.w["o", l]))
            close(h["ffn", l], *gated(h["o", l], self.w["gate", l], self.w["up", l], 0))
            close(h["y", l], *product(h["ffn", l], *self.w["down", l]))
            x = h["y", l]
        close(h["logits"], *product(x, *self.w["head"]))
        lp = log_softmax(h["logits"])[np.arange(len(x)), h["targets"]]
        assert abs(h["lp"] - lp).max() <= 5e-6

    def close(self):
        for x in (*self.kvs, self.prefix, self.rope):
            x.close()
        for t in self.t.values():
            t.free()


def fill(b, rng):
    b["x"].copy_(torch.from_numpy(rng.standard_normal(tuple(b["x"].shape)).astype(np.float32)))
    b["targets"].copy_(torch.from_numpy(rng.integers(0, VOCAB, len(b["targets"])).astype(np.int32)))
    torch.cuda.synchronize()


def _serve(net, rng, plan):
    pos = [PREFIX] * len(net.kvs)
    for n_tokens in plan:
        b = net.buffers(sum(n_tokens))
        fill(b, rng)
        live = [i for i, n in enumerate(n_tokens) if n]
        args = [net.kvs[i] for i in live], [pos[i] for i in live], [n_tokens[i] for i in live]
        net.step(b, *args)
        net.ctx.synchronize()
        net.check(b, *args)
        pos = [p + n for p, n in zip(pos, n_tokens)]
    return pos


@pytest.mark.parametrize("kv_type", [capi.MVH_KV_F16, capi.MVH_KV_Q8])
def test_prompts_then_tokens(ctx, kv_type):
    """Ragged prompts behind the prefix, then tokens one by one, some sequences pausing."""
    rng = np.random.default_rng(kv_type)
    net = _Net(ctx, rng, kv_type, 5)
    _serve(net, rng, [[40, 3, 17, 1, 90], [1] * 5, [1] * 5, [0, 1, 1, 0, 2], [1] * 5])
    net.close()


def test_captured_step(ctx):
    """A batch's token captured into a graph and replayed with other inputs, eager work between the replays."""
    rng = np.random.default_rng(3)
    c = capi.Context(0)
    net = _Net(c, rng, capi.MVH_KV_F16, 20)
    pos = _serve(net, rng, [[int(n) for n in rng.integers(1, 12, 20)]])
    b, ones = net.buffers(20), [1] * 20
    fill(b, rng)
    net.step(b, net.kvs, pos, ones)  # once before the capture: pages and workspaces are there
    c.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(c.stream)):
        net.step(b, net.kvs, pos, ones)
    big = net.buffers(400)
    for _ in range(4):
        fill(b, rng)
        with torch.cuda.stream(torch.cuda.ExternalStream(c.stream)):
            g.replay()
        c.synchronize()
        net.check(b, net.kvs, pos, ones)
        got = {k: v.clone() for k, v in b.items()}
        torch.cuda.synchronize()
        net.step(b, net.kvs, pos, ones)
        c.synchronize()
        assert all(torch.equal(got[k], b[k]) for k in b)
        c.matmul_fp8(net.t["head"], big["x"], big["logits"])  # a larger workspace
        c.synchronize()
    net.close()
    c.close()


def test_two_contexts(ctx):
    """Two threads serve their own batches at the same time."""
    plan, fails = [[9, 2, 30], [1] * 3, [1] * 3, [2, 1, 40]], []

    def run(seed):
        try:
            rng = np.random.default_rng(seed)
            c = capi.Context(0)
            net = _Net(c, rng, (capi.MVH_KV_F16, capi.MVH_KV_Q8)[seed % 2], 3)
            _serve(net, rng, plan)
            net.close()
            c.close()
        except BaseException as e:  # reported by the test's own thread
            fails.append(e)

    threads = [threading.Thread(target=run, args=(s,)) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails, fails
