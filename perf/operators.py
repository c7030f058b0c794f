"""The steps of a served token that a program calls one by one, as timed cases: rotary positions, appending K and V to
the paged cache with the rotation on the way, attention over a cache held in 4 bits, and the log probabilities of the
step's tokens.

  rope      y = x rotated by its position: half or interleaved pairs, part of the head, scaled for long contexts
  append    q rotated, k rotated and stored, v stored, in pages of each cache type; the stored rows read back as values
  attend    attention of one token or a chunk of tokens over a paged cache held in 4 bits
  logprobs  log probability of a given token, entropy of the distribution, the most probable tokens, per row of logits

run() computes a case in elementary torch operations, or, where `own` is true, with the calls of memvanta_amd.capi.
Shapes are those of the model configurations in memvanta_amd/synth.py and of this repository's tests (32 heads of 128 or
64 with 32, 8 or 4 kv heads, 6 heads of 48, a vocabulary of 32000), with longer contexts.
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = {"7b": (32, 32, 128), "gqa8": (32, 8, 128), "1.1b": (32, 4, 64), "288": (6, 6, 48)}
SCALING = {"none": 0, "linear": 1, "turns": 2, "index": 3}
LAYOUT = {"half": 0, "interleaved": 1}
KV = {"f32": 0, "f16": 1, "q8": 2, "q4": 3}


def listed():
    return [
        # decode: q and k of one token in the fused projection's output
        {"name": "rope_decode", "kind": "rope", "heads": 40, "hd": 128, "rot": 128, "layout": "half", "scaling": "none",
         "tokens": 1, "far": 2048, "scattered": False, "pad": 1024},
        # a long prompt (or the tokens of many requests, each at a position of its own), scaled for long contexts
        {"name": "rope_prompt_2048", "kind": "rope", "heads": 32, "hd": 128, "rot": 128, "layout": "interleaved",
         "scaling": "index", "tokens": 2048, "far": 131072, "scattered": True, "pad": 0},
        # decode, the cache type a model has by default
        {"name": "append_f16_1", "kind": "append", "kv": "f16", "shape": "7b", "pos": 1500, "tokens": 1, "page": 128,
         "layout": "half", "rot": 128, "scaling": "none"},
        # the ragged end of a prompt, small pages
        {"name": "append_q8_77", "kind": "append", "kv": "q8", "shape": "1.1b", "pos": 435, "tokens": 77, "page": 16,
         "layout": "half", "rot": 64, "scaling": "none"},
        # a prompt taken as one chunk into a 4-bit cache
        {"name": "append_q4_512", "kind": "append", "kv": "q4", "shape": "gqa8", "pos": 480, "tokens": 512, "page": 128,
         "layout": "half", "rot": 128, "scaling": "turns"},
        # decode early in a conversation
        {"name": "attend_1_pos100", "kind": "attend", "shape": "1.1b", "pos": 100, "tokens": 1, "page": 128},
        # decode far into a conversation, a kv head for every head
        {"name": "attend_1_pos1500", "kind": "attend", "shape": "7b", "pos": 1500, "tokens": 1, "page": 128},
        # decode in a long context
        {"name": "attend_1_pos65000", "kind": "attend", "shape": "gqa8", "pos": 65000, "tokens": 1, "page": 128},
        # a prefill chunk late in a prompt
        {"name": "attend_256_pos1700", "kind": "attend", "shape": "gqa8", "pos": 1700, "tokens": 256, "page": 128},
        # a sampled token with its alternatives
        {"name": "logprobs_1_top20", "kind": "logprobs", "rows": 1, "n": 32000, "top": 20, "target": True, "masked": 0.0},
        # one step of a batch of requests, some of them with a grammar that masks tokens
        {"name": "logprobs_77_top5", "kind": "logprobs", "rows": 77, "n": 32003, "top": 5, "target": True, "masked": 0.3},
        # scoring a prompt: the log probability of each of its tokens
        {"name": "logprobs_2048", "kind": "logprobs", "rows": 2048, "n": 32000, "top": 0, "target": True, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: the same calls over the whole range of shapes, lengths, positions, types and options."""
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "logprobs":
        n = _log(rng, 300, 130000)
        return {"kind": kind, "rows": _log(rng, 1, min(2048, 2048 * 32000 // n)), "n": n,
                "top": rng.choice([0, 1, 5, 20, 64]), "target": rng.random() < 0.8,
                "masked": rng.choice([0.0, 0.0, 0.5, 0.999])}
    shape = rng.choice(sorted(HEADS))
    heads, kv_heads, hd = HEADS[shape]
    if kind == "attend":
        tokens = rng.choice([1, 1, _log(rng, 2, 256)])
        most = 65000 * 1024 // (kv_heads * hd) if tokens == 1 else 1700
        return {"kind": kind, "shape": shape, "pos": _log(rng, 1, most), "tokens": tokens, "page": rng.choice([16, 128, 20])}
    layout, scaling = rng.choice(sorted(LAYOUT)), rng.choice(sorted(SCALING))
    rot = rng.choice([hd, hd, hd // 2])
    if kind == "rope":
        return {"kind": kind, "heads": rng.choice([heads, heads + kv_heads, 1]), "hd": hd, "rot": rot, "layout": layout,
                "scaling": scaling, "tokens": _log(rng, 1, 2048), "far": _log(rng, 2048, 131072),
                "scattered": rng.random() < 0.5, "pad": rng.choice([0, 4, kv_heads * hd])}
    return {"kind": kind, "kv": rng.choice(sorted(KV) + ["q4"]), "shape": shape, "pos": _log(rng, 1, 4000),
            "tokens": rng.choice([1, _log(rng, 2, 512)]), "page": rng.choice([16, 128, 20]), "layout": layout, "rot": rot,
            "scaling": scaling}


# ---- inputs -------------------------------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + salt)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda")


def _keys(seed, salt, n, dim):
    """N(0, 1) keys around a mean per channel, one channel in 64 four times as wide."""
    wide = torch.where(torch.rand(dim, generator=_gen(seed, salt + 100), device="cuda") < 1 / 64, 4.0, 1.0)
    return _randn(seed, salt, n, dim) * wide + _randn(seed, salt + 200, dim)


def _rope_options(case):
    """(base, factor, context of training, low and high turns, scale of the rotated vector)."""
    if case["scaling"] == "none":
        return 10000.0, 1.0, 0.0, 0.0, 0.0, 1.0
    if case["scaling"] == "linear":
        return 10000.0, 4.0, 0.0, 0.0, 0.0, 1.0
    if case["scaling"] == "turns":
        return 500000.0, 8.0, 8192.0, 1.0, 4.0, 1.0
    return 10000.0, 16.0, 4096.0, 1.0, 32.0, 0.1 * math.log(16.0) + 1.0


def _positions(case, seed):
    if case["scattered"]:
        return torch.randint(0, case["far"], (case["tokens"],), generator=_gen(seed, 5), device="cuda", dtype=torch.int32)
    first = (seed * 7919 + 13) % max(1, case["far"] - case["tokens"])
    return torch.arange(first, first + case["tokens"], device="cuda", dtype=torch.int32)


def _logits(case, seed):
    """Logits of a few likely tokens above a wide floor; a share of each row masked."""
    l = _randn(seed, 6, case["rows"], case["n"]).mul_(2.5)
    peak = torch.randint(0, case["n"], (case["rows"], 3), generator=_gen(seed, 7), device="cuda")
    l.scatter_add_(1, peak, torch.full(peak.shape, 9.0, device="cuda"))
    if case["masked"]:
        off = torch.rand(l.shape, generator=_gen(seed, 8), device="cuda") < case["masked"]
        off.scatter_(1, peak, False)
        l.masked_fill_(off, -math.inf)
    return l, peak[:, 1].to(torch.int32).contiguous()


class _State:
    pass


_context = None  # a program has one context


def prepare(case, seed):
    global _context
    s = _State()
    s.case = case
    if own:
        from memvanta_amd import capi

        if _context is None:
            _context = capi.Context(0)
        s.ctx = _context
    kind = case["kind"]
    if kind == "logprobs":
        s.logits, s.targets = _logits(case, seed)
        if not case["target"]:
            s.targets = None
        if own:
            rows, top = case["rows"], case["top"]
            s.lp = torch.empty(rows, device="cuda") if case["target"] else None
            s.entropy = torch.empty(rows, device="cuda")
            s.top_ids = torch.empty((rows, top), dtype=torch.int32, device="cuda") if top else None
            s.top_lp = torch.empty((rows, top), device="cuda") if top else None
    elif kind == "rope":
        width = case["heads"] * case["hd"]
        s.x = _randn(seed, 1, case["tokens"], width + case["pad"])[:, :width]
        s.positions = _positions(case, seed)
        s.first = int(s.positions[0])
        if own:
            s.rope = _rope_handle(s.ctx, case, case["hd"])
            s.y = torch.empty((case["tokens"], width), device="cuda")
        else:
            s.freq = _frequencies(case, case["hd"])
    else:
        heads, kv_heads, hd = HEADS[case["shape"]]
        kv_dim, n = kv_heads * hd, case["pos"] + case["tokens"]
        if kind == "append":
            qkv = _randn(seed, 1, case["tokens"], heads * hd + 2 * kv_dim)
            s.q, s.k, s.v = qkv[:, : heads * hd], qkv[:, heads * hd:-kv_dim], qkv[:, -kv_dim:]
            if own:
                s.rope = _rope_handle(s.ctx, case, hd)
                s.kv = s.ctx.kv_cache(1, kv_dim, page_tokens=case["page"], max_tokens=n, kv_type=KV[case["kv"]])
                s.q_out = torch.empty((case["tokens"], heads * hd), device="cuda")
                s.k_rows, s.v_rows = (torch.empty((case["tokens"], kv_dim), device="cuda") for _ in range(2))
            else:
                s.freq = _frequencies(case, hd)
                s.cache = _Cache(case["kv"], n, kv_dim)
        else:
            s.q = 1.5 * _randn(seed, 1, case["tokens"], heads * hd)
            k, v = _keys(seed, 2, n, kv_dim), _randn(seed, 3, n, kv_dim)
            if own:
                s.kv = s.ctx.kv_cache(1, kv_dim, page_tokens=case["page"], max_tokens=n, kv_type=KV["q4"])
                torch.cuda.synchronize()
                s.kv.write(0, 0, k, v)
                s.ctx.synchronize()
                s.out = torch.empty_like(s.q)
            else:
                s.cache = _Cache("q4", n, kv_dim)
                s.cache.write(0, k, v)
    torch.cuda.synchronize()
    return s


def _rope_handle(ctx, case, hd):
    base, factor, trained, low, high, scale = _rope_options(case)
    return ctx.rope(hd, rot_dim=case["rot"], layout=LAYOUT[case["layout"]], base=base, scaling=SCALING[case["scaling"]],
                    factor=factor, orig_ctx=trained, low=low, high=high, attn_scale=scale)


# ---- the operators in their plain form ------------------------------------------------------------------------

def _frequencies(case, hd):
    """Angle per position of each pair, in 64 bits: base^(-2i/rot), scaled."""
    base, factor, trained, low, high, _ = _rope_options(case)
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(i * (-2.0 / rot * math.log(base)))
    if case["scaling"] == "linear":
        return f / factor
    if case["scaling"] == "turns":  # kept above `high` turns over the training context, divided below `low`, blended
        g = ((trained / (2 * math.pi) * f - low) / (high - low)).clamp(0, 1)
    elif case["scaling"] == "index":  # the same ends, blended along the pair index
        at = [rot * math.log(trained / (2 * math.pi * t)) / (2 * math.log(base)) for t in (high, low)]
        a, b = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        g = 1 - ((i - a) / max(b - a, 0.001)).clamp(0, 1)
    else:
        return f
    return f * g + f / factor * (1 - g)


def _rotated(x, heads, case, freq, positions):
    """x [tokens][heads * hd] rotated: angles, cos and sin in 64 bits, rounded once to 32; products and sums in 32."""
    scale = _rope_options(case)[5]
    rot = case["rot"]
    angle = positions.double()[:, None] * freq[None, :]
    c, s = (scale * torch.cos(angle)).float()[:, None, :], (scale * torch.sin(angle)).float()[:, None, :]
    x = x.reshape(x.shape[0], heads, -1)
    y = x.clone()
    if case["layout"] == "half":
        x0, x1 = x[..., : rot // 2], x[..., rot // 2: rot]
        y[..., : rot // 2], y[..., rot // 2: rot] = x0 * c - x1 * s, x0 * s + x1 * c
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = x0 * c - x1 * s, x0 * s + x1 * c
    return y.reshape(y.shape[0], -1)


class _Cache:
    """K and V rows as the cache types hold them: codes, with a scale per row, or a step and a middle per block of 32."""

    def __init__(self, kind, n, kv_dim):
        self.kind = kind
        code = {"f32": torch.float32, "f16": torch.int16, "q8": torch.int8, "q4": torch.uint8}[kind]
        self.codes = [torch.zeros((n, kv_dim), dtype=code, device="cuda") for _ in range(2)]
        per = {"q8": [1], "q4": [2, kv_dim // 32]}.get(kind)
        half = torch.float16 if kind == "q4" else torch.float32
        self.scales = [torch.zeros([n] + per, dtype=half, device="cuda") for _ in range(2)] if per else None

    def write(self, pos, k, v):
        for which, x in ((0, k), (1, v)):
            n = x.shape[0]
            if self.kind == "f32":
                self.codes[which][pos:pos + n] = x
            elif self.kind == "f16":
                self.codes[which][pos:pos + n] = _half_bits(x)
            elif self.kind == "q8":  # one scale per row: max |x| / 127, ties away from zero
                top = x.abs().amax(dim=1, keepdim=True)
                one = torch.ones_like(top)
                sc = torch.where(top > 0, top / (127 * one), one)
                z = x / sc
                self.codes[which][pos:pos + n] = (torch.sign(z) * torch.floor(z.abs().double() + 0.5)).clamp(-127, 127).to(torch.int8)
                self.scales[which][pos:pos + n] = sc
            else:
                b = x.reshape(n, -1, 32)
                lo, hi = b.amin(dim=2), b.amax(dim=2)
                sc = ((hi - lo) / torch.full_like(lo, 15.0)).clamp(max=512.0).half()
                mid = (lo + 8 * sc.float()).clamp(-65504.0, 65504.0).half()
                z = (b - mid.float()[..., None]) / sc.float()[..., None]
                code = torch.where(sc[..., None] > 0, (torch.round(z) + 8).clamp(0, 15), torch.full_like(z, 8))
                self.codes[which][pos:pos + n] = code.reshape(n, -1).to(torch.uint8)
                self.scales[which][pos:pos + n, 0], self.scales[which][pos:pos + n, 1] = sc, mid

    def values(self, which, pos, n):
        c = self.codes[which][pos:pos + n]
        if self.kind == "f32":
            return c.clone()
        if self.kind == "f16":
            return c.view(torch.float16).float()
        sc = self.scales[which][pos:pos + n]
        if self.kind == "q8":
            return c.float() * sc
        return ((c.float() - 8).reshape(n, -1, 32) * sc[:, 0].float()[..., None] + sc[:, 1].float()[..., None]).reshape(n, -1)


def _half_bits(x):
    """fp16 bits as this library's cache holds them: ties away from zero, a carry out of the mantissa OR-ed into the exponent."""
    i = x.contiguous().view(torch.int32)
    sign = torch.where(i < 0, 0x8000, 0)
    e, mant = ((i >> 23) & 255) - 112, i & 0x7FFFFF
    normal = (e.clamp(min=1) << 10) | ((mant + 0x1000) >> 13)
    small = (((mant | 0x800000) >> (1 - e).clamp(0, 31)) + 0x1000) >> 13
    return (torch.where(e <= 0, torch.where(e < -10, torch.zeros_like(small), small), normal) | sign).to(torch.int16)


def _attention(cache, q, pos, heads, kv_heads, hd):
    tokens = q.shape[0]
    n, group = pos + tokens, heads // kv_heads
    k, v = (cache.values(which, 0, n).reshape(n, kv_heads, hd).permute(1, 0, 2).contiguous() for which in (0, 1))
    rows = q.reshape(tokens, kv_heads, group, hd).permute(1, 2, 0, 3).reshape(kv_heads, group * tokens, hd)
    score = torch.matmul(rows, k.transpose(1, 2)) / math.sqrt(hd)
    if tokens > 1:
        seen = pos + torch.arange(tokens, device="cuda").repeat(group)
        score = score.masked_fill(torch.arange(n, device="cuda")[None, :] > seen[:, None], -math.inf)
    p = torch.exp(score - score.amax(dim=2, keepdim=True))
    out = torch.matmul(p, v) / p.sum(dim=2, keepdim=True)
    return out.reshape(kv_heads, group, tokens, hd).permute(2, 0, 1, 3).reshape(tokens, heads * hd)


def _log_probabilities(logits, targets, top):
    m = logits.amax(dim=1, keepdim=True)
    d = logits - m
    p = torch.exp(d)
    total = p.sum(dim=1)
    log_total = torch.log(total)
    out = {"entropy": log_total - torch.where(p > 0, p * d, torch.zeros_like(p)).sum(dim=1) / total}
    if targets is not None:
        out["logprob"] = d.gather(1, targets.long()[:, None])[:, 0] - log_total
    if top:
        best, at = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: the lowest index first
        out["top_ids"] = at[:, :top].to(torch.int32)
        out["top_logprobs"] = best[:, :top] - m - log_total[:, None]
    return out


def run(s):
    case, kind = s.case, s.case["kind"]
    if kind == "logprobs":
        if own:
            s.ctx.logprobs(s.logits, s.targets, case["top"], logprob=s.lp, entropy=s.entropy, top_ids=s.top_ids,
                           top_logprobs=s.top_lp)
            out = {"entropy": s.entropy}
            if case["target"]:
                out["logprob"] = s.lp
            if case["top"]:
                out["top_ids"], out["top_logprobs"] = s.top_ids, s.top_lp
            return out
        return _log_probabilities(s.logits, s.targets, case["top"])
    if kind == "rope":
        if own:
            if case["scattered"]:
                return s.rope.apply(s.x, case["heads"], positions=s.positions, out=s.y)
            return s.rope.apply(s.x, case["heads"], pos=s.first, out=s.y)
        return _rotated(s.x, case["heads"], case, s.freq, s.positions)
    heads, kv_heads, hd = HEADS[case["shape"]]
    pos, tokens = case["pos"], case["tokens"]
    if kind == "append":
        if own:
            s.kv.append(0, pos, s.k, s.v, rope=s.rope, q=s.q, q_out=s.q_out)
            s.kv.read(0, pos, tokens, s.k_rows, s.v_rows)
            return {"q": s.q_out, "k": s.k_rows, "v": s.v_rows}
        positions = torch.arange(pos, pos + tokens, device="cuda")
        s.cache.write(pos, _rotated(s.k, kv_heads, case, s.freq, positions), s.v)
        return {"q": _rotated(s.q, heads, case, s.freq, positions), "k": s.cache.values(0, pos, tokens),
                "v": s.cache.values(1, pos, tokens)}
    if own:
        if tokens == 1:
            return s.kv.attn_decode(0, s.q, pos, heads, kv_heads, hd, s.out)
        return s.kv.attn_batch(0, s.q, pos, tokens, heads, kv_heads, hd, s.out)
    return _attention(s.cache, s.q, pos, heads, kv_heads, hd)


# ---- what a pass cannot do without ----------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        rows, n, top = case["rows"], case["n"], case["top"]
        return {"bytes": 4 * rows * n + rows * (4 + 8 * bool(case["target"]) + 8 * top), "flops": 5 * rows * n}
    if kind == "rope":
        x = case["tokens"] * case["heads"]
        return {"bytes": 8 * x * case["hd"], "flops": 3 * x * case["rot"]}
    heads, kv_heads, hd = HEADS[case["shape"]]
    kv_dim, pos, tokens = kv_heads * hd, case["pos"], case["tokens"]
    if kind == "append":  # q in and out, k and v in, the stored rows, the rows read back
        row = {"f32": 4 * kv_dim, "f16": 2 * kv_dim, "q8": kv_dim + 4, "q4": kv_dim * 5 // 8}[case["kv"]]
        return {"bytes": tokens * (8 * heads * hd + 16 * kv_dim + 2 * row), "flops": 3 * tokens * case["rot"] * (heads + kv_heads)}
    pairs = tokens * pos + tokens * (tokens + 1) // 2
    return {"bytes": (pos + tokens) * kv_dim * 5 // 4 + 8 * tokens * heads * hd, "flops": 4 * hd * heads * pairs}


# ---- the same results in 64 bits ------------------------------------------------------------------------------

def _turn(x, heads, case, positions):
    """x rotated, as complex numbers: (x0 + i x1) * scale * e^(i position f)."""
    base, factor, trained, low, high, scale = _rope_options(case)
    rot, f = case["rot"], []
    ends = [rot / 2 * math.log(trained / t / (2 * math.pi), base) for t in (high, low)] if case["scaling"] == "index" else None
    for i in range(rot // 2):
        keep = {"none": 1.0, "linear": 0.0}.get(case["scaling"])
        plain = base ** (-2 * i / rot)
        if case["scaling"] == "turns":
            keep = min(max((plain * trained / math.tau - low) / (high - low), 0.0), 1.0)
        elif case["scaling"] == "index":
            first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rot - 1)
            keep = 1.0 - min(max((i - first) / max(last - first, 0.001), 0.0), 1.0)
        f.append(plain * (keep + (1.0 - keep) / factor))
    turn = torch.polar(torch.tensor(scale, dtype=torch.float64, device="cuda"),
                       positions.double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))
    x = x.double().reshape(x.shape[0], heads, -1)
    part, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "half":
        y = torch.complex(*part.chunk(2, dim=2)) * turn
        y = torch.cat([y.real, y.imag], dim=2)
    else:
        y = torch.view_as_real(torch.view_as_complex(part.reshape(*part.shape[:2], -1, 2).contiguous()) * turn).flatten(2)
    return torch.cat([y, rest], dim=2).flatten(1)


def _stored(x, kind):
    """The values that rows x of 32 bits have once stored: the steps of the formats' definitions, which round to 32 bits."""
    if kind == "f32":
        return x.double()
    if kind == "f16":
        return _half_bits(x).view(torch.float16).double()
    if kind == "q8":
        top = x.abs().max(dim=1, keepdim=True).values
        step = torch.where(top == 0, torch.ones_like(top), torch.div(top, torch.full_like(top, 127)))
        z = torch.div(x, step).double()
        return torch.copysign((z.abs() + 0.5).floor().clamp(max=127), z) * step.double()
    blocks = x.reshape(-1, 32)
    small, large = torch.aminmax(blocks, dim=1, keepdim=True)
    step = torch.minimum(torch.div(large - small, torch.full_like(small, 15)), torch.full_like(small, 512)).to(torch.float16)
    middle = (small + step.float() * 8).clamp(-65504, 65504).to(torch.float16).float()
    level = torch.where(step > 0, torch.div(blocks - middle, step.float()), torch.zeros_like(blocks)).round().clamp(-8, 7)
    return (level.double() * step.double() + middle.double()).reshape(x.shape)


def exact(case, seed):
    kind = case["kind"]
    if kind == "logprobs":
        l, targets = _logits(case, seed)
        l = l.double()
        lse = torch.logsumexp(l, dim=1)
        lp = l - lse[:, None]
        out = {"entropy": torch.special.entr(torch.exp(lp)).sum(dim=1)}
        if case["target"]:
            out["logprob"] = lp[torch.arange(case["rows"], device="cuda"), targets.long()]
        if case["top"]:
            out["top_ids"] = None
            out["top_logprobs"] = torch.topk(lp, case["top"], dim=1).values
        return out
    if kind == "rope":
        width = case["heads"] * case["hd"]
        x = _randn(seed, 1, case["tokens"], width + case["pad"])[:, :width]
        return _turn(x, case["heads"], case, _positions(case, seed))
    heads, kv_heads, hd = HEADS[case["shape"]]
    kv_dim, pos, tokens = kv_heads * hd, case["pos"], case["tokens"]
    if kind == "append":
        q, k, v = _randn(seed, 1, tokens, heads * hd + 2 * kv_dim).split([heads * hd, kv_dim, kv_dim], dim=1)
        at = torch.arange(pos, pos + tokens, device="cuda")
        k = _turn(k, kv_heads, case, at)
        # a rotated key next to a border between two codes may go either way: no value of its own in 8 or 4 bits
        k = k if case["kv"] == "f32" else _stored(k.float(), "f16") if case["kv"] == "f16" else None
        return {"q": _turn(q, heads, case, at), "k": k, "v": _stored(v.contiguous(), case["kv"])}
    n, group = pos + tokens, heads // kv_heads
    q = (1.5 * _randn(seed, 1, tokens, heads * hd)).double().reshape(tokens, heads, hd)
    k, v = (_stored(x, "q4").reshape(n, kv_heads, hd) for x in (_keys(seed, 2, n, kv_dim), _randn(seed, 3, n, kv_dim)))
    late = torch.arange(n, device="cuda")[None, :] > (pos + torch.arange(tokens, device="cuda"))[:, None]
    out = torch.empty_like(q)
    for h in range(heads):
        score = q[:, h] @ k[:, h // group].T.contiguous() / math.sqrt(hd)
        out[:, h] = torch.softmax(score.masked_fill(late, -math.inf), dim=1) @ v[:, h // group].contiguous()
    return out.flatten(1)
