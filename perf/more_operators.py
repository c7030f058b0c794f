"""The steps of a served batch that a program calls one by one, as timed cases: products with weights in 8-bit floating
point, the gated feed-forward block on such weights, and attention of sequences that share a long prefix.

  matmul   y = x W^T: weights in e4m3 with a scale per 128 x 128 block, x brought to e4m3 with a scale per row and 128 columns
  ffn      h = act(x Wg^T) * (x Wu^T) on two such weights
  shared   attention of a batch: every token sees a prefix that all sequences share, then its own sequence's rows

run() computes a case in elementary torch operations, or, where `own` is true, with the calls of memvanta_amd.capi.
Shapes are those of the model configurations in memvanta_amd/synth.py and of this repository's tests (4096 and 11008, 2048 and
5632, a vocabulary of 32000; 32 heads of 128 or 64 with 32, 8 or 4 kv heads, 6 heads of 48), and generic ones beside them.
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = {"7b": (32, 32, 128), "gqa8": (32, 8, 128), "1.1b": (32, 4, 64), "288": (6, 6, 48)}
KV = {"f16": 1, "q8": 2}
GATE = {"silu": 0, "gelu": 1}
TOP = 448.0  # the largest e4m3 value


def listed():
    return [
        # one request's token through a square projection
        {"name": "matmul_1", "kind": "matmul", "k": 4096, "n": 4096, "batch": 1},
        # the output head for a few requests
        {"name": "matmul_8_head", "kind": "matmul", "k": 4096, "n": 32000, "batch": 8},
        # one step of a batch of requests, the product after the feed-forward block
        {"name": "matmul_64", "kind": "matmul", "k": 11008, "n": 4096, "batch": 64},
        # the ragged end of a prompt
        {"name": "matmul_333", "kind": "matmul", "k": 2048, "n": 2560, "batch": 333},
        # a long prompt
        {"name": "matmul_2048", "kind": "matmul", "k": 11008, "n": 4096, "batch": 2048},
        # one request's token
        {"name": "ffn_1", "kind": "ffn", "k": 4096, "n": 11008, "batch": 1, "gate": "silu"},
        # one step of a batch of requests, a smaller model
        {"name": "ffn_45", "kind": "ffn", "k": 2048, "n": 5632, "batch": 45, "gate": "gelu"},
        # a long prompt
        {"name": "ffn_2048", "kind": "ffn", "k": 4096, "n": 11008, "batch": 2048, "gate": "silu"},
        # a few requests behind a short system prompt
        {"name": "shared_3", "kind": "shared", "kv": "f16", "shape": "1.1b", "prefix": 435, "seqs": 3, "own": 60, "tokens": 1,
         "page": 128},
        # a batch of requests behind a long prompt
        {"name": "shared_64", "kind": "shared", "kv": "f16", "shape": "gqa8", "prefix": 8000, "seqs": 64, "own": 700,
         "tokens": 1, "page": 128},
        # the same with a kv head for every head and an 8-bit cache
        {"name": "shared_32_q8", "kind": "shared", "kv": "q8", "shape": "7b", "prefix": 12000, "seqs": 32, "own": 300,
         "tokens": 1, "page": 128},
        # the questions after a shared document: a chunk of each, of lengths of their own
        {"name": "shared_12_chunks", "kind": "shared", "kv": "f16", "shape": "gqa8", "prefix": 3001, "seqs": 12, "own": 90,
         "tokens": 75, "page": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: the same calls over the whole range of shapes, batches, lengths, types and options."""
    kind = rng.choice(["matmul", "matmul", "matmul", "ffn", "ffn", "shared", "shared", "shared"])
    if kind != "shared":
        k = rng.choice([4096, 11008, 2048, 5632, 288, 16 * _log(rng, 2, 688)])
        n = rng.choice([4096, 11008, 2048, 5632, 768, _log(rng, 1, 32000)])
        most = 2048 * 4096 * 11008 // (k * n)
        case = {"kind": kind, "k": k, "n": n, "batch": rng.choice([1, _log(rng, 2, 64), _log(rng, 2, max(2, min(2048, most)))])}
        if kind == "ffn":
            case["gate"] = rng.choice(sorted(GATE))
        return case
    shape = rng.choice(sorted(HEADS))
    heads, kv_heads, hd = HEADS[shape]
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 96)])
    seqs = _log(rng, 1, 64 if tokens == 1 else 12)
    return {"kind": kind, "kv": rng.choice(sorted(KV)), "shape": shape, "prefix": _log(rng, 16, 8000 if tokens == 1 else 3001),
            "seqs": seqs, "own": _log(rng, 1, 700 if kv_heads < 32 else 300), "tokens": tokens, "page": rng.choice([16, 128, 20])}


# ---- inputs -------------------------------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + salt)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda")


def _activations(seed, salt, rows, cols):
    """N(0, 1) with one channel in 64 sixteen times as wide, as the residual stream's outlier channels are."""
    wide = torch.where(torch.rand(cols, generator=_gen(seed, salt + 50), device="cuda") < 1 / 64, 16.0, 1.0)
    return _randn(seed, salt, rows, cols) * wide


def _weights(seed, salt, n, k):
    """Codes [n][k] (e4m3 bytes) and scales [ceil(n / 128)][ceil(k / 128)] of a matrix of deviation 0.02, its rows of
    different sizes."""
    w = _randn(seed, salt, n, k) * (0.02 * torch.exp(0.5 * _randn(seed, salt + 50, n, 1)))
    nb, kb = (n + 127) // 128, (k + 127) // 128
    p = torch.nn.functional.pad(w.abs(), (0, kb * 128 - k, 0, nb * 128 - n))
    scale = p.reshape(nb, 128, kb, 128).amax(dim=(1, 3)) / TOP
    return (w / _spread(scale, n, k)).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _spread(scale, n, k):
    return scale.repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]


def _rows(seed, salt, n, dim, kv):
    """Rows of K or V as the cache type holds them: values of 16 bits, or whole numbers up to 127 times a step per row."""
    mean = _randn(seed, salt + 50, dim)
    x = _randn(seed, salt, n, dim) + mean
    if kv == "f16":
        return x.half(), None
    step = (x.abs().amax(dim=1, keepdim=True) / 127).bfloat16().float()  # few bits, so that code times step is exact
    code = torch.round(x / step).clamp(-127, 127)
    code[:, 0] = 127  # the largest: the step is what the cache computes
    return code.to(torch.int8), step


def _values(codes, step):
    return codes.float() if step is None else codes.float() * step


def _lengths(case, seed):
    """Per sequence: rows of its own before this call's tokens, and its tokens of this call."""
    g = torch.Generator()
    g.manual_seed(1000003 * int(seed) + 17)
    before = torch.randint(0, case["own"], (case["seqs"],), generator=g).tolist()
    return before, [case["tokens"] - 37 * i * i % case["tokens"] for i in range(case["seqs"])]


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
    if case["kind"] != "shared":
        k, n = case["k"], case["n"]
        s.x = _activations(seed, 1, case["batch"], k)
        s.w = [_weights(seed, 200 + 100 * i, n, k) for i in range(1 if case["kind"] == "matmul" else 2)]
        if own:
            s.bytes = [torch.cat([c.reshape(-1), sc.reshape(-1).view(torch.uint8)]) for c, sc in s.w]
            s.t = [s.ctx.wrap("w", capi.MVH_TYPE_FP8_B128, k, n, b.data_ptr(), b.numel()) for b in s.bytes]
            s.y = torch.empty((case["batch"], n), device="cuda")
    else:
        heads, kv_heads, hd = HEADS[case["shape"]]
        kv_dim, prefix = kv_heads * hd, case["prefix"]
        before, s.tokens = _lengths(case, seed)
        s.pos = [prefix + b for b in before]
        s.q = 1.5 * _randn(seed, 1, sum(s.tokens), heads * hd)
        s.k, s.v = (_rows(seed, salt, prefix, kv_dim, case["kv"]) for salt in (2, 3))
        ends = [b + t for b, t in zip(before, s.tokens)]
        own_k, own_v = (_rows(seed, salt, sum(ends), kv_dim, case["kv"]) for salt in (4, 5))
        cut = lambda rows: list(zip(*(a.split(ends) if a is not None else [None] * len(ends) for a in rows)))
        s.own_k, s.own_v = cut(own_k), cut(own_v)
        if own:
            make = lambda most: s.ctx.kv_cache(1, kv_dim, page_tokens=case["page"], max_tokens=most, kv_type=KV[case["kv"]])
            s.prefix, s.kvs = make(prefix), [make(prefix + e) for e in ends]
            values = [(_values(*s.k), _values(*s.v))] + [(_values(*k), _values(*v)) for k, v in zip(s.own_k, s.own_v)]
            torch.cuda.synchronize()
            s.prefix.write(0, 0, *values[0])
            for kv, (k, v) in zip(s.kvs, values[1:]):
                kv.write(0, prefix, k, v)
            s.ctx.synchronize()
            s.out = torch.empty_like(s.q)
    torch.cuda.synchronize()
    return s


# ---- the operators in their plain form ------------------------------------------------------------------------

def _eight_bits(x):
    """x [rows][cols] as it is in e4m3 with a scale s per 128 columns: s = the largest |x| / 448, codes x (1 / s), ties to
    even; a block whose scale is no normal number is held as zeros."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % 128)).reshape(rows, -1, 128)
    top = b.abs().amax(dim=2, keepdim=True)
    scale = top / torch.full_like(top, TOP)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    z = torch.where(scale > 0, b * (torch.ones_like(scale) / scale), torch.zeros_like(b))
    exponent = (torch.frexp(z)[1] - 1).clamp(min=-6)  # 3 bits after the leading one; steps of 2^-9 below 2^-6
    z = torch.ldexp(torch.round(torch.ldexp(z, 3 - exponent)), exponent - 3)
    return (z * scale).reshape(rows, -1)[:, :cols]


def _product(x, codes, scale):
    w = codes.view(torch.float8_e4m3fn).float() * _spread(scale, *codes.shape)
    return torch.matmul(x, w.T)


def _gated(g, u, gate):
    if gate == "silu":
        return g / (1 + torch.exp(-g)) * u
    return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5))) * u


def _heads(x, kv_heads):
    """Rows [n][kv_heads * hd] as [kv_heads][n][hd]."""
    return x.reshape(x.shape[0], kv_heads, -1).permute(1, 0, 2).contiguous()


def _attention(s, heads, kv_heads, hd):
    """softmax(q K^T / sqrt(hd)) V over the prefix and the rows of a token's own sequence up to it: the prefix's products for
    all tokens at once, then each sequence's, joined by their maxima."""
    group = heads // kv_heads
    k, v = _heads(_values(*s.k), kv_heads), _heads(_values(*s.v), kv_heads)
    q = s.q.reshape(-1, kv_heads, group, hd).permute(1, 0, 2, 3).contiguous()  # [kv_heads][token][group][hd]
    rows = lambda x: x.reshape(kv_heads, -1, x.shape[-1])
    score = torch.matmul(rows(q), k.transpose(1, 2).contiguous()) / math.sqrt(hd)
    top = score.amax(dim=2, keepdim=True)
    p = torch.exp(score - top)
    total, summed = p.sum(dim=2, keepdim=True), torch.matmul(p, v)
    out, at = torch.empty_like(rows(q)), 0
    for n, own_k, own_v in zip(s.tokens, s.own_k, s.own_v):
        k, v = _heads(_values(*own_k), kv_heads), _heads(_values(*own_v), kv_heads)
        here = slice(at * group, (at + n) * group)
        score = torch.matmul(rows(q)[:, here], k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        if n > 1:
            last = k.shape[1] - n + torch.arange(n, device="cuda").repeat_interleave(group)
            score = score.masked_fill(torch.arange(k.shape[1], device="cuda")[None, :] > last[:, None], -math.inf)
        m = torch.maximum(top[:, here], score.amax(dim=2, keepdim=True))
        p, old = torch.exp(score - m), torch.exp(top[:, here] - m)
        out[:, here] = (old * summed[:, here] + torch.matmul(p, v)) / (old * total[:, here] + p.sum(dim=2, keepdim=True))
        at += n
    return out.reshape(kv_heads, -1, group, hd).permute(1, 0, 2, 3).reshape(-1, heads * hd)


def run(s):
    case, kind = s.case, s.case["kind"]
    if kind == "matmul":
        if own:
            return s.ctx.matmul_fp8(s.t[0], s.x, s.y)
        return _product(_eight_bits(s.x), *s.w[0])
    if kind == "ffn":
        if own:
            return s.ctx.gated_ffn_fp8(s.t[0], s.t[1], s.x, GATE[case["gate"]], s.y)
        x = _eight_bits(s.x)
        return _gated(_product(x, *s.w[0]), _product(x, *s.w[1]), case["gate"])
    heads, kv_heads, hd = HEADS[case["shape"]]
    if own:
        return s.ctx.attn_shared(s.kvs, 0, s.q, s.pos, heads, kv_heads, hd, out=s.out, prefix=s.prefix,
                                 prefix_len=case["prefix"], n_tokens=s.tokens)
    return _attention(s, heads, kv_heads, hd)


# ---- what a pass cannot do without ----------------------------------------------------------------------------

def work(case):
    if case["kind"] != "shared":
        k, n, b = case["k"], case["n"], case["batch"]
        both = 2 if case["kind"] == "ffn" else 1
        return {"bytes": both * (n * k + 4 * ((n + 127) // 128) * ((k + 127) // 128)) + 4 * b * (k + n),
                "flops": 2 * both * b * n * k}
    heads, kv_heads, hd = HEADS[case["shape"]]
    tokens = _lengths(case, 0)[1]
    before = (case["own"] - 1) / 2  # on average
    row = kv_heads * hd * 2 if case["kv"] == "f16" else kv_heads * hd + 4
    seen = sum(n * (case["prefix"] + before) + n * (n + 1) / 2 for n in tokens)
    return {"bytes": round(2 * row * (case["prefix"] + sum(before + n for n in tokens)) + 8 * sum(tokens) * heads * hd),
            "flops": round(4 * hd * heads * seen)}


# ---- the same results in 64 bits ------------------------------------------------------------------------------

def _quantised(x):
    """Codes and scales of the definition, whose steps round to 32 bits (the rounding of a code is torch's own)."""
    rows, cols = x.shape
    parts = []
    for block in x.split(128, dim=1):
        largest = torch.linalg.vector_norm(block, ord=math.inf, dim=1, keepdim=True)
        scale = torch.div(largest, torch.full_like(largest, 448))
        inverse = torch.reciprocal(scale.double()).float()
        code = torch.mul(block, inverse).to(torch.float8_e4m3fn).double() * scale.double()
        parts.append(torch.where(scale.double() < 2.0 ** -126, torch.zeros_like(code), code))
    return torch.cat(parts, dim=1)


def exact(case, seed):
    if case["kind"] != "shared":
        k, n = case["k"], case["n"]
        x = _quantised(_activations(seed, 1, case["batch"], k))
        y = []
        for i in range(1 if case["kind"] == "matmul" else 2):
            codes, scale = _weights(seed, 200 + 100 * i, n, k)
            blocks = torch.arange(n, device="cuda") // 128
            total = torch.zeros((case["batch"], n), dtype=torch.float64, device="cuda")
            for b in range((k + 127) // 128):
                part = codes[:, 128 * b:128 * b + 128].contiguous().view(torch.float8_e4m3fn).double()
                total += x[:, 128 * b:128 * b + 128] @ (part * scale[blocks, b, None].double()).T.contiguous()
            y.append(total)
        if case["kind"] == "matmul":
            return y[0]
        g = y[0]
        act = g * torch.special.expit(g) if case["gate"] == "silu" else g * torch.special.ndtr(g)
        return act * y[1]
    heads, kv_heads, hd = HEADS[case["shape"]]
    kv_dim, prefix, group = kv_heads * hd, case["prefix"], heads // kv_heads
    before, tokens = _lengths(case, seed)
    held = lambda salt, n: [c.double() if st is None else c.double() * st.double() for c, st in [_rows(seed, salt, n, kv_dim, case["kv"])]][0]
    q = (1.5 * _randn(seed, 1, sum(tokens), heads * hd)).double().reshape(-1, heads, hd)
    shared_k, shared_v = (held(salt, prefix).reshape(prefix, kv_heads, hd) for salt in (2, 3))
    total = sum(before) + sum(tokens)
    own_k, own_v = (held(salt, total).reshape(total, kv_heads, hd) for salt in (4, 5))
    out, row, at = torch.empty_like(q), 0, 0
    for b, n in zip(before, tokens):
        k = torch.cat([shared_k, own_k[row:row + b + n]]).permute(1, 2, 0).contiguous()
        v = torch.cat([shared_v, own_v[row:row + b + n]]).permute(1, 0, 2).contiguous()
        x = q[at:at + n].reshape(n, kv_heads, group, hd).permute(1, 0, 2, 3).reshape(kv_heads, n * group, hd)
        score = (torch.bmm(x, k) / math.sqrt(hd)).reshape(kv_heads, n, group, -1)
        late = torch.arange(prefix + b + n, device="cuda")[None, :] > prefix + b + torch.arange(n, device="cuda")[:, None]
        weight = torch.softmax(score.masked_fill(late[:, None, :], -math.inf), dim=3).reshape(kv_heads, n * group, -1)
        out[at:at + n] = torch.bmm(weight, v).reshape(kv_heads, n, group, hd).permute(1, 0, 2, 3).reshape(n, heads, hd)
        row, at = row + b + n, at + n
    return out.reshape(-1, heads * hd)
