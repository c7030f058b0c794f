"""Attention behind a shared prefix with as many heads as a call takes: its workgroups go in several launches."""
import numpy as np
import pytest

from memvanta_amd import capi

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_many_heads_and_a_chunk(ctx):
    """2^24 query rows: 127 sequences of one token and a chunk of 129, 65536 heads of 8, a kv head each."""
    heads, hd, n = 65536, 8, [1] * 100 + [129] + [1] * 27
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda m: torch.randn((m, heads * hd), generator=g, device="cuda")
    kvs = [ctx.kv_cache(1, heads * hd, 1, m) for m in n]
    q = rows(sum(n))
    held = []
    for kv, m in zip(kvs, n):
        k, v = rows(m), rows(m)
        torch.cuda.synchronize()
        kv.write(0, 0, k, v)
        ctx.synchronize()
        held.append([torch.from_numpy(x).cuda() for x in kv.read(0, 0, m)])
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    ctx.attn_shared(kvs, 0, q, [0] * len(n), heads, heads, hd, out=out, n_tokens=n)
    ctx.synchronize()
    for i, (k, v) in enumerate(held):
        if n[i] == 1:  # one row: its values, the 22 bits of a weight and four roundings apart
            at = i if i < 100 else i + 128
            assert (out[at] - v[0]).abs().le(2.0 ** -21 * v[0].abs()).all(), i
    k, v = (x.float().reshape(129, heads, hd).transpose(0, 1) for x in held[100])
    late = torch.ones(129, 129, device="cuda").triu(1).bool()
    for h in range(0, heads, 8192):
        part = slice(h, h + 8192)
        x = q[100:229].reshape(129, heads, hd).transpose(0, 1)[part].double()
        s = (x.contiguous() @ k[part].double().transpose(1, 2).contiguous() / np.sqrt(hd)).masked_fill(late, -np.inf)
        w = torch.softmax(s, 2)
        want, size = w @ v[part].double().contiguous(), w @ v[part].double().abs().contiguous()
        got = out[100:229].reshape(129, heads, hd).transpose(0, 1)[part]
        # scores up to 16 of four times that in magnitudes, q and weights of 22 bits
        assert ((got - want).abs() <= (2 * 4 * 16 + 4) * 2.0 ** -22 * size).all(), h
    for kv in kvs:
        kv.close()
