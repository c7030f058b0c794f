"""Attention behind a shared prefix over Q8 rows near fp32's ends, against 64 bits over the stored rows."""
import numpy as np
import pytest

from test_gpu_attn_shared import Q8, F, _Batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("power", [-118, -100, 100, 114, 119, 124])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (5, 1, 72)])
@pytest.mark.parametrize("prefix,own,n_tokens", [(0, 5, [1]), (300, 40, [1] * 5), (129, 20, [1] * 40), (33, 7, [65, 1, 40]), (5, 3, [150])])
def test_sizes_of_values(ctx, power, heads, kv_heads, hd, prefix, own, n_tokens):
    """Values up to 2^127: their means are finite, whatever the sums of their weights."""
    rng = np.random.default_rng(prefix + hd)
    b = _Batch(ctx, rng, Q8, prefix, [prefix + own + i for i in range(len(n_tokens))], n_tokens, heads, kv_heads, hd,
               value=lambda k, v: (k, v * F(2.0 ** power)))
    b.check()
    b.close()


@pytest.mark.parametrize("n_tokens", [[1] * 3, [40, 9]])
def test_rows_of_both_ends(ctx, n_tokens):
    """Tiny and huge rows in turn."""
    rng = np.random.default_rng(3)
    def value(k, v):
        return k, v * F(2.0) ** rng.choice([-110, 0, 123], (len(v), 1)).astype(F)
    b = _Batch(ctx, rng, Q8, 200, [210, 300, 230][: len(n_tokens)], n_tokens, 4, 2, 64, value=value)
    b.check()
    b.close()


@pytest.mark.parametrize("power", [-110, -60, 60, 100, 110])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (2, 2, 256)])
@pytest.mark.parametrize("prefix,n_tokens", [(300, [1] * 5), (33, [65, 1, 40])])
def test_sizes_of_keys(ctx, power, heads, kv_heads, hd, prefix, n_tokens):
    """Keys up to 2^113 and queries that make ordinary scores of them."""
    rng = np.random.default_rng(power + 200)
    b = _Batch(ctx, rng, Q8, prefix, [prefix + 20 + i for i in range(len(n_tokens))], n_tokens, heads, kv_heads, hd,
               value=lambda k, v: (k * F(2.0 ** power), v))
    b.check((b.q * F(2.0 ** -power)).astype(F))
    b.close()
