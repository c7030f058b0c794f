"""A model on a 4-bit cache is held to the limits of the cache's own entry point, before it needs a device."""
import pytest

from memvanta_amd import capi, synth

LIMIT = 2 ** 20


@pytest.mark.parametrize("n_ctx,ctx,page,kind", [(LIMIT + 1, 0, 128, "n_ctx"), (256, 0, LIMIT + 1, "page"), (LIMIT + 1, LIMIT, 128, None),
                                                 (256, 0, LIMIT, None)])
def test_limits(tmp_path, n_ctx, ctx, page, kind):
    cfg = synth.ModelConfig("limits", 64, 64, 1, 2, 2, 32, n_ctx, synth.Q8_0, synth.Q8_0, synth.Q8_0)
    path = str(tmp_path / "m.gguf")
    synth.write_model(cfg, path, seed=1, digest=False, blocks="random")
    # a device that is not there: what passes the check fails after it
    with pytest.raises(capi.MvhError) as e:
        capi.Model(path, device=4096, ctx=ctx, page_tokens=page, kv_type=capi.MVH_KV_Q4)
    assert ("4-bit KV cache takes up to 1048576 tokens" in str(e.value)) == (kind is not None), e.value
