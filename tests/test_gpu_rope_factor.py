"""Factors that stretch angles instead of shortening them."""
import numpy as np
import pytest

from memvanta_amd import capi
from served_ops import angles, rotate

pytestmark = pytest.mark.gpu

TURNS = dict(orig_ctx=4096.0, low=1.0, high=32.0)


@pytest.mark.parametrize("scaling,more", [(1, {}), (2, TURNS), (3, TURNS)])
def test_small_factors(ctx, scaling, more):
    for factor in (1e-310, 1e-300, 9e-7):  # 1 / factor overflows, or leaves angles without a meaning
        with pytest.raises(capi.MvhError, match="factor") as e:
            ctx.rope(64, scaling=scaling, factor=factor, **more)
        assert e.value.code == 5
    ctx.rope(64, scaling=0, factor=1e-300).close()  # not read
    positions = np.array([2 ** 31 - 1, -2 ** 31, 12345, 0], np.int32)
    x = np.random.default_rng(scaling).standard_normal((4, 64), dtype=np.float32)
    for factor in (0.5, 0.25, 2.0 ** -20):
        r = ctx.rope(64, scaling=scaling, factor=factor, **more)
        f = angles(64, scaling=scaling, factor=factor, **more)
        assert np.allclose(r.angles(), f, rtol=16 * 2.0 ** -53, atol=0)
        # the angle's own last places: rotate() by the library's f, which carries their roundings
        want, err = rotate(x[:, None], positions, r.angles(), 64, False)
        assert (abs(r.apply(x, 1, positions=positions)[:, None] - want) <= err).all()
        r.close()
