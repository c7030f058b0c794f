"""Token ids and positions of host calls beyond 32 bits are refused before the call, not wrapped to other ones."""
import numpy as np
import pytest

from memvanta_amd import capi


def _no_device(cls, **fields):
    o = object.__new__(cls)
    for k, v in fields.items():
        setattr(o, k, v)
    return o


@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 2 ** 63])
def test_refused(far):
    ctx = _no_device(capi.Context)
    with pytest.raises(ValueError, match="targets must be 32-bit"):
        ctx.logprobs(np.zeros((2, 10), np.float32), np.array([3, far]))
    rope = _no_device(capi.Rope, ctx=ctx, head_dim=4, rot_dim=4)
    with pytest.raises(ValueError, match="positions must be 32-bit"):
        rope.apply(np.zeros((2, 4), np.float32), 1, positions=np.array([0, far]))


def test_taken():
    for a in ([2 ** 31 - 1, -2 ** 31], np.array([2 ** 31 - 1, -2 ** 31]), np.array([7], np.uint64), [], np.array([3], np.int32)):
        got = capi._host_int32(a, "")
        assert got.dtype == np.int32 and (got == np.asarray(a)).all()
