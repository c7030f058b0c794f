"""What the calls of a served batch refuse before they need a device."""
import numpy as np
import pytest

from memvanta_amd import capi


def test_null_handles():
    lib = capi.load_library()
    for rc in (lambda: lib.mvh_quantize_fp8(None, None, 1, 16, 1, None, None, 0),
               lambda: lib.mvh_matmul_fp8(None, None, None, None, 1, 0),
               lambda: lib.mvh_gated_ffn_fp8(None, None, None, 0, None, None, 1, 0),
               lambda: lib.mvh_attn_shared(None, None, 0, None, None, None, 1, 0, None, 1, 1, 64, None, 0)):
        assert rc() == 1
        assert b"null" in lib.mvh_last_error()


def _context():
    return object.__new__(capi.Context)  # no device: the checks come before the call


class _Weights:
    ne0, ne1, h = 32, 20, None


@pytest.mark.parametrize("x,y", [(np.zeros((2, 48), np.float32), None), (np.zeros((2, 32), np.float32), np.zeros((2, 21), np.float32)),
                                 (np.zeros((2, 32), np.float32), np.zeros((3, 20), np.float32))])
def test_rows_that_do_not_fit(x, y):
    with pytest.raises(ValueError, match="ne0|ne1"):
        _context().matmul_fp8(_Weights(), x, y)
    with pytest.raises(ValueError, match="ne0|ne1"):
        _context().gated_ffn_fp8(_Weights(), _Weights(), x, capi.MVH_GATE_SILU, y)


def test_tensors_in_host_memory():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 32)
    with pytest.raises(ValueError, match="device"):
        _context().matmul_fp8(_Weights(), x, torch.zeros(2, 20))
    with pytest.raises(ValueError, match="mix of host and device|need a y"):
        _context().matmul_fp8(_Weights(), x)
    with pytest.raises(ValueError, match="device"):
        _context().quantize_fp8(x, 1, torch.zeros(64, dtype=torch.uint8), torch.zeros(2))
    with pytest.raises(ValueError, match="device"):
        _context().attn_shared([_Weights()], 0, torch.zeros(1, 256), [3], 4, 2, 64, out=torch.zeros(1, 256))


@pytest.mark.parametrize("more", [dict(pos=[3]), dict(pos=[3, -1]), dict(n_tokens=[1]), dict(n_tokens=[1, -1]),
                                  dict(n_tokens=[1, 2]), dict(out=np.zeros((1, 256), np.float32)),
                                  dict(out=np.zeros((2, 256), np.float64))])
def test_batches_that_do_not_fit(more):
    args = dict(kvs=[_Weights(), _Weights()], layer=0, q=np.zeros((2, 256), np.float32), pos=[3, 4], n_head=4, n_head_kv=2,
                head_dim=64)
    with pytest.raises(ValueError):
        _context().attn_shared(**{**args, **more})


@pytest.mark.parametrize("codes,scales", [(np.zeros(63, np.uint8), np.zeros(2, np.float32)),
                                          (np.zeros(64, np.int8), np.zeros(2, np.float32)),
                                          (np.zeros(64, np.uint8), np.zeros(1, np.float32)), (np.zeros(64, np.uint8), None)])
def test_quantised_rows_need_room(codes, scales):
    with pytest.raises(ValueError):
        _context().quantize_fp8(np.zeros((2, 32), np.float32), 1, codes, scales)
