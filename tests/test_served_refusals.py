"""What the rotary, cache, attention and log probability calls refuse before they need a device."""
import ctypes

import pytest

from memvanta_amd import capi


def _refused(rc, text):
    assert rc == 1
    assert text in capi.load_library().mvh_last_error()


def test_null_handles():
    lib = capi.load_library()
    out, n = ctypes.c_void_p(), ctypes.c_size_t()
    _refused(lib.mvh_rope_create(None, None, ctypes.byref(out)), b"null")
    _refused(lib.mvh_rope_angles(None, None), b"null")
    assert lib.mvh_rope_destroy(None) == 0
    _refused(lib.mvh_rope_apply(None, None, None, 0, 1, 1, None, 0, None, 0, 0), b"null")
    _refused(lib.mvh_kv_append(None, None, 0, 0, 1, None, None, 0, 0, None, 0, None, 0, None, 0, 0), b"null")
    _refused(lib.mvh_kv_read(None, None, 0, 0, 1, None, None, 0), b"null")
    _refused(lib.mvh_kv_write(None, None, 0, 0, 1, None, None, 0), b"null")
    _refused(lib.mvh_attn_decode(None, None, 0, None, 0, 1, 1, 64, None, 0), b"null")
    _refused(lib.mvh_attn_batch(None, None, 0, None, 0, 1, 1, 1, 64, None, 0), b"null")
    _refused(lib.mvh_logprobs(None, None, 1, 1, None, 0, None, None, None, None, 0), b"null")
    _refused(lib.mvh_kv_bytes_allocated(None, ctypes.byref(n)), b"null")


def test_q4_type_name():
    assert capi.kv_parse_type("q4") == capi.MVH_KV_Q4 == 3
    assert capi.kv_type_name(capi.MVH_KV_Q4) == "q4"
    with pytest.raises(capi.MvhError, match="unknown KV cache type: q4_0"):
        capi.kv_parse_type("q4_0")


def test_rows_in_host_tensors():
    """A tensor in host memory is not taken for device rows."""
    torch = pytest.importorskip("torch")
    for rows in (torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.float16), torch.zeros(64, 2).t()):
        with pytest.raises(ValueError, match="device"):
            capi._rows(rows)
    ctx = object.__new__(capi.Context)  # no device: the check comes before the call
    with pytest.raises(ValueError, match="device memory"):
        ctx.logprobs(torch.zeros(2, 64))
