"""ctypes binding of the C ABI in include/memvanta_hip.h (libmemvanta_hip.so).

There is no fallback: if the HIP library is missing or a call fails, an
exception is raised.  Host arrays are numpy; device buffers are anything with
an integer device address (torch tensors' ``data_ptr()``).
"""
from __future__ import annotations

import ctypes as C
import os
import re
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmemvanta_hip.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "memvanta_hip.h")

MVH_HOST, MVH_DEVICE = 0, 1
MVH_ACT_REF, MVH_ACT_Q8 = 0, 1
MVH_KV_F32, MVH_KV_F16, MVH_KV_Q8 = 0, 1, 2  # KVCacheType order
MVH_KV_Q4 = 3  # 4-bit codes, a step and a middle per block of 32
MVH_ROPE_HALF, MVH_ROPE_INTERLEAVED = 0, 1
MVH_ROPE_SCALE_NONE, MVH_ROPE_SCALE_LINEAR, MVH_ROPE_SCALE_TURNS, MVH_ROPE_SCALE_INDEX = 0, 1, 2, 3
MVH_TYPE_NATIVE_Q4_0, MVH_TYPE_NATIVE_Q8_0 = 0x1002, 0x1008  # BlockQ4_0 (20 B) / BlockQ8_0 (36 B) of quant.hpp
MVH_TYPE_FP8_B128 = 0x1010  # e4m3 codes, a float scale per 128 x 128
MVH_GATE_SILU, MVH_GATE_GELU = 0, 1
KV_DTYPE = {MVH_KV_F32: np.float32, MVH_KV_F16: np.uint16, MVH_KV_Q8: np.int8,
            MVH_KV_Q4: np.float32}
STATUS = {0: "MVH_OK", 1: "MVH_E_INVALID", 2: "MVH_E_SHAPE", 3: "MVH_E_TYPE", 4: "MVH_E_DEVICE",
          5: "MVH_E_RANGE", 6: "MVH_E_NOMEM"}


class MvhError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{STATUS.get(code, code)}: {msg}")
        self.code = code
        self.msg = msg


def header_functions(path: str = HEADER) -> list[str]:
    """Names of every function the C header declares."""
    text = open(path).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(mvh_[a-z0-9_]+)\s*\(", text)))


_vp, _sz, _u32, _u64, _int = C.c_void_p, C.c_size_t, C.c_uint32, C.c_uint64, C.c_int
_SIGS = {
    "mvh_last_error": (C.c_char_p, []),
    "mvh_version": (_int, []),
    "mvh_device_count": (_int, [C.POINTER(_int)]),
    "mvh_context_create": (_int, [_int, C.POINTER(_vp)]),
    "mvh_context_destroy": (_int, [_vp]),
    "mvh_context_stream": (_int, [_vp, C.POINTER(_vp)]),
    "mvh_context_synchronize": (_int, [_vp]),
    "mvh_tensor_upload": (_int, [_vp, C.c_char_p, _u32, _u64, _u64, _vp, _u64, C.POINTER(_vp)]),
    "mvh_tensor_wrap": (_int, [_vp, C.c_char_p, _u32, _u64, _u64, _vp, _u64, C.POINTER(_vp)]),
    "mvh_tensor_free": (_int, [_vp]),
    "mvh_tensor_info": (_int, [_vp, C.POINTER(_u32), C.POINTER(_u64), C.POINTER(_u64), C.POINTER(_u64),
                               C.POINTER(_vp)]),
    "mvh_quantize_q8": (_int, [_vp, _vp, _sz, _sz, _vp, _vp, _int]),
    "mvh_matvec": (_int, [_vp, _vp, _vp, _vp, _int]),
    "mvh_matvec_q8": (_int, [_vp, _vp, _vp, _vp, _vp, _int]),
    "mvh_matmul_batch": (_int, [_vp, _vp, _vp, _vp, _sz, _int]),
    "mvh_matmul_batch_v06": (_int, [_vp, _vp, _vp, _vp, _sz, _int, _int]),
    "mvh_matmul_batch_v06_noalloc": (_int, [_vp, _vp, _vp, _vp, _sz, _int]),
    "mvh_read_row_f32": (_int, [_vp, _vp, _sz, _vp, _sz, _int]),
    "mvh_argmax": (_int, [_vp, _vp, _sz, _sz, _vp, _int]),
    "mvh_stream_read": (_int, [_vp, _vp, _sz, _vp, _sz]),
    "mvh_fp32_to_fp16": (_int, [_vp, _vp, _vp, _sz, _int]),
    "mvh_fp16_to_fp32": (_int, [_vp, _vp, _vp, _sz, _int]),
    "mvh_kv_parse_type": (_int, [C.c_char_p, C.POINTER(_int)]),
    "mvh_kv_type_name": (C.c_char_p, [_int]),
    "mvh_kv_create": (_int, [_vp, _sz, _sz, _sz, _sz, _int, C.POINTER(_vp)]),
    "mvh_kv_type": (_int, [_vp, C.POINTER(_int)]),
    "mvh_kv_destroy": (_int, [_vp]),
    "mvh_kv_reset": (_int, [_vp]),
    "mvh_kv_bytes_allocated": (_int, [_vp, C.POINTER(_sz)]),
    "mvh_kv_write": (_int, [_vp, _vp, _sz, _sz, _sz, _vp, _vp, _int]),
    "mvh_kv_read_row": (_int, [_vp, _vp, _sz, _sz, _int, _vp, C.POINTER(C.c_float)]),
    "mvh_attn_decode": (_int, [_vp, _vp, _sz, _vp, _sz, _sz, _sz, _sz, _vp, _int]),
    "mvh_attn_batch": (_int, [_vp, _vp, _sz, _vp, _sz, _sz, _sz, _sz, _sz, _vp, _int]),
    "mvh_kv_read": (_int, [_vp, _vp, _sz, _sz, _sz, _vp, _vp, _int]),
    "mvh_rope_create": (_int, [_vp, _vp, C.POINTER(_vp)]),
    "mvh_rope_destroy": (_int, [_vp]),
    "mvh_rope_angles": (_int, [_vp, _vp]),
    "mvh_rope_apply": (_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _sz, _int]),
    "mvh_kv_append": (_int, [_vp, _vp, _sz, _sz, _sz, _vp, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _int]),
    "mvh_logprobs": (_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp, _int]),
    "mvh_quantize_fp8": (_int, [_vp, _vp, _sz, _sz, _sz, _vp, _vp, _int]),
    "mvh_matmul_fp8": (_int, [_vp, _vp, _vp, _vp, _sz, _int]),
    "mvh_gated_ffn_fp8": (_int, [_vp, _vp, _vp, _int, _vp, _vp, _sz, _int]),
    "mvh_attn_shared": (_int, [_vp, _vp, _sz, _vp, _vp, _vp, _sz, _sz, _vp, _sz, _sz, _sz, _vp, _int]),
    "mvh_model_open": (_int, [C.c_char_p, _int, _sz, _sz, _int, _int, _sz, C.POINTER(_vp)]),
    "mvh_model_kv_type": (_int, [_vp, C.POINTER(_int)]),
    "mvh_model_close": (_int, [_vp]),
    "mvh_model_config": (_int, [_vp, C.POINTER(_sz)]),
    "mvh_model_reset": (_int, [_vp]),
    "mvh_model_forward": (_int, [_vp, _int, _vp]),
    "mvh_model_prefill": (_int, [_vp, _vp, _sz, _sz, _vp]),
    "mvh_model_generate_greedy": (_int, [_vp, _int, _sz, _vp, _vp]),
    "mvh_model_position": (_int, [_vp, C.POINTER(_sz)]),
    "mvh_model_kv_bytes": (_int, [_vp, C.POINTER(_sz)]),
    "mvh_model_stream": (_int, [_vp, C.POINTER(_vp)]),
    "mvh_quantize_q8_0": (_int, [_vp, _vp, _sz, _vp, _int]),
    "mvh_quantize_q4_0": (_int, [_vp, _vp, _sz, _vp, _int]),
    "mvh_matvec_q4_q8": (_int, [_vp, _vp, _vp, _vp, _int]),
    "mvh_matmul_q4_0_batch": (_int, [_vp, _vp, _vp, _vp, _sz, _int]),
    "mvh_matvec_q4_0": (_int, [_vp, _vp, _vp, _vp, _int]),
    "mvh_matvec_q8_0": (_int, [_vp, _vp, _vp, _vp, _int]),
    "mvh_profile_enable": (None, [_int]),
    "mvh_profile_reset": (None, []),
    "mvh_profile_snapshot": (_int, [_vp, _sz, C.POINTER(_sz)]),
    "mvh_profile_kind_name": (C.c_char_p, [_int]),
}


class ProfileEntry(C.Structure):
    """mvh_profile_entry (KernelProfileEntry of include/memvanta/gguf_kernels.hpp:12-19)."""

    _fields_ = [("layer", C.c_int), ("kind", C.c_int), ("tensor", C.c_char * 192), ("calls", C.c_size_t),
                ("batch", C.c_size_t), ("ms", C.c_double)]


class RopeConfig(C.Structure):
    """mvh_rope_config."""

    _fields_ = [("head_dim", _sz), ("rot_dim", _sz), ("layout", _int), ("scaling", _int), ("base", C.c_double),
                ("factor", C.c_double), ("orig_ctx", C.c_double), ("low", C.c_double), ("high", C.c_double),
                ("attn_scale", C.c_double)]


_lib = None


def _finalize(release, _finalizing=sys.is_finalizing) -> None:
    """Release a handle from __del__, except while the interpreter is finalizing.

    At interpreter exit the HIP runtime (torch's and this library's) may already
    be tearing down its device state; a hipFree / hipStreamDestroy issued then
    from a garbage-collected handle can touch freed runtime structures.  The
    process is ending and the driver reclaims every allocation, so the handle
    is left alone.  Explicit close()/free() calls are unaffected.  The
    finalizing test and this function are bound as default arguments: module
    globals may already be cleared when a late __del__ runs."""
    if _finalizing():
        return
    try:
        release()
    except Exception:
        pass


def load_library(path: str = LIB_PATH) -> C.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(f"HIP backend not built: {path} is missing (run __graft_entry__.build())")
    # One HIP runtime per process: PyTorch ships its own libamdhip64.  Loaded
    # first, it also serves this library (same soname); loaded after this
    # library had brought in the system runtime, torch finds no device.  So
    # when torch is installed it is imported before the library is opened.
    if "torch" not in sys.modules:
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
    lib = C.CDLL(path)
    for name, (res, args) in _SIGS.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _lib = lib
    return lib


def _ptr(a) -> int | None:
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        if not a.flags["C_CONTIGUOUS"]:
            raise ValueError("host array must be C-contiguous")
        return a.ctypes.data
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return int(a)


def _kind(*arrs) -> int:
    dev = [not isinstance(a, np.ndarray) for a in arrs if a is not None]
    if all(dev):
        return MVH_DEVICE
    if not any(dev):
        return MVH_HOST
    raise ValueError("mix of host and device buffers in one call")


_f32 = None


def _torch_f32():
    global _f32
    if _f32 is None:
        _f32 = sys.modules["torch"].float32
    return _f32


def _host_rows(a):
    """A host array as [rows][elements] of float32."""
    a = np.ascontiguousarray(a, np.float32)
    return a[None] if a.ndim == 1 else a


def _host_int32(a, name: str):
    """Host integers as int32; what does not fit is refused, not wrapped."""
    a = np.asarray(a)
    if a.size and not ((a >= -2 ** 31) & (a < 2 ** 31)).all():
        raise ValueError(f"{name} must be 32-bit integers")
    return np.ascontiguousarray(a, np.int32)


def _rows(a):
    """(address, rows, elements of a row, elements from one row to the next) of float32 rows: a host array from
    _host_rows, or a device tensor, which may be a view with a row stride."""
    if isinstance(a, np.ndarray):
        if a.dtype != np.float32 or a.ndim != 2 or not a.flags["C_CONTIGUOUS"]:
            raise ValueError("host rows must be 2-D, C-contiguous and float32")
        n, width = a.shape
        return a.ctypes.data, n, width, width
    if a.dtype is not _torch_f32() or not a.is_cuda:
        raise ValueError("device rows must be float32 in device memory")
    shape = a.shape
    if len(shape) == 1:
        n, width = 1, shape[0]
    elif len(shape) == 2:
        n, width = shape
    else:
        raise ValueError("rows must be 2-D")
    if a.is_contiguous():
        return a.data_ptr(), n, width, width
    stride = a.stride()
    if stride[-1] != 1 and width > 1:
        raise ValueError("a row's elements must be consecutive")
    return a.data_ptr(), n, width, stride[0] if n > 1 else width


def _flat(a, dtype: str, count: int, host: bool, name: str) -> int:
    """Address of a contiguous array of at least count elements, on the side that the call is on."""
    if isinstance(a, np.ndarray):
        good = host and a.dtype == dtype and a.size >= count and a.flags["C_CONTIGUOUS"]
    else:
        good = (not host and a is not None and str(a.dtype) == "torch." + dtype and a.numel() >= count
                and a.is_contiguous() and a.is_cuda)
    if not good:
        raise ValueError(f"{name} must be {count} contiguous elements of {dtype} in {'host' if host else 'device'} memory")
    return _ptr(a)


class Context:
    """One device + one HIP stream (mvh_context)."""

    def __init__(self, device: int = 0):
        self.lib = load_library()
        h = _vp()
        self._check(self.lib.mvh_context_create(device, C.byref(h)))
        self.h = h.value
        self.device = device

    def _check(self, rc: int):
        if rc != 0:
            raise MvhError(rc, self.lib.mvh_last_error().decode())

    def close(self):
        if getattr(self, "h", None):
            self.lib.mvh_context_destroy(self.h)
            self.h = None

    def __del__(self, _fin=_finalize):
        _fin(self.close)

    @property
    def stream(self) -> int:
        s = _vp()
        self._check(self.lib.mvh_context_stream(self.h, C.byref(s)))
        return s.value

    def synchronize(self):
        self._check(self.lib.mvh_context_synchronize(self.h))

    # -- weights --
    def upload(self, name: str, ggml_type: int, ne0: int, ne1: int, data: np.ndarray) -> "Tensor":
        data = np.ascontiguousarray(data, dtype=np.uint8)
        t = _vp()
        self._check(self.lib.mvh_tensor_upload(self.h, name.encode(), ggml_type, ne0, ne1, data.ctypes.data,
                                               data.nbytes, C.byref(t)))
        return Tensor(self, t.value, name, ggml_type, ne0, ne1)

    def wrap(self, name: str, ggml_type: int, ne0: int, ne1: int, dev_ptr: int, nbytes: int) -> "Tensor":
        t = _vp()
        self._check(self.lib.mvh_tensor_wrap(self.h, name.encode(), ggml_type, ne0, ne1, dev_ptr, nbytes,
                                             C.byref(t)))
        return Tensor(self, t.value, name, ggml_type, ne0, ne1)

    # -- kernels (host numpy in/out, or device pointers) --
    def quantize_q8(self, x, q=None, d=None):
        if isinstance(x, np.ndarray):
            x = np.ascontiguousarray(x, np.float32)
            m = 1 if x.ndim == 1 else x.shape[0]
            k = x.shape[-1]
            q = np.empty(x.shape, np.int8)
            d = np.empty(x.shape[:-1] + (k // 32,), np.float32)
            self._check(self.lib.mvh_quantize_q8(self.h, x.ctypes.data, m, k, q.ctypes.data, d.ctypes.data, MVH_HOST))
            return q, d
        m = 1 if x.dim() == 1 else x.shape[0]
        k = x.shape[-1]
        self._check(self.lib.mvh_quantize_q8(self.h, _ptr(x), m, k, _ptr(q), _ptr(d), MVH_DEVICE))
        return q, d

    def matvec(self, w: "Tensor", x, y=None):
        if y is None:
            y = np.empty(w.ne1, np.float32)
            x = np.ascontiguousarray(x, np.float32)
        self._check(self.lib.mvh_matvec(self.h, w.h, _ptr(x), _ptr(y), _kind(x, y)))
        return y

    def matvec_q8(self, w: "Tensor", q, d, y=None):
        if y is None:
            q = np.ascontiguousarray(q, np.int8)
            d = np.ascontiguousarray(d, np.float32)
            y = np.empty(w.ne1, np.float32)
        self._check(self.lib.mvh_matvec_q8(self.h, w.h, _ptr(q), _ptr(d), _ptr(y), _kind(q, d, y)))
        return y

    def matmul_batch(self, w: "Tensor", x, y=None):
        b = x.shape[0]
        if y is None:
            x = np.ascontiguousarray(x, np.float32)
            y = np.empty((b, w.ne1), np.float32)
        self._check(self.lib.mvh_matmul_batch(self.h, w.h, _ptr(x), _ptr(y), b, _kind(x, y)))
        return y

    def matmul_batch_v06(self, w: "Tensor", x, act_mode: int = MVH_ACT_REF, y=None):
        b = x.shape[0]
        if y is None:
            x = np.ascontiguousarray(x, np.float32)
            y = np.empty((b, w.ne1), np.float32)
        self._check(self.lib.mvh_matmul_batch_v06(self.h, w.h, _ptr(x), _ptr(y), b, act_mode, _kind(x, y)))
        return y

    def matmul_batch_v06_noalloc(self, w: "Tensor", x, y, act_mode: int = MVH_ACT_REF):
        """mvh_matmul_batch_v06_noalloc: device x [batch][ne0] -> device y [batch][ne1], no device allocation."""
        self._check(self.lib.mvh_matmul_batch_v06_noalloc(self.h, w.h, _ptr(x), _ptr(y), x.shape[0], act_mode))
        return y

    def read_row(self, w: "Tensor", row: int, out=None, cols: int | None = None):
        """tensor_read_row_f32: row `row` of w as fp32 (cols defaults to ne0)."""
        cols = w.ne0 if cols is None else cols
        if out is None:
            out = np.empty(cols, np.float32)
        self._check(self.lib.mvh_read_row_f32(self.h, w.h, row, _ptr(out), cols, _kind(out)))
        return out

    def stream_read(self, buf, nbytes: int, sink, sink_words: int):
        """Enqueue the streaming-read probe over nbytes of device buffer buf (device sink of sink_words words)."""
        self._check(self.lib.mvh_stream_read(self.h, _ptr(buf), nbytes, _ptr(sink), sink_words))

    def argmax(self, logits, out=None):
        """Greedy sampling per row (first index of the max) of [rows][n] logits."""
        if out is None:
            logits = np.ascontiguousarray(logits, np.float32)
            rows = 1 if logits.ndim == 1 else logits.shape[0]
            out = np.empty(rows, np.int32)
        else:
            rows = 1 if logits.dim() == 1 else logits.shape[0]
        n = logits.shape[-1]
        self._check(self.lib.mvh_argmax(self.h, _ptr(logits), n, rows, _ptr(out), _kind(logits, out)))
        return out

    def logprobs(self, logits, targets=None, top_k: int = 0, logprob=None, entropy=None, top_ids=None,
                 top_logprobs=None):
        """mvh_logprobs of [rows][n] logits.  Host arrays: {"logprob" (with targets), "entropy", "top_ids",
        "top_logprobs" (with top_k)} are returned; device buffers: the given outputs are written."""
        if isinstance(logits, np.ndarray):
            logits = np.ascontiguousarray(logits, np.float32)
            logits = logits[None] if logits.ndim == 1 else logits
            rows, n = logits.shape
            out = {"entropy": np.empty(rows, np.float32)}
            if targets is not None:
                targets = _host_int32(targets, "targets").reshape(rows)
                out["logprob"] = np.empty(rows, np.float32)
            if top_k:
                out["top_ids"] = np.empty((rows, top_k), np.int32)
                out["top_logprobs"] = np.empty((rows, top_k), np.float32)
            self._check(self.lib.mvh_logprobs(self.h, _ptr(logits), n, rows, _ptr(targets), top_k,
                                              _ptr(out.get("logprob")), _ptr(out["entropy"]), _ptr(out.get("top_ids")),
                                              _ptr(out.get("top_logprobs")), MVH_HOST))
            return out
        torch = sys.modules["torch"]
        shape = logits.shape
        rows, n = (1, shape[0]) if len(shape) == 1 else shape
        if logits.dtype is not torch.float32 or not logits.is_contiguous() or not logits.is_cuda:
            raise ValueError("logits must be contiguous float32 rows in device memory")

        def at(a, dtype, count, name):
            if a is None:
                return None
            if isinstance(a, np.ndarray):
                raise ValueError("mix of host and device buffers in one call")
            if a.dtype is not dtype or a.numel() < count or not a.is_contiguous() or not a.is_cuda:
                raise ValueError(f"{name} must be {count} contiguous elements of {dtype} in device memory")
            return a.data_ptr()

        f32, i32 = torch.float32, torch.int32
        self._check(self.lib.mvh_logprobs(self.h, logits.data_ptr(), n, rows, at(targets, i32, rows, "targets"), top_k,
                                          at(logprob, f32, rows, "logprob"), at(entropy, f32, rows, "entropy"),
                                          at(top_ids, i32, rows * top_k, "top_ids"),
                                          at(top_logprobs, f32, rows * top_k, "top_logprobs"), MVH_DEVICE))
        return None

    def rope(self, head_dim: int, rot_dim: int = 0, layout: int = MVH_ROPE_HALF, base: float = 10000.0,
             scaling: int = MVH_ROPE_SCALE_NONE, factor: float = 1.0, orig_ctx: float = 0.0, low: float = 0.0,
             high: float = 0.0, attn_scale: float = 1.0) -> "Rope":
        return Rope(self, RopeConfig(head_dim, rot_dim, layout, scaling, base, factor, orig_ctx, low, high, attn_scale))

    def fp32_to_fp16(self, x, out=None):
        if out is None:
            x = np.ascontiguousarray(x, np.float32).ravel()
            out = np.empty(x.size, np.uint16)
        n = x.size if isinstance(x, np.ndarray) else x.numel()
        self._check(self.lib.mvh_fp32_to_fp16(self.h, _ptr(x), _ptr(out), n, _kind(x, out)))
        return out

    def fp16_to_fp32(self, h, out=None):
        if out is None:
            h = np.ascontiguousarray(h, np.uint16).ravel()
            out = np.empty(h.size, np.float32)
        n = h.size if isinstance(h, np.ndarray) else h.numel()
        self._check(self.lib.mvh_fp16_to_fp32(self.h, _ptr(h), _ptr(out), n, _kind(h, out)))
        return out

    # -- native block formats (src/quant.cpp, src/quant_kernels.cpp) --
    def quantize_native(self, x, bsize: int, out=None):
        """quantize_q8_0 (bsize 36) / quantize_q4_0 (bsize 20) of the flattened x -> uint8 [n/32, bsize]."""
        fn = self.lib.mvh_quantize_q8_0 if bsize == 36 else self.lib.mvh_quantize_q4_0
        if out is None:
            x = np.ascontiguousarray(x, np.float32).ravel()
            out = np.empty((x.size // 32, bsize), np.uint8)
        n = x.size if isinstance(x, np.ndarray) else x.numel()
        self._check(fn(self.h, _ptr(x), n, _ptr(out), _kind(x, out)))
        return out

    def matvec_q4_q8(self, a: "Tensor", xq, y=None):
        if y is None:
            xq = np.ascontiguousarray(xq, np.uint8)
            y = np.empty(a.ne1, np.float32)
        self._check(self.lib.mvh_matvec_q4_q8(self.h, a.h, _ptr(xq), _ptr(y), _kind(xq, y)))
        return y

    def matmul_q4_0_batch(self, a: "Tensor", x, y=None):
        b = 1 if x.ndim == 1 else x.shape[0]
        if y is None:
            x = np.ascontiguousarray(x, np.float32)
            y = np.empty((b, a.ne1), np.float32)
        self._check(self.lib.mvh_matmul_q4_0_batch(self.h, a.h, _ptr(x), _ptr(y), b, _kind(x, y)))
        return y

    def matvec_native(self, a: "Tensor", x, y=None):
        """matvec_q4_0 / matvec_q8_0 by the tensor's native type."""
        fn = self.lib.mvh_matvec_q8_0 if a.type == MVH_TYPE_NATIVE_Q8_0 else self.lib.mvh_matvec_q4_0
        if y is None:
            x = np.ascontiguousarray(x, np.float32)
            y = np.empty(a.ne1, np.float32)
        self._check(fn(self.h, a.h, _ptr(x), _ptr(y), _kind(x, y)))
        return y

    # -- 8-bit floating point weights --
    def quantize_fp8(self, x, block_rows: int = 1, codes=None, scales=None):
        """mvh_quantize_fp8 of rows x: (codes uint8 [rows][cols], scales float32 [ceil(rows/block_rows)][ceil(cols/128)]);
        device rows need both outputs."""
        host = isinstance(x, np.ndarray)
        if host:
            x = _host_rows(x)
        at, n, cols, pitch = _rows(x)
        if pitch != cols:
            raise ValueError("x must be contiguous rows")
        shape = ((n + block_rows - 1) // max(1, block_rows), (cols + 127) // 128)
        if host and codes is None and scales is None:
            codes, scales = np.empty((n, cols), np.uint8), np.empty(shape, np.float32)
        c_at = _flat(codes, "uint8", n * cols, host, "codes")
        s_at = _flat(scales, "float32", shape[0] * shape[1], host, "scales")
        self._check(self.lib.mvh_quantize_fp8(self.h, at, n, cols, block_rows, c_at, s_at, MVH_HOST if host else MVH_DEVICE))
        return codes, scales

    def upload_fp8(self, name: str, w: np.ndarray) -> "Tensor":
        """A host matrix [rows][cols] as a MVH_TYPE_FP8_B128 tensor."""
        codes, scales = self.quantize_fp8(w, 128)
        return self.upload(name, MVH_TYPE_FP8_B128, codes.shape[1], codes.shape[0],
                           np.concatenate([codes.ravel(), scales.ravel().view(np.uint8)]))

    def _fp8_rows(self, w: "Tensor", x, y):
        """(x, y, addresses, rows) of a product with w."""
        host = isinstance(x, np.ndarray)
        if host:
            x = _host_rows(x)
            y = np.empty((x.shape[0], w.ne1), np.float32) if y is None else y
        elif y is None:
            raise ValueError("device rows need a y")
        if isinstance(y, np.ndarray) != host:
            raise ValueError("mix of host and device buffers in one call")
        x_at, n, width, pitch = _rows(x)
        y_at, y_n, y_width, y_pitch = _rows(y)
        if width != w.ne0 or y_width != w.ne1 or y_n != n or pitch != width or y_pitch != y_width:
            raise ValueError("x must be contiguous rows of ne0 elements and y as many of ne1")
        return y, x_at, y_at, n, MVH_HOST if host else MVH_DEVICE

    def matmul_fp8(self, w: "Tensor", x, y=None):
        """mvh_matmul_fp8: rows x [batch][ne0] times the FP8 tensor w."""
        y, x_at, y_at, n, kind = self._fp8_rows(w, x, y)
        self._check(self.lib.mvh_matmul_fp8(self.h, w.h, x_at, y_at, n, kind))
        return y

    def gated_ffn_fp8(self, gate: "Tensor", up: "Tensor", x, act: int = MVH_GATE_SILU, y=None):
        """mvh_gated_ffn_fp8: act(x gate^T) * (x up^T)."""
        y, x_at, y_at, n, kind = self._fp8_rows(gate, x, y)
        self._check(self.lib.mvh_gated_ffn_fp8(self.h, gate.h, up.h, act, x_at, y_at, n, kind))
        return y

    def attn_shared(self, kvs, layer: int, q, pos, n_head: int, n_head_kv: int, head_dim: int, out=None, prefix=None,
                    prefix_len: int = 0, n_tokens=None):
        """mvh_attn_shared: the tokens of sequence i (n_tokens[i] of them, one by default, at positions pos[i]..) see
        rows 0 .. prefix_len-1 of the cache prefix and their own cache kvs[i]'s from there on.  q and out: rows of
        n_head*head_dim, the sequences' tokens in turn."""
        n_seq = len(kvs)
        count = n_seq if n_tokens is None else int(sum(n_tokens))
        if len(pos) != n_seq or (n_tokens is not None and len(n_tokens) != n_seq):
            raise ValueError("pos and n_tokens must have one entry per sequence")
        if any(p < 0 for p in pos) or (n_tokens is not None and any(n < 0 for n in n_tokens)):
            raise ValueError("pos and n_tokens must not be negative")
        host = isinstance(q, np.ndarray)
        if host:
            q = _host_rows(q)
            out = np.empty_like(q) if out is None else out
        q_at = _flat(q, "float32", count * n_head * head_dim, host, "q")
        o_at = _flat(out, "float32", count * n_head * head_dim, host, "out")
        handles = (_vp * n_seq)(*[kv.h for kv in kvs])
        at = (_sz * n_seq)(*pos)
        counts = None if n_tokens is None else (_sz * n_seq)(*n_tokens)
        self._check(self.lib.mvh_attn_shared(self.h, None if prefix is None else prefix.h, prefix_len, handles, at, counts,
                                             n_seq, layer, q_at, n_head, n_head_kv, head_dim, o_at,
                                             MVH_HOST if host else MVH_DEVICE))
        return out

    def kv_cache(self, n_layer: int, kv_dim: int, page_tokens: int = 128, max_tokens: int = 2048,
                 kv_type: int = MVH_KV_F16) -> "KVCache":
        return KVCache(self, n_layer, kv_dim, page_tokens, max_tokens, kv_type)


class Tensor:
    def __init__(self, ctx: Context, h: int, name: str, ggml_type: int, ne0: int, ne1: int):
        self.ctx, self.h, self.name, self.type, self.ne0, self.ne1 = ctx, h, name, ggml_type, ne0, ne1

    def free(self):
        if self.h:
            self.ctx.lib.mvh_tensor_free(self.h)
            self.h = None

    def __del__(self, _fin=_finalize):
        _fin(self.free)

    def info(self):
        ty, n0, n1, nb, dp = _u32(), _u64(), _u64(), _u64(), _vp()
        self.ctx._check(self.ctx.lib.mvh_tensor_info(self.h, C.byref(ty), C.byref(n0), C.byref(n1), C.byref(nb),
                                                     C.byref(dp)))
        return ty.value, n0.value, n1.value, nb.value, dp.value


class Rope:
    """Rotary positions (mvh_rope)."""

    def __init__(self, ctx: Context, config: RopeConfig):
        self.ctx, self.head_dim, self.rot_dim = ctx, config.head_dim, config.rot_dim or config.head_dim
        h = _vp()
        ctx._check(ctx.lib.mvh_rope_create(ctx.h, C.byref(config), C.byref(h)))
        self.h = h.value

    def close(self):
        if getattr(self, "h", None):
            self.ctx.lib.mvh_rope_destroy(self.h)
            self.h = None

    def __del__(self, _fin=_finalize):
        _fin(self.close)

    def angles(self) -> np.ndarray:
        """Angle per position of each pair, scaled (float64)."""
        out = np.empty(self.rot_dim // 2, np.float64)
        self.ctx._check(self.ctx.lib.mvh_rope_angles(self.h, out.ctypes.data))
        return out

    def apply(self, x, n_head: int, pos: int = 0, out=None, positions=None):
        """Rows of n_head heads rotated: row t by position positions[t] (int32), or pos + t.  Device rows may be a
        view with a row stride; out may be x itself."""
        host = isinstance(x, np.ndarray)
        if host:
            x = _host_rows(x)
            out = np.empty((x.shape[0], n_head * self.head_dim), np.float32) if out is None else out
            if positions is not None:
                positions = _host_int32(positions, "positions")
        elif out is None:
            raise ValueError("device rows need an out")
        if isinstance(out, np.ndarray) != host:
            raise ValueError("mix of host and device buffers in one call")
        x_at, n, width, pitch = _rows(x)
        y_at, out_n, out_width, out_pitch = _rows(out)
        if min(width, out_width) < n_head * self.head_dim or out_n < n:
            raise ValueError("rows shorter than n_head heads, or fewer out than x")
        at = None
        if positions is not None:
            if isinstance(positions, np.ndarray) != host:
                raise ValueError("mix of host and device buffers in one call")
            if len(positions) != n or str(positions.dtype) not in ("int32", "torch.int32"):
                raise ValueError("positions must be one int32 per row")
            if not host and not (positions.is_contiguous() and positions.is_cuda):
                raise ValueError("positions must be contiguous and in device memory")
            at = _ptr(positions)
        ctx = self.ctx
        ctx._check(ctx.lib.mvh_rope_apply(ctx.h, self.h, x_at, pitch, n, n_head, at, pos, y_at, out_pitch,
                                          MVH_HOST if host else MVH_DEVICE))
        return out


PROFILE_KINDS = ("q_proj", "k_proj", "v_proj", "o_proj", "ffn_gate", "ffn_up", "ffn_down", "output", "other")


def profile_enable(on: bool = True) -> None:
    """enable_kernel_profiling: time every tensor call and model GEMV/GEMM on the device."""
    load_library().mvh_profile_enable(1 if on else 0)


def profile_reset() -> None:
    """reset_kernel_profile."""
    load_library().mvh_profile_reset()


def profile_snapshot() -> list[dict]:
    """kernel_profile_snapshot: one dict per (layer, kind, tensor, batch) entry, in first-call order."""
    lib = load_library()
    n = _sz()
    if lib.mvh_profile_snapshot(None, 0, C.byref(n)) != 0:
        raise MvhError(1, lib.mvh_last_error().decode())
    arr = (ProfileEntry * max(1, n.value))()
    if lib.mvh_profile_snapshot(C.cast(arr, _vp), n.value, C.byref(n)) != 0:
        raise MvhError(1, lib.mvh_last_error().decode())
    return [{"layer": e.layer, "kind": e.kind, "kind_name": profile_kind_name(e.kind), "tensor": e.tensor.decode(),
             "calls": e.calls, "batch": e.batch, "ms": e.ms} for e in arr[: n.value]]


def profile_kind_name(kind: int) -> str:
    """kernel_profile_kind_name."""
    return load_library().mvh_profile_kind_name(kind).decode()


def kv_parse_type(s: str) -> int:
    """parse_kv_cache_type: "f32" / "f16" / "q8" / "q8_0" -> MVH_KV_*."""
    lib = load_library()
    t = _int()
    if lib.mvh_kv_parse_type(s.encode(), C.byref(t)) != 0:
        raise MvhError(1, lib.mvh_last_error().decode())
    return t.value


def kv_type_name(t: int) -> str:
    return load_library().mvh_kv_type_name(t).decode()


class KVCache:
    def __init__(self, ctx: Context, n_layer, kv_dim, page_tokens, max_tokens, kv_type: int = MVH_KV_F16):
        self.ctx, self.kv_dim, self.kv_type = ctx, kv_dim, kv_type
        h = _vp()
        ctx._check(ctx.lib.mvh_kv_create(ctx.h, n_layer, kv_dim, page_tokens, max_tokens, kv_type, C.byref(h)))
        self.h = h.value

    def close(self):
        if getattr(self, "h", None):
            self.ctx.lib.mvh_kv_destroy(self.h)
            self.h = None

    def __del__(self, _fin=_finalize):
        _fin(self.close)

    def reset(self):
        self.ctx._check(self.ctx.lib.mvh_kv_reset(self.h))

    def bytes_allocated(self) -> int:
        n = _sz()
        self.ctx._check(self.ctx.lib.mvh_kv_bytes_allocated(self.h, C.byref(n)))
        return n.value

    def write(self, layer, pos, k, v):
        if isinstance(k, np.ndarray):
            k = np.ascontiguousarray(k, np.float32)
            v = np.ascontiguousarray(v, np.float32)
            n = k.size // self.kv_dim
        else:
            n = k.numel() // self.kv_dim
        self.ctx._check(self.ctx.lib.mvh_kv_write(self.ctx.h, self.h, layer, pos, n, _ptr(k), _ptr(v), _kind(k, v)))

    def read_row(self, layer, pos, which):
        """(stored row: float32 / fp16 bits / int8 by cache type, Q8 row scale or 1.0)"""
        out = np.empty(self.kv_dim, KV_DTYPE[self.kv_type])
        sc = C.c_float()
        self.ctx._check(self.ctx.lib.mvh_kv_read_row(self.ctx.h, self.h, layer, pos, which, out.ctypes.data,
                                                     C.byref(sc)))
        return out, np.float32(sc.value)

    def append(self, layer, pos, k, v, rope: Rope, q=None, q_out=None):
        """k rotated and v stored at positions pos.., and q (when given) rotated to q_out (which may be q).  Device
        rows may be views of one fused buffer."""
        host = isinstance(k, np.ndarray)
        if host:
            k, v = _host_rows(k), _host_rows(v)
        k_at, n, k_width, k_pitch = _rows(k)
        v_at, v_n, v_width, v_pitch = _rows(v)
        if v_n != n or k_width != self.kv_dim or v_width != self.kv_dim:
            raise ValueError("k and v must be rows of kv_dim elements")
        q_at, y_at, n_head, q_pitch, out_pitch = None, None, 0, 0, 0
        if q is not None:
            if host:
                q = _host_rows(q)
                q_out = np.empty_like(q) if q_out is None else q_out
            elif q_out is None:
                raise ValueError("device rows need a q_out")
            q_at, q_n, q_width, q_pitch = _rows(q)
            y_at, y_n, y_width, out_pitch = _rows(q_out)
            if q_n != n or y_n != n or q_width % rope.head_dim or y_width != q_width:
                raise ValueError("q and q_out must be one row of whole heads per row of k")
            n_head = q_width // rope.head_dim
        if isinstance(v, np.ndarray) != host or (q is not None and (isinstance(q, np.ndarray) != host
                                                                    or isinstance(q_out, np.ndarray) != host)):
            raise ValueError("mix of host and device buffers in one call")
        ctx = self.ctx
        ctx._check(ctx.lib.mvh_kv_append(ctx.h, self.h, layer, pos, n, rope.h, q_at, q_pitch, n_head, y_at, out_pitch, k_at,
                                         k_pitch, v_at, v_pitch, MVH_HOST if host else MVH_DEVICE))
        return q_out

    def read(self, layer, pos, n, k=None, v=None):
        """Rows pos .. pos+n-1 of K and V as float32 [n][kv_dim]: into device buffers, or returned as host arrays."""
        if k is None and v is None:
            k, v = (np.empty((n, self.kv_dim), np.float32) for _ in range(2))
        k_at = v_at = None
        if k is not None:
            k_at, rows, width, pitch = _rows(k)
            if rows < n or width != self.kv_dim or pitch != width:
                raise ValueError("k must be n contiguous rows of kv_dim elements")
        if v is not None:
            v_at, rows, width, pitch = _rows(v)
            if rows < n or width != self.kv_dim or pitch != width:
                raise ValueError("v must be n contiguous rows of kv_dim elements")
        host = isinstance(k if k is not None else v, np.ndarray)
        if k is not None and v is not None and isinstance(v, np.ndarray) != host:
            raise ValueError("mix of host and device buffers in one call")
        ctx = self.ctx
        ctx._check(ctx.lib.mvh_kv_read(ctx.h, self.h, layer, pos, n, k_at, v_at, MVH_HOST if host else MVH_DEVICE))
        return k, v

    def type(self) -> int:
        t = _int()
        self.ctx._check(self.ctx.lib.mvh_kv_type(self.h, C.byref(t)))
        return t.value

    def attn_batch(self, layer, q, pos, n_tokens, n_head, n_head_kv, head_dim, out=None):
        """causal attention of n_tokens query tokens at positions pos.. (q: [n_tokens][n_head*head_dim])"""
        if out is None:
            q = np.ascontiguousarray(q, np.float32)
            out = np.empty((n_tokens, n_head * head_dim), np.float32)
        self.ctx._check(self.ctx.lib.mvh_attn_batch(self.ctx.h, self.h, layer, _ptr(q), pos, n_tokens, n_head,
                                                    n_head_kv, head_dim, _ptr(out), _kind(q, out)))
        return out

    def attn_decode(self, layer, q, pos, n_head, n_head_kv, head_dim, out=None):
        if out is None:
            q = np.ascontiguousarray(q, np.float32)
            out = np.empty(n_head * head_dim, np.float32)
        self.ctx._check(self.ctx.lib.mvh_attn_decode(self.ctx.h, self.h, layer, _ptr(q), pos, n_head, n_head_kv,
                                                     head_dim, _ptr(out), _kind(q, out)))
        return out


class Model:
    """LlamaModel on one device (mvh_model_*)."""

    def __init__(self, path: str, device: int = 0, ctx: int = 0, page_tokens: int = 128,
                 act_mode: int = MVH_ACT_Q8, max_batch: int = 64, kv_type: int = MVH_KV_F16):
        self.lib = load_library()
        h = _vp()
        rc = self.lib.mvh_model_open(path.encode(), device, ctx, page_tokens, kv_type, act_mode, max_batch,
                                     C.byref(h))
        self._check(rc)
        self.h = h.value
        cfg = (_sz * 7)()
        self._check(self.lib.mvh_model_config(self.h, cfg))
        self.n_ctx, self.n_embd, self.n_ff, self.n_layer, self.n_head, self.n_head_kv, self.vocab = list(cfg)

    def _check(self, rc):
        if rc != 0:
            raise MvhError(rc, self.lib.mvh_last_error().decode())

    def close(self):
        if getattr(self, "h", None):
            self.lib.mvh_model_close(self.h)
            self.h = None

    def __del__(self, _fin=_finalize):
        _fin(self.close)

    def reset(self):
        self._check(self.lib.mvh_model_reset(self.h))

    def forward(self, token: int, logits: bool = True):
        out = np.empty(self.vocab, np.float32) if logits else None
        self._check(self.lib.mvh_model_forward(self.h, int(token), out.ctypes.data if logits else None))
        return out

    def prefill(self, tokens, batch: int = 32, logits: bool = True):
        t = np.ascontiguousarray(tokens, np.int32)
        out = np.empty(self.vocab, np.float32) if logits else None
        self._check(self.lib.mvh_model_prefill(self.h, t.ctypes.data, t.size, batch, out.ctypes.data if logits else None))
        return out

    def generate_greedy(self, token: int, n: int, logits: bool = False):
        ids = np.empty(n, np.int32)
        out = np.empty(self.vocab, np.float32) if logits else None
        self._check(self.lib.mvh_model_generate_greedy(self.h, int(token), n, ids.ctypes.data,
                                                       out.ctypes.data if logits else None))
        return (ids, out) if logits else ids

    @property
    def position(self) -> int:
        p = _sz()
        self._check(self.lib.mvh_model_position(self.h, C.byref(p)))
        return p.value

    def kv_type(self) -> int:
        t = _int()
        self._check(self.lib.mvh_model_kv_type(self.h, C.byref(t)))
        return t.value

    def kv_bytes(self) -> int:
        p = _sz()
        self._check(self.lib.mvh_model_kv_bytes(self.h, C.byref(p)))
        return p.value

    @property
    def stream(self) -> int:
        s = _vp()
        self._check(self.lib.mvh_model_stream(self.h, C.byref(s)))
        return s.value
