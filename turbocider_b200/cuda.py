"""ctypes binding of libturbocider_cuda.so (include/turbocider_cuda.h).

This is the Python face of the C ABI, in the style of the reference's own
ctypes-driven op tests (tests/native/test_gguf_execution.py:67-85).  Device
buffers are torch tensors (PyTorch is used for device memory and streams
only); every computation runs in the CUDA library.  There is no CPU
fallback: loading fails loudly when the library is missing.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

import numpy as np

# TURBOCIDER_CHECKED=1 loads the bounds-checked build (-DTC_BOUNDS_CHECK:
# out-of-range indices set STATUS_BOUNDS instead of faulting).
LIB_PATH = Path(__file__).resolve().parent / ("libturbocider_cuda_checked.so"
                                             if os.environ.get("TURBOCIDER_CHECKED") == "1"
                                             else "libturbocider_cuda.so")

Q4_K, Q5_K, Q6_K = 12, 13, 14
F32, F16, BF16 = 0, 1, 2
STAGE_BF16, STAGE_F16, STAGE_F16_X16 = 0, 1, 2
STATUS_NONFINITE_SCALE, STATUS_F16_OVERFLOW, STATUS_TIMEOUT, STATUS_GEOMETRY, STATUS_BF16_OVERFLOW = 1, 2, 4, 8, 16
STATUS_BOUNDS = 32
EPI_BIAS, EPI_GELU_TANH, EPI_GELU_ERF, EPI_SWIGLU, EPI_GATE_RESIDUAL = 1, 2, 4, 8, 16
BLOCK_BYTES = {Q4_K: 144, Q5_K: 176, Q6_K: 210}

_lib = None


class BackendError(RuntimeError):
    """A failed C-ABI call (status 1); the message is tc_cuda_last_error()."""


class DecodeError(BackendError):
    """Mirror of tc::gguf::DecodeError (reference native/core/gguf_decode.hpp:10-16)."""


class Cancelled(BackendError):
    """A call stopped by its cancel flag (status TC_CUDA_CANCELLED = 2; the
    reference's tc::Cancelled, native/core/common.hpp:19-21)."""


class CancelFlag:
    """A caller-owned cancel flag (int32, nonzero = cancel) for the calls that
    take one: tc_gguf_read, tc_relayout_host, tc_cuda_weight_load_gguf and
    LayerStream.  Thread-safe to set from another thread while a call runs
    (the reference's std::atomic<bool> cancel, gguf_decode.cpp:44-47)."""

    def __init__(self):
        self._v = C.c_int32(0)

    def set(self):
        self._v.value = 1

    def clear(self):
        self._v.value = 0

    @property
    def is_set(self) -> bool:
        return self._v.value != 0

    @property
    def pointer(self):
        return C.byref(self._v)


def _cancel_ptr(cancel):
    return cancel.pointer if cancel is not None else None


class LoadStats(C.Structure):
    """struct tc_gguf_load_stats."""
    _fields_ = [("bytes", C.c_uint64), ("chunks", C.c_uint64), ("seconds", C.c_double),
                ("read_seconds", C.c_double), ("wait_seconds", C.c_double)]


_vp, _u32, _u64, _i32 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int32


class Epilogue(C.Structure):
    """struct tc_epilogue (include/turbocider_cuda.h)."""
    _fields_ = [("flags", _u32), ("n_gate_rows", _u32), ("bias", _vp), ("bias_up_offset", _u64), ("gate", _vp),
                ("ld_gate", _u64), ("seg_gate", C.POINTER(_i32)), ("residual", _vp), ("ld_residual", _u64)]


class _Heads(C.Structure):
    """struct tc_heads."""
    _fields_ = [("x", _vp), ("out", _vp), ("weight", _vp), ("ld_token", _u64), ("ld_head", _u64),
                ("ld_out_token", _u64), ("ld_out_head", _u64), ("n_heads", _u32), ("reserved", _u32)]


class _Rope(C.Structure):
    """struct tc_rope."""
    _fields_ = [("freq", _vp), ("positions", _vp), ("rotary_dim", _u32), ("layout", _u32), ("n_axes", _u32),
                ("sections", _u32 * 4), ("amplitude", C.c_float)]


class _PagedCache(C.Structure):
    """struct tc_paged_cache."""
    _fields_ = [("k", _vp), ("v", _vp), ("ld_page", _u64), ("ld_head", _u64), ("ld_token", _u64), ("n_pages", _u32),
                ("page_size", _u32), ("n_heads", _u32), ("head_dim", _u32), ("dtype", _u32), ("reserved", _u32)]


class _PagedBatch(C.Structure):
    """struct tc_paged_batch."""
    _fields_ = [("new_offsets", _vp), ("lengths", _vp), ("page_table", _vp), ("n_seq", _u32), ("table_width", _u32),
                ("ld_table", _u32), ("n_tokens", _u32), ("max_new", _u32), ("max_length", _u32)]


class _Attention(C.Structure):
    """struct tc_attention."""
    _fields_ = [("q", _vp), ("out", _vp), ("lse", _vp), ("ld_q_token", _u64), ("ld_q_head", _u64),
                ("ld_out_token", _u64), ("ld_out_head", _u64), ("n_heads", _u32), ("causal", _i32), ("window", _i32),
                ("scale", C.c_float)]


class AttentionPlan(C.Structure):
    """struct tc_attention_plan."""
    _fields_ = [("many_rows", _u32), ("rows", _u32), ("ctas_per_sm", _u32), ("share_keys", _u32), ("shares", _u32),
                ("launches", _u32), ("workspace_bytes", _u64)]


EXPORTS = {
    # name: (restype, argtypes)
    "tc_cuda_abi_version": (_u32, []),
    "tc_cuda_last_error": (C.c_char_p, []),
    "tc_cuda_init": (C.c_int, [C.c_int, C.POINTER(_vp)]),
    "tc_cuda_free": (None, [_vp]),
    "tc_cuda_status": (C.c_int, [_vp, C.POINTER(_u32), C.c_int]),
    "tc_cuda_weight_upload": (C.c_int, [_vp, _u32, _u64, _u64, _vp, _u64, _u64, _u64, C.POINTER(_vp)]),
    "tc_cuda_weight_create": (C.c_int, [_vp, _u32, _u64, _u64, C.POINTER(_vp)]),
    "tc_cuda_weight_fill_device": (C.c_int, [_vp, _vp, _vp, _u64, _vp]),
    "tc_cuda_weight_free": (None, [_vp]),
    "tc_cuda_weight_info": (C.c_int, [_vp, C.POINTER(_u32), C.POINTER(_u64), C.POINTER(_u64), C.POINTER(_u64)]),
    "tc_cuda_dequant": (C.c_int, [_vp, _vp, C.c_int, _vp, _u64, _vp]),
    "tc_cuda_decode": (C.c_int, [_vp, _u32, _vp, _u64, _u64, _u64, _u64, _u64, _u64, _u64, C.c_int, _vp, _u64,
                                 _u64, _u64, _vp]),
    "tc_cuda_decode_gather": (C.c_int, [_vp, _u32, _vp, _u64, _u64, _u64, _vp, _u64, _u64, _u64, C.c_int, _vp,
                                        _u64, _u64, _u64, _vp]),
    "tc_cuda_qlinear": (C.c_int, [_vp, C.POINTER(_vp), _u32, C.POINTER(_i32), C.POINTER(_i32), _u32, _vp, _vp,
                                  _u64, C.c_int, C.c_int, _vp]),
    "tc_cuda_qlinear_ex": (C.c_int, [_vp, C.POINTER(_vp), _u32, C.POINTER(_i32), C.POINTER(_i32), _u32, _vp, _vp,
                                     _u64, C.c_int, C.c_int, C.POINTER(Epilogue), _vp]),
    "tc_cuda_weight_upload_glu": (C.c_int, [_vp, _u32, _u64, _u64, _vp, _vp, _u64, _u64, _u64, C.POINTER(_vp)]),
    "tc_cuda_qlinear_gather": (C.c_int, [_vp, C.POINTER(_vp), _u32, C.POINTER(_i32), C.POINTER(_i32), _u32, _vp,
                                         _vp, _u64, C.c_int, C.c_int, C.POINTER(Epilogue), C.POINTER(_vp), _u32,
                                         _vp]),
    "tc_cuda_peer_alloc": (C.c_int, [_vp, _u64, C.POINTER(_vp), _vp]),
    "tc_cuda_peer_open": (C.c_int, [_vp, _vp, C.POINTER(_vp)]),
    "tc_cuda_peer_close": (C.c_int, [_vp, _vp]),
    "tc_cuda_peer_free": (C.c_int, [_vp, _vp]),
    "tc_cuda_peer_barrier": (C.c_int, [_vp, C.POINTER(_vp), _u32, _u32, _u32, _u32, _vp]),
    "tc_cuda_peer_push": (C.c_int, [_vp, _vp, C.POINTER(_vp), _u32, _u64, _u64, _u64, _u64, _vp]),
    "tc_cuda_set_push_fanout": (C.c_int, [_vp, C.c_int]),
    "tc_cuda_set_push_kernel": (C.c_int, [_vp, C.c_int]),
    "tc_cuda_set_path": (C.c_int, [_vp, C.c_int]),
    "tc_cuda_qlinear_batched": (C.c_int, [_vp, C.POINTER(_vp), _u32, _vp, _u32, C.POINTER(_vp), C.POINTER(_u64),
                                          C.c_int, _vp]),
    "tc_cuda_set_sm_limit": (C.c_int, [_vp, C.c_int]),
    "tc_cuda_qlinear_plan": (C.c_int, [_vp, _vp, _u32, C.c_int, C.POINTER(_u32), C.POINTER(_u32)]),
    "tc_quantize": (C.c_int, [_u32, _vp, _u64, _u64, _vp, _u64, C.c_int]),
    "tc_cuda_qlinear_small_static": (C.c_int, [_vp, _vp, _u32, _vp, _u64, C.c_int, _vp]),
    "tc_cuda_small_static_status": (C.c_int, [C.c_int, C.POINTER(_u32), C.c_int]),
    "tc_panel_bytes": (_u64, [_u32, _u64, _u64]),
    "tc_relayout_host": (C.c_int, [_u32, _vp, _u64, _u64, _u64, _u64, _u64, _vp, _u64, C.c_int, _vp]),
    "tc_cuda_weight_copy_panels": (C.c_int, [_vp, _vp, _vp, _u64, _vp]),
    "tc_gguf_open": (C.c_int, [C.c_char_p, C.c_char_p, C.POINTER(_vp)]),
    "tc_gguf_close": (None, [_vp]),
    "tc_gguf_info": (C.c_int, [_vp, C.POINTER(_u32), C.POINTER(_u32), C.POINTER(_u64), C.POINTER(_u64),
                               C.POINTER(_u64)]),
    "tc_gguf_tensor": (C.c_int, [_vp, _u64, C.c_char_p, _u64, C.POINTER(_u32), C.POINTER(_u32), C.POINTER(_u64),
                                 C.POINTER(_u64), C.POINTER(_u64)]),
    "tc_gguf_find": (C.c_int, [_vp, C.c_char_p, C.POINTER(_u64)]),
    "tc_gguf_meta": (C.c_int, [_vp, C.c_char_p, C.POINTER(_u32), C.POINTER(_u64), C.POINTER(C.c_int64),
                               C.POINTER(C.c_double), C.c_char_p, _u64, C.POINTER(_u64)]),
    "tc_gguf_read": (C.c_int, [_vp, _u64, _u64, _u64, _vp, _u64, _vp]),
    "tc_cuda_weight_load_gguf": (C.c_int, [_vp, _vp, _u64, _u64, _u64, _u64, _vp, C.POINTER(_vp),
                                           C.POINTER(LoadStats)]),
    "tc_gguf_validate_split": (C.c_int, [C.POINTER(_vp), _u32]),
    "tc_rope_freqs": (C.c_int, [_u32, C.c_double, _u32, C.c_double, C.c_double, C.c_double, C.c_double, _vp,
                                C.POINTER(C.c_float)]),
    "tc_cuda_qk_norm_rope": (C.c_int, [_vp, C.POINTER(_Heads), C.POINTER(_Heads), _u64, _u32, C.c_int, C.c_int,
                                       C.c_float, C.POINTER(_Rope), _vp]),
    "tc_cuda_kv_append": (C.c_int, [_vp, C.POINTER(_PagedCache), C.POINTER(_PagedBatch), C.POINTER(_Heads),
                                    C.POINTER(_Heads), C.POINTER(_Heads), C.c_int, C.c_float, C.POINTER(_Rope), _vp]),
    "tc_paged_attention_plan": (C.c_int, [_u32, _u32, _u32, _u32, _u32, C.POINTER(_PagedBatch), _i32, _i32,
                                          C.POINTER(AttentionPlan)]),
    "tc_cuda_paged_attention": (C.c_int, [_vp, C.POINTER(_PagedCache), C.POINTER(_PagedBatch),
                                          C.POINTER(_Attention), _vp]),
}


def lib() -> C.CDLL:
    """Load the backend library (built in-tree by turbocider_b200.build)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(f"{LIB_PATH} is missing: run `python -m turbocider_b200.build` "
                              "(the CUDA backend has no CPU fallback)")
        handle = C.CDLL(str(LIB_PATH))
        for name, (res, args) in EXPORTS.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def _check(rc: int, cls=BackendError):
    if rc == 2:
        raise Cancelled(lib().tc_cuda_last_error().decode())
    if rc != 0:
        raise cls(lib().tc_cuda_last_error().decode())


def _stream_ptr(stream) -> int | None:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


def quantize(ggml_type: int, w: np.ndarray, threads: int | None = None) -> np.ndarray:
    """Quantise a fp32 [rows, cols] matrix to raw GGUF blocks (uint8 array)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    rows, cols = w.shape
    out = np.empty(rows * (cols // 256) * BLOCK_BYTES[ggml_type], dtype=np.uint8)
    rc = lib().tc_quantize(ggml_type, w.ctypes.data, rows, cols, out.ctypes.data, out.nbytes,
                           threads or os.cpu_count() or 1)
    if rc != 0:
        raise BackendError("tc_quantize rejected the input (type, shape or nonfinite values)")
    return out


def panel_bytes(ggml_type: int, n: int, k: int) -> int:
    """Bytes of the panel layout of an [n, k] weight (0 = unsupported)."""
    return int(lib().tc_panel_bytes(ggml_type, n, k))


def relayout_host(ggml_type: int, raw, n: int, k: int, n_begin: int = 0, n_count: int = 0, out=None,
                  threads: int | None = None, cancel: CancelFlag | None = None):
    """Panel layout of rows [n_begin, +n_count) of a raw GGUF matrix, built on
    the CPU (uint8 numpy array in, uint8 numpy array or pinned torch tensor
    out).  Raises Cancelled when `cancel` is set while it runs."""
    raw = np.ascontiguousarray(np.frombuffer(raw, dtype=np.uint8) if isinstance(raw, (bytes, bytearray))
                               else raw).view(np.uint8).reshape(-1)
    rows = n_count or (n - n_begin)
    size = panel_bytes(ggml_type, rows, k)
    if out is None:
        out = np.empty(size, dtype=np.uint8)
    ptr = out.data_ptr() if hasattr(out, "data_ptr") else out.ctypes.data
    cap = out.numel() if hasattr(out, "numel") else out.nbytes
    _check(lib().tc_relayout_host(ggml_type, raw.ctypes.data, raw.nbytes, n, k, n_begin, n_count, ptr, cap,
                                  threads or os.cpu_count() or 1, _cancel_ptr(cancel)), DecodeError)
    return out


class Context:
    """A device context: status word and workspace on one GPU."""

    def __init__(self, device: int = 0):
        self._h = _vp()
        _check(lib().tc_cuda_init(device, C.byref(self._h)))
        self.device = device

    @property
    def handle(self):
        return self._h

    def status(self, clear: bool = True) -> int:
        bits = _u32()
        _check(lib().tc_cuda_status(self._h, C.byref(bits), int(clear)))
        return bits.value

    def set_path(self, path: int):
        _check(lib().tc_cuda_set_path(self._h, path))

    def set_sm_limit(self, sms: int):
        """SMs the tensor-core GEMM may occupy (0 = all)."""
        _check(lib().tc_cuda_set_sm_limit(self._h, sms))

    def plan(self, weight, m: int, stage: int = STAGE_BF16) -> tuple[int, int]:
        """(kernel family, K splits) a one-segment call with m rows would use:
        kernel 1 GEMV, 2 2-CTA GEMM, 3 one-CTA GEMM, 4 dense."""
        kern, split = _u32(), _u32()
        _check(lib().tc_cuda_qlinear_plan(self._h, weight.handle, m, stage, C.byref(kern), C.byref(split)))
        return kern.value, split.value

    def set_push_fanout(self, streams: int):
        """Peer pushes spread over `streams` side streams (>= 2) or back to
        back on the caller's stream (0 / 1, the default)."""
        _check(lib().tc_cuda_set_push_fanout(self._h, int(streams)))

    def set_push_kernel(self, ctas: int):
        """Peer pushes by a kernel of `ctas` 128-thread blocks (the SMs store
        over NVLink) for 16-byte-aligned regions; 0 (the default): by the
        copy engines."""
        _check(lib().tc_cuda_set_push_kernel(self._h, int(ctas)))

    def close(self):
        if self._h:
            lib().tc_cuda_free(self._h)
            self._h = _vp()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Weight:
    """A K-quant weight resident in HBM (panel layout)."""

    def __init__(self, ctx: Context, handle, glu: bool = False):
        self.ctx, self._h = ctx, handle
        t, n, k, b = _u32(), _u64(), _u64(), _u64()
        _check(lib().tc_cuda_weight_info(handle, C.byref(t), C.byref(n), C.byref(k), C.byref(b)))
        self.ggml_type, self.n, self.k, self.device_bytes = t.value, n.value, k.value, b.value
        self.glu = glu
        self.n_out = n.value // 2 if glu else n.value   # output columns

    @classmethod
    def upload_glu(cls, ctx: Context, ggml_type: int, f: int, k: int, gate_raw, up_raw, col_begin: int = 0,
                   col_count: int = 0):
        """Gate and up halves of a SwiGLU projection ([f, k] raw GGUF rows each)
        as one interleaved weight for the fused SwiGLU epilogue."""
        def flat(r):
            return np.ascontiguousarray(np.frombuffer(r, dtype=np.uint8) if isinstance(r, (bytes, bytearray))
                                        else r).view(np.uint8).reshape(-1)
        g, u = flat(gate_raw), flat(up_raw)
        h = _vp()
        _check(lib().tc_cuda_weight_upload_glu(ctx.handle, ggml_type, f, k, g.ctypes.data, u.ctypes.data,
                                               min(g.nbytes, u.nbytes), col_begin, col_count, C.byref(h)),
               DecodeError)
        return cls(ctx, h, glu=True)

    @classmethod
    def upload(cls, ctx: Context, ggml_type: int, n: int, k: int, raw, n_begin: int = 0, n_count: int = 0):
        raw = np.ascontiguousarray(np.frombuffer(raw, dtype=np.uint8) if isinstance(raw, (bytes, bytearray))
                                   else raw).view(np.uint8).reshape(-1)
        h = _vp()
        _check(lib().tc_cuda_weight_upload(ctx.handle, ggml_type, n, k, raw.ctypes.data, raw.nbytes, n_begin,
                                           n_count, C.byref(h)), DecodeError)
        return cls(ctx, h)

    @classmethod
    def load_gguf(cls, ctx: Context, file: "GGUFFile", name_or_index, n_begin: int = 0, n_count: int = 0,
                  chunk_bytes: int = 0, cancel: CancelFlag | None = None):
        """Stream a K-quant tensor (or a row shard of it) from a GGUF file into
        HBM with read-ahead (tc_cuda_weight_load_gguf).  Returns (Weight,
        stats dict); raises Cancelled when `cancel` is set while it runs."""
        idx = name_or_index if isinstance(name_or_index, int) else file.tensor(name_or_index)["index"]
        h = _vp()
        st = LoadStats()
        _check(lib().tc_cuda_weight_load_gguf(ctx.handle, file._h, idx, n_begin, n_count, chunk_bytes,
                                              _cancel_ptr(cancel), C.byref(h), C.byref(st)), DecodeError)
        stats = {f: getattr(st, f) for f, _ in LoadStats._fields_}
        return cls(ctx, h), stats

    @classmethod
    def create(cls, ctx: Context, ggml_type: int, n: int, k: int):
        h = _vp()
        _check(lib().tc_cuda_weight_create(ctx.handle, ggml_type, n, k, C.byref(h)))
        return cls(ctx, h)

    def copy_panels(self, panels, stream=None):
        """Asynchronous copy of panel-layout bytes (tc_relayout_host output,
        pinned host or device torch uint8 tensor) into this weight."""
        _check(lib().tc_cuda_weight_copy_panels(self.ctx.handle, self._h, panels.data_ptr(), panels.numel(),
                                                _stream_ptr(stream)))

    def fill_device(self, raw_device, stream=None):
        """Re-layout raw GGUF rows already in device memory (torch uint8 tensor)."""
        _check(lib().tc_cuda_weight_fill_device(self.ctx.handle, self._h, raw_device.data_ptr(),
                                                raw_device.numel(), _stream_ptr(stream)))

    @property
    def handle(self):
        return self._h

    def free(self):
        if self._h:
            lib().tc_cuda_weight_free(self._h)
            self._h = _vp()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def dequant(ctx: Context, w: Weight, dtype: int = BF16, out=None, stream=None):
    """Dequantise an uploaded weight into a dense torch tensor [n, k]."""
    import torch
    tdt = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[dtype]
    if out is None:
        out = torch.empty((w.n, w.k), dtype=tdt, device=f"cuda:{ctx.device}")
    _check(lib().tc_cuda_dequant(ctx.handle, w.handle, dtype, out.data_ptr(), out.stride(0), _stream_ptr(stream)))
    return out


def decode(ctx: Context, ggml_type: int, source, source_rows: int, source_columns: int, row_begin: int, rows: int,
           column_begin: int, columns: int, dtype: int, target, row_stride: int, column_stride: int,
           stream=None, check: bool = True):
    """Device mirror of decode_cpu_into on raw GGUF bytes (torch uint8 tensors).

    Raises DecodeError with the reference's message for geometry errors, and
    (when check=True, which synchronises) for nonfinite scales / fp16
    overflow detected by the kernel.
    """
    _check(lib().tc_cuda_decode(ctx.handle, ggml_type, source.data_ptr(), source.numel() * source.element_size(),
                                source_rows, source_columns, row_begin, rows, column_begin, columns, dtype,
                                target.data_ptr(), target.numel() * target.element_size(), row_stride,
                                column_stride, _stream_ptr(stream)), DecodeError)
    if check:
        bits = ctx.status(clear=True)
        if bits & STATUS_NONFINITE_SCALE:
            # The reference's checked copy (same floating type as the target,
            # contiguous columns) words this error differently from its
            # decoder (gguf_decode.cpp:136-158 vs :43).
            same = (ggml_type, dtype) in ((0, F32), (1, F16), (30, BF16))
            if same and column_stride == (4 if dtype == F32 else 2):
                raise DecodeError("nonfinite source float")
            raise DecodeError("nonfinite weight/scale or conversion overflow")
        if bits & STATUS_F16_OVERFLOW:
            raise DecodeError("FP16 conversion overflow")
        if bits & STATUS_BF16_OVERFLOW:
            raise DecodeError("BF16 conversion overflow")


def decode_gather(ctx: Context, ggml_type: int, source, source_rows: int, source_columns: int, indices,
                  column_begin: int, columns: int, dtype: int, target, row_stride: int, column_stride: int,
                  stream=None, check: bool = True):
    """Device mirror of decode_cpu_gather: target row r = source row
    indices[r] (device int64 / uint64 tensor).  Raises DecodeError with the
    reference's messages; with check=True (synchronises) also for an index
    past the matrix and for value errors detected by the kernel."""
    _check(lib().tc_cuda_decode_gather(ctx.handle, ggml_type, source.data_ptr(),
                                       source.numel() * source.element_size(), source_rows, source_columns,
                                       indices.data_ptr(), indices.numel(), column_begin, columns, dtype,
                                       target.data_ptr(), target.numel() * target.element_size(), row_stride,
                                       column_stride, _stream_ptr(stream)), DecodeError)
    if check:
        bits = ctx.status(clear=True)
        if bits & STATUS_GEOMETRY:
            raise DecodeError("gather row out of bounds")
        if bits & STATUS_NONFINITE_SCALE:
            raise DecodeError("nonfinite weight/scale or conversion overflow")
        if bits & STATUS_F16_OVERFLOW:
            raise DecodeError("FP16 conversion overflow")
        if bits & STATUS_BF16_OVERFLOW:
            raise DecodeError("BF16 conversion overflow")


def _torch_dtype(out_dtype: int):
    import torch
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[out_dtype]


def qlinear(ctx: Context, weights, x, seg_offsets=None, seg_weight=None, out_dtype: int = BF16,
            stage: int = STAGE_BF16, out=None, stream=None, bias=None, activation: str | None = None,
            gate=None, residual=None, seg_gate=None, bias_up_offset: int | None = None, peers=None):
    """Y = X * W^T through tc_cuda_qlinear_ex.  `weights` is a Weight or a list
    of them; seg_offsets / seg_weight describe ragged request segments along M.

    Fused epilogue (all optional; f32 device tensors unless noted):
      bias        [rows] (SwiGLU weight: gate biases then up biases, up at
                  bias_up_offset, default n_out);
      activation  "gelu_tanh" | "gelu_erf" (SwiGLU weights always apply
                  silu(gate) * up);
      gate, residual  y = residual + gate[seg_gate[s]] * t; gate [G, n_out]
                  f32, residual [M, n_out] in the output dtype (may be `out`).
    peers: device addresses of replicas of `out` on other ranks (same layout;
    tc_cuda_qlinear_gather) -- every output is also stored there.
    """
    import torch
    ws = weights if isinstance(weights, (list, tuple)) else [weights]
    m = x.shape[0]
    if seg_offsets is None:
        seg_offsets = [0, m]
    seg_offsets = list(seg_offsets)
    n_seg = len(seg_offsets) - 1
    offs = (_i32 * len(seg_offsets))(*seg_offsets)
    sw = (_i32 * n_seg)(*seg_weight) if seg_weight is not None else None
    handles = (_vp * len(ws))(*[w.handle for w in ws])
    n_out = getattr(ws[0], "n_out", ws[0].n)
    if out is None:
        out = torch.empty((m, n_out), dtype=_torch_dtype(out_dtype), device=x.device)
    epi = Epilogue()
    if bias is not None:
        epi.flags |= EPI_BIAS
        epi.bias = bias.data_ptr()
        epi.bias_up_offset = n_out if bias_up_offset is None else bias_up_offset
    if activation is not None:
        epi.flags |= {"gelu_tanh": EPI_GELU_TANH, "gelu_erf": EPI_GELU_ERF}[activation]
    if getattr(ws[0], "glu", False):
        epi.flags |= EPI_SWIGLU
    if gate is not None or residual is not None:
        epi.flags |= EPI_GATE_RESIDUAL
        epi.gate = gate.data_ptr() if gate is not None else None
        epi.ld_gate = gate.stride(0) if gate is not None else 0
        epi.n_gate_rows = gate.shape[0] if gate is not None else 0
        epi.residual = residual.data_ptr() if residual is not None else None
        epi.ld_residual = residual.stride(0) if residual is not None else 0
        if seg_gate is not None:
            epi.seg_gate = (_i32 * n_seg)(*seg_gate)
    peers = list(peers or [])
    pv = (_vp * max(1, len(peers)))(*peers) if peers else None
    _check(lib().tc_cuda_qlinear_gather(ctx.handle, handles, len(ws), offs, sw, n_seg, x.data_ptr(),
                                        out.data_ptr(), out.stride(0), out_dtype, stage,
                                        C.byref(epi) if epi.flags else None, pv, len(peers), _stream_ptr(stream)))
    return out


def qlinear_batched(ctx: Context, weights, x, out_dtype: int = BF16, outs=None, stream=None):
    """[X * W_i^T for W_i in weights] in one GEMV launch per weight type (1..16
    rows of bf16 X, weights sharing K)."""
    import torch
    if outs is None:
        outs = [torch.empty((x.shape[0], w.n), dtype=_torch_dtype(out_dtype), device=x.device) for w in weights]
    handles = (_vp * len(weights))(*[w.handle for w in weights])
    ys = (_vp * len(outs))(*[o.data_ptr() for o in outs])
    lds = (_u64 * len(outs))(*[o.stride(0) for o in outs])
    _check(lib().tc_cuda_qlinear_batched(ctx.handle, handles, len(weights), x.data_ptr(), x.shape[0], ys, lds,
                                         out_dtype, _stream_ptr(stream)))
    return outs


def qlinear_small_static(weight: Weight, x, out_dtype: int = BF16, out=None, stream=None):
    """Y = X * W^T for 1..16 rows of X through the allocation-free entry point
    (static device scratch instead of a context workspace)."""
    import torch
    if out is None:
        out = torch.empty((x.shape[0], weight.n), dtype=_torch_dtype(out_dtype), device=x.device)
    _check(lib().tc_cuda_qlinear_small_static(weight.handle, x.data_ptr(), x.shape[0], out.data_ptr(),
                                              out.stride(0), out_dtype, _stream_ptr(stream)))
    return out


def small_static_status(device: int = 0, clear: bool = True) -> int:
    """TC_STATUS_* bits accumulated by qlinear_small_static on `device`
    (synchronises the device; clear resets them)."""
    bits = _u32()
    _check(lib().tc_cuda_small_static_status(device, C.byref(bits), int(clear)))
    return bits.value


# ------------------------------------------------------------ attention
_ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
_ROPE_SCALINGS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
_torch = None          # torch, its types and its stream query, looked up once: these calls are short


def _torch_once():
    global _torch
    if _torch is None:
        import torch

        class T:
            dtypes = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
            f32, f64, i32, dense = torch.float32, torch.float64, torch.int32, torch.contiguous_format
            empty, empty_like = torch.empty, torch.empty_like
            # address of a device's current stream without building a Stream object
            raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
                lambda device: torch.cuda.current_stream(device).cuda_stream)
        _torch = T
    return _torch


def _dtype_id(t) -> int:
    i = _torch_once().dtypes.get(t.dtype)
    if i is None:
        raise BackendError("tensors must be f32, f16 or bf16")
    return i


def _stream_of(ctx: Context, stream) -> int:
    """Address of `stream`; None: the current stream of the context's device."""
    if stream is None:
        return _torch_once().raw_stream(ctx.device)
    return getattr(stream, "cuda_stream", stream)


def _ints(t, what: str, dims: int, device: int) -> int:
    """Address of a contiguous int32 tensor on `device`."""
    if t.dtype is not _torch_once().i32 or t.get_device() != device or t.dim() != dims or not t.is_contiguous():
        raise BackendError(f"{what} must be a contiguous int32 tensor of {dims} dimension(s) on the others' device")
    return t.data_ptr()


def _same_device(device: int, *parts) -> None:
    for part in parts:
        if part is not None and part.device != device:
            raise BackendError("every tensor of a call must be on the context's device")


def rope_freqs(rotary_dim: int, theta: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
               trained_length: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None):
    """(freq, amplitude) of a rotation for Rope: freq a float64 tensor
    [rotary_dim / 2] of radians per position on `device` (None: the CPU).
    scaling: "plain", "linear", "ntk", "yarn" or "bands" (struct tc_rope's
    helper tc_rope_freqs has the formulas)."""
    import torch
    if scaling not in _ROPE_SCALINGS:
        raise BackendError("unknown rotation scaling")
    freq = torch.empty(max(rotary_dim // 2, 1), dtype=torch.float64)
    amplitude = C.c_float()
    _check(lib().tc_rope_freqs(rotary_dim, theta, _ROPE_SCALINGS[scaling], factor, trained_length, beta_fast,
                               beta_slow, freq.data_ptr(), C.byref(amplitude)))
    return (freq if device is None else freq.to(device)), amplitude.value


class Rope:
    """A position rotation (struct tc_rope).  freq: float64 device tensor of
    radians per position, one for each rotated pair (rope_freqs).  positions:
    int32 device tensor [tokens] or [tokens, axes]; None with kv_append: each
    token's place in its cache.  layout: "half" (pairs i, i + rotary_dim / 2)
    or "interleaved" (2i, 2i + 1).  sections: pairs of each axis."""

    __slots__ = ("c", "freq", "positions", "device")

    def __init__(self, freq, positions=None, layout: str = "half", sections=None, amplitude: float = 1.0):
        device = self.device = freq.get_device()
        if freq.dtype is not _torch_once().f64 or device < 0 or freq.dim() != 1 or not freq.is_contiguous():
            raise BackendError("freq must be a contiguous float64 device vector")
        layout = _ROPE_LAYOUTS.get(layout)
        if layout is None:
            raise BackendError("invalid rotation layout")
        c, pairs, axes = _Rope(), freq.numel(), 1
        self.freq, self.positions, self.c = freq, positions, c
        if positions is not None:
            shape = positions.shape
            if len(shape) == 2:
                axes = shape[1]
            c.positions = _ints(positions, "positions", 2 if len(shape) == 2 else 1, device)
        if axes != (1 if sections is None else len(sections)) or not 1 <= axes <= 4:
            raise BackendError("one section for each of 1 to 4 position axes")
        if axes > 1:
            c.sections = tuple(sections) + (0,) * (4 - axes)
        elif sections is not None and sections[0] != pairs:
            raise BackendError("the sections must add up to rotary_dim / 2")
        c.freq, c.rotary_dim, c.layout, c.n_axes, c.amplitude = freq.data_ptr(), 2 * pairs, layout, axes, amplitude


class PagedCache:
    """Keys and values in pages (struct tc_paged_cache): two f16 or bf16
    device tensors [pages, heads, page_size, head_dim], or with
    token_major=True [pages, page_size, heads, head_dim], of the same strides,
    the last one contiguous."""

    __slots__ = ("c", "k", "v", "dtype", "head_dim", "n_heads", "page_size", "device")

    def __init__(self, k, v, token_major: bool = False):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise BackendError("keys and values must be 4-dimensional tensors of the same shape, strides and type")
        self.device = k.get_device()
        if self.device < 0 or v.get_device() != self.device or k.stride(3) != 1:
            raise BackendError("the cache must be device tensors with a contiguous head dimension")
        token, head = (1, 2) if token_major else (2, 1)
        self.k, self.v, self.dtype = k, v, k.dtype
        self.head_dim, self.n_heads, self.page_size = k.shape[3], k.shape[head], k.shape[token]
        c = self.c = _PagedCache()
        c.k, c.v, c.dtype = k.data_ptr(), v.data_ptr(), _dtype_id(k)
        c.ld_page, c.ld_head, c.ld_token = k.stride(0), k.stride(head), k.stride(token)
        c.n_pages, c.page_size, c.n_heads, c.head_dim = k.shape[0], self.page_size, self.n_heads, self.head_dim


class PagedBatch:
    """The new tokens of a step (struct tc_paged_batch): int32 device tensors
    new_offsets [requests + 1], lengths [requests] (cached tokens, the new
    ones included) and page_table [requests, width]; max_new and max_length
    bound the new tokens and the length of every request."""

    __slots__ = ("c", "tensors", "device")

    def __init__(self, new_offsets, lengths, page_table, max_new: int, max_length: int):
        n, shape, strides = lengths.numel(), page_table.shape, page_table.stride()
        if len(shape) != 2 or shape[0] != n or new_offsets.numel() != n + 1:
            raise BackendError("new_offsets, lengths and page_table must have requests + 1, requests and requests rows")
        device = self.device = page_table.get_device()
        if page_table.dtype is not _torch_once().i32 or device < 0 or (strides[1] != 1 and shape[1] > 1):
            raise BackendError("page_table must be an int32 device tensor with contiguous rows")
        if not (0 <= max_new < 2**32 and 0 <= max_length < 2**32):
            raise BackendError("max_new and max_length must not be negative nor pass 32 bits")
        self.tensors = (new_offsets, lengths, page_table)
        c = self.c = _PagedBatch()
        c.new_offsets, c.lengths = _ints(new_offsets, "new_offsets", 1, device), _ints(lengths, "lengths", 1, device)
        c.page_table, c.n_seq, c.table_width = page_table.data_ptr(), n, shape[1]
        c.ld_table = strides[0] if n > 1 else shape[1]
        c.max_new, c.max_length = max_new, max_length


def _heads(device: int, x, out, weight, what: str, fresh: bool = False):
    """(struct tc_heads, out) of a [tokens, heads, head_dim] tensor on the
    context's device; fresh: a contiguous result is allocated where out is
    None."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or x.get_device() != device or (strides[2] != 1 and shape[2] > 1):
        raise BackendError(f"{what} must be [tokens, heads, head_dim] with a contiguous last dimension on the "
                           "context's device")
    _, heads, dim = shape
    h = _Heads()
    h.x, h.n_heads, h.ld_token, h.ld_head = x.data_ptr(), heads, strides[0], strides[1]
    if out is not None:
        strides = out.stride()
        if out.shape != shape or out.dtype is not x.dtype or out.get_device() != device or \
                (strides[2] != 1 and dim > 1):
            raise BackendError(f"the result of {what} must have its shape, type and device")
        h.out, h.ld_out_token, h.ld_out_head = out.data_ptr(), strides[0], strides[1]
    elif fresh:
        out = _torch.empty_like(x, memory_format=_torch.dense)
        h.out, h.ld_out_token, h.ld_out_head = out.data_ptr(), heads * dim, dim
    if weight is not None:
        if weight.dtype is not _torch.f32 or weight.shape != (dim,) or not weight.is_contiguous() or \
                weight.get_device() != device:
            raise BackendError("norm weights must be float32 device vectors of head_dim elements")
        h.weight = weight.data_ptr()
    return h, out


def qk_norm_rope(ctx: Context, q, k=None, rope: Rope | None = None, q_weight=None, k_weight=None,
                 eps: float | None = None, q_out=None, k_out=None, stream=None):
    """RMS norm over each head (eps None: no norm) and position rotation (rope
    None: none) of query and key heads [tokens, heads, head_dim] in one
    launch.  Weights: f32 [head_dim], the norm's (not read without one).
    q_out / k_out may be q / k.  Returns (q_out, k_out).  Results that are not
    passed in come from the current stream's memory: with another `stream`,
    pass them or order the two."""
    dtype, hk = _dtype_id(q), None
    device = ctx.device
    hq, q_out = _heads(device, q, q_out, q_weight, "q", True)
    tokens, _, dim = q.shape
    if k is not None:
        shape = k.shape
        if len(shape) != 3 or k.dtype is not q.dtype or shape[0] != tokens or shape[2] != dim:
            raise BackendError("q and k must share their type, tokens and head_dim")
        hk, k_out = _heads(device, k, k_out, k_weight, "k", True)
    _same_device(device, rope)
    if rope is not None and rope.positions is not None and rope.positions.shape[0] != tokens:
        raise BackendError("one position for each token")
    _check(lib().tc_cuda_qk_norm_rope(ctx.handle, hq, hk, tokens, dim, dtype, eps is not None, eps or 0.0,
                                      None if rope is None else rope.c, _stream_of(ctx, stream)))
    return q_out, k_out


def kv_append(ctx: Context, cache: PagedCache, batch: PagedBatch, k, v, rope: Rope | None = None, q=None,
              q_weight=None, k_weight=None, eps: float | None = None, q_out=None, stream=None):
    """Writes the step's keys (normed with eps not None, rotated with rope)
    and values [tokens, heads, head_dim] to the cache and, in the same launch,
    norms and rotates the queries.  Returns q_out (None without q; where it is
    not passed in it comes from the current stream's memory, as with
    qk_norm_rope)."""
    shape, device = k.shape, ctx.device
    if k.dtype is not cache.dtype or v.dtype is not cache.dtype or v.shape != shape or len(shape) != 3 or \
            shape[2] != cache.head_dim:
        raise BackendError("keys and values must have the cache's type and head_dim")
    tokens, hq = shape[0], None
    if rope is not None and rope.positions is not None and rope.positions.shape[0] != tokens:
        raise BackendError("one position for each token")
    if q is not None:
        if q.dtype is not cache.dtype or len(q.shape) != 3 or q.shape[0] != tokens or q.shape[2] != shape[2]:
            raise BackendError("queries must have the cache's type and head_dim and one row for each key")
        hq, q_out = _heads(device, q, q_out, q_weight, "q", True)
    _same_device(device, cache, batch, rope)
    batch.c.n_tokens = tokens
    _check(lib().tc_cuda_kv_append(ctx.handle, cache.c, batch.c, _heads(device, k, None, k_weight, "k")[0],
                                   _heads(device, v, None, None, "v")[0], hq, eps is not None, eps or 0.0,
                                   None if rope is None else rope.c, _stream_of(ctx, stream)))
    return q_out if q is not None else None


def paged_attention(ctx: Context, cache: PagedCache, batch: PagedBatch, q, scale: float | None = None,
                    causal: bool = True, window: int = 0, out=None, return_lse: bool = False, stream=None):
    """softmax(scale q K^T) V of the step's queries [tokens, heads, head_dim]
    over each request's cache (scale None: head_dim ** -0.5); query heads share
    cache heads in equal groups.  window > 0: only positions nearer than that.
    Returns out, or (out, lse) with lse f32 [tokens, heads], of the current
    stream's memory where they are not passed in, as with qk_norm_rope.  Calls
    on one context share its workspace and follow one another in stream
    order."""
    t = _torch_once()
    shape, strides = q.shape, q.stride()
    device = ctx.device
    if len(shape) != 3 or q.dtype is not cache.dtype or q.get_device() != device or shape[2] != cache.head_dim or \
            strides[2] != 1:
        raise BackendError("queries must be [tokens, heads, head_dim] of the cache's type and head_dim on the "
                           "context's device")
    a = _Attention()
    a.q, a.ld_q_token, a.ld_q_head, a.n_heads = q.data_ptr(), strides[0], strides[1], shape[1]
    if out is None:
        out = t.empty_like(q, memory_format=t.dense)
        strides = (shape[1] * shape[2], shape[2])
    else:
        strides = out.stride()
        if out.shape != shape or out.dtype is not q.dtype or out.get_device() != device or strides[2] != 1:
            raise BackendError("the result must have the queries' shape, type and device")
    a.out, a.ld_out_token, a.ld_out_head = out.data_ptr(), strides[0], strides[1]
    if return_lse:
        lse = t.empty(shape[:2], dtype=t.f32, device=q.device)
        a.lse = lse.data_ptr()
    # (positions stay below 2^30: a wider window hides as much as the widest one the struct holds)
    a.causal, a.window, a.scale = causal, min(max(window, -1), 2**31 - 1), shape[2] ** -0.5 if scale is None else scale
    _same_device(device, cache, batch)
    batch.c.n_tokens = shape[0]
    _check(lib().tc_cuda_paged_attention(ctx.handle, cache.c, batch.c, a, _stream_of(ctx, stream)))
    return (out, lse) if return_lse else out


def attention_plan(n_heads: int, cache_heads: int, head_dim: int, requests: int, tokens: int, max_new: int,
                   max_length: int, causal: bool = True, window: int = 0, page_size: int = 16,
                   table_width: int | None = None, sms: int = 148) -> AttentionPlan:
    """How paged_attention divides a call of these sizes on a GPU of `sms` SMs
    (tc_paged_attention_plan; needs no GPU)."""
    b, plan = _PagedBatch(), AttentionPlan()
    b.n_seq, b.n_tokens, b.max_new, b.max_length = requests, tokens, max_new, max_length
    b.table_width = -(-max_length // page_size) if table_width is None else table_width
    _check(lib().tc_paged_attention_plan(sms, n_heads, cache_heads, head_dim, page_size, b, causal,
                                         min(max(window, -1), 2**31 - 1), plan))
    return plan


class GGUFError(BackendError):
    """A GGUF file the reader rejects (message as the reference's gguf_invalid: ...)."""


class GGUFFile:
    """A parsed GGUF container (tc_gguf_*): directory, metadata lookup and
    row-range payload reads into host memory."""

    def __init__(self, path, limit: str | None = None):
        self._h = _vp()
        rc = lib().tc_gguf_open(str(path).encode(), limit.encode() if limit else None, C.byref(self._h))
        _check(rc, GGUFError)
        v, a, n, d, nm = _u32(), _u32(), _u64(), _u64(), _u64()
        _check(lib().tc_gguf_info(self._h, C.byref(v), C.byref(a), C.byref(n), C.byref(d), C.byref(nm)), GGUFError)
        self.version, self.alignment, self.data_offset = v.value, a.value, d.value
        self.tensors = [self._tensor(i) for i in range(n.value)]
        self.n_metadata = nm.value

    def _tensor(self, i: int) -> dict:
        name = C.create_string_buffer(4096)
        t, r, off, nb = _u32(), _u32(), _u64(), _u64()
        dims = (_u64 * 4)()
        _check(lib().tc_gguf_tensor(self._h, i, name, 4096, C.byref(t), C.byref(r), dims, C.byref(off),
                                    C.byref(nb)), GGUFError)
        d = list(dims)[:r.value]
        rows = 1
        for x in d[1:]:
            rows *= x
        return {"name": name.value.decode(), "type": t.value, "dims": d, "rows": rows, "columns": d[0],
                "file_offset": off.value, "bytes": nb.value}

    def tensor(self, name: str) -> dict:
        idx = _u64()
        _check(lib().tc_gguf_find(self._h, name.encode(), C.byref(idx)), GGUFError)
        return dict(self.tensors[idx.value], index=idx.value)

    def meta(self, key: str):
        t, u, i, f, cnt = _u32(), _u64(), C.c_int64(), C.c_double(), _u64()
        text = C.create_string_buffer(1 << 20)
        _check(lib().tc_gguf_meta(self._h, key.encode(), C.byref(t), C.byref(u), C.byref(i), C.byref(f), text,
                                  1 << 20, C.byref(cnt)), GGUFError)
        kind = t.value
        if kind == 8:
            return text.value.decode()
        if kind == 9:
            return ("array", cnt.value)
        if kind in (6, 12):
            return f.value
        if kind in (1, 3, 5, 11):
            return i.value
        return u.value

    def read(self, name_or_index, row_begin: int = 0, rows: int | None = None, out=None,
             cancel: CancelFlag | None = None) -> np.ndarray:
        """Raw block bytes of rows [row_begin, +rows) into `out` (a uint8
        numpy array or a pinned torch uint8 tensor; allocated if None).
        Raises Cancelled when `cancel` is set while it reads."""
        info = self.tensors[name_or_index] if isinstance(name_or_index, int) else self.tensor(name_or_index)
        idx = name_or_index if isinstance(name_or_index, int) else info["index"]
        rows = info["rows"] - row_begin if rows is None else rows
        nbytes = info["bytes"] // info["rows"] * rows
        if out is None:
            out = np.empty(nbytes, dtype=np.uint8)
        ptr = out.data_ptr() if hasattr(out, "data_ptr") else out.ctypes.data
        size = out.numel() if hasattr(out, "numel") else out.nbytes
        _check(lib().tc_gguf_read(self._h, idx, row_begin, rows, ptr, size, _cancel_ptr(cancel)), GGUFError)
        return out

    @staticmethod
    def validate_split(files) -> None:
        arr = (_vp * len(files))(*[f._h for f in files])
        _check(lib().tc_gguf_validate_split(arr, len(files)), GGUFError)

    def close(self):
        if self._h:
            lib().tc_gguf_close(self._h)
            self._h = _vp()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
