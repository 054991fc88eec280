"""ctypes binding of the op-level C ABI (include/omni_b200.h).

Mirrors the reference's binding style (omni-tokenizer
python/omni_tokenizer/native.py:36-139: one Library object, every signature
declared at load, non-zero status raised as NativeError with the thread-local
message).  No tensor framework is needed here; the helpers at the bottom
accept torch tensors only as holders of device pointers.
"""

from __future__ import annotations

import contextlib
import ctypes as C
import functools
import os
from pathlib import Path

PKG = Path(__file__).resolve().parent

F32, BF16, F16, E4M3 = 0, 1, 2, 3

# omni_status (include/omni/omni.h)
OK, INVALID_ARGUMENT, IO_ERROR, INVALID_MODEL, UNSUPPORTED, OUT_OF_MEMORY, CANCELLED, INTERNAL_ERROR = range(8)


class NativeError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(message)
        self.status = status


_P = C.c_void_p
SIGNATURES = {
    "omni_b200_last_error": (C.c_char_p, []),
    "omni_b200_version": (C.c_char_p, []),
    "omni_b200_sync_check": (C.c_int, [_P]),
    "omni_b200_wait_selftest": (C.c_int, [C.c_uint, _P]),
    "omni_b200_debug_fail_allocations": (None, [C.c_int]),
    "omni_b200_attention_bhld": (
        C.c_int,
        [_P, _P, _P, _P, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, _P, C.c_int, C.c_int, C.c_float, _P],
    ),
    "omni_b200_attention_rows_workspace": (C.c_size_t, [C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_int]),
    "omni_b200_attention_rows": (
        C.c_int,
        [_P, _P, _P, _P, C.c_size_t, C.c_int, C.c_int, C.c_size_t, C.c_size_t, C.c_int, C.c_int, C.c_int, _P,
         C.c_size_t, _P],
    ),
    "omni_b200_attention_rows_batch_workspace": (
        C.c_size_t, [C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "omni_b200_attention_rows_batch": (
        C.c_int,
        [_P, _P, _P, _P, C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_size_t, _P, C.c_int, C.c_int,
         C.c_int, _P, C.c_size_t, _P],
    ),
    "omni_b200_gelu": (C.c_int, [_P, C.c_size_t, C.c_int, _P]),
    "omni_b200_rms_norm": (
        C.c_int,
        [_P, _P, _P, _P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_float,
         C.c_int, C.c_int, _P],
    ),
    "omni_b200_quantize_e4m3": (
        C.c_int, [_P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int, C.c_int, _P],
    ),
    "omni_b200_linear_e4m3": (
        C.c_int,
        [_P, _P, _P, _P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int, _P],
    ),
    "omni_b200_attention_window": (
        C.c_int,
        [_P, _P, _P, _P, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, _P, _P, _P, C.c_int, C.c_int, C.c_int,
         C.c_float, C.c_int, C.c_int, _P],
    ),
    "omni_b200_rotary": (C.c_int, [_P] * 7 + [C.c_int] * 7 + [_P, _P] + [C.c_int] * 5 + [_P]),
    "omni_b200_cache_e2m1_bytes": (C.c_size_t, [C.c_size_t, C.c_int]),
    "omni_b200_cache_write_e2m1": (C.c_int, [_P] * 5 + [C.c_int] * 4 + [_P, C.c_int, _P]),
    "omni_b200_cache_read_e2m1": (C.c_int, [_P] * 5 + [C.c_int] * 4 + [_P, C.c_int, _P]),
    "omni_b200_attention_window_e2m1_workspace": (C.c_size_t, [C.c_int] * 9),
    "omni_b200_attention_window_e2m1": (
        C.c_int,
        [_P] * 5 + [C.c_int] * 6 + [_P, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int, C.c_int, _P, C.c_size_t, _P],
    ),
    "omni_b200_squares": (C.c_int, [_P, _P, C.c_size_t, C.c_size_t, C.c_int, C.c_int, _P]),
    "omni_b200_vq_argmin": (
        C.c_int,
        [_P, _P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int, C.c_int, _P, C.c_size_t, _P],
    ),
    "omni_b200_vq_argmin_cancellable": (
        C.c_int,
        [_P, _P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int, C.c_int, _P, C.c_size_t, _P, _P],
    ),
    "omni_b200_vq_workspace": (C.c_size_t, [C.c_size_t, C.c_size_t, C.c_size_t, C.c_int]),
    "omni_b200_context_create": (C.c_int, [C.c_int, C.POINTER(_P)]),
    "omni_b200_context_free": (None, [_P]),
    "omni_b200_context_peak_workspace": (C.c_uint64, [_P]),
    "omni_b200_attention_bhld_host": (
        C.c_int,
        [_P, _P, _P, _P, _P, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, _P, C.c_int, C.c_int, C.c_float],
    ),
    "omni_b200_vq_argmin_host": (
        C.c_int, [_P, _P, _P, _P, _P, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int, C.c_int],
    ),
}


class Library:
    """The B200 hot-path library.  Raises NativeError(UNSUPPORTED) when the
    shared library is missing -- there is no CPU fallback."""

    def __init__(self, path=None):
        explicit = path or os.environ.get("OMNI_B200_LIBRARY")
        found = Path(explicit) if explicit else PKG / "libomni_b200.so"
        if not found.is_file():
            raise NativeError(UNSUPPORTED, f"B200 library not found at {found}; run omni-tokenizer_b200/build.py")
        self.path = found.resolve()
        self.lib = C.CDLL(str(self.path))
        missing = [name for name in SIGNATURES if not hasattr(self.lib, name)]
        if missing:
            raise NativeError(UNSUPPORTED, f"{self.path} lacks {', '.join(missing)}; rebuild it")
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(self.lib, name)
            fn.restype, fn.argtypes = res, args

    def check(self, status):
        if status:
            msg = self.lib.omni_b200_last_error()
            raise NativeError(status, msg.decode("utf-8", "replace") if msg else f"native error {status}")

    def version(self):
        return self.lib.omni_b200_version().decode()

    def sync_check(self, stream=None):
        self.check(self.lib.omni_b200_sync_check(stream))


_LIB = None


def library() -> Library:
    global _LIB
    if _LIB is None:
        _LIB = Library()
    return _LIB


# ----------------------------------------------------------------- torch helpers
def _dtype_code(t):
    import torch

    return {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}[t.dtype]


def _stream_ptr(stream):
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _on(what, stream, t):
    """The context in which a helper that was given a stream makes tensors on t's device (t may
    be its number): a call with stream=s is the call made inside torch.cuda.stream(s).  Outputs and workspaces, those
    that are dropped at once among them, are memory of that stream, so that no kernel
    pending on the current stream has it, and none there gets it before the call is over.
    (Entering the stream takes the host 8 us; calls that make no tensor are launched on it
    without.)"""
    device = t if isinstance(t, int) else t.get_device()
    if not hasattr(stream, "device_index"):  # another library's, known by its cuda_stream
        stream = _t.cuda.ExternalStream(stream.cuda_stream, device=device)
    if 0 <= device != stream.device_index:
        _refuse(f"{what}: stream must be on the tensors' device")
    if device >= 0 and device == _t.current_device() and stream.cuda_stream == _t.raw_stream(device):
        return contextlib.nullcontext()
    return _t.cuda.stream(stream)


def attention_bhld(q, k, v, out=None, lengths=None, block=0, skip_padded_queries=False, scale=0.0,
                   out_dtype=None, stream=None):
    """Head-major batched attention: q, k, v are CUDA tensors [B, H, L, D]."""
    import torch

    if stream is not None and out is None:
        with _on("attention_bhld", stream, q):
            return attention_bhld(q, k, v, out, lengths, block, skip_padded_queries, scale, out_dtype)
    B, H, L, D = q.shape
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=q.device)
    lib = library()
    lib.check(lib.lib.omni_b200_attention_bhld(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, L, D, _dtype_code(q),
        _dtype_code(out), lengths.data_ptr() if lengths is not None else None, block,
        int(bool(skip_padded_queries)), float(scale), _stream_ptr(stream)))
    return out


class Context:
    """Host-buffer entry points bound to one device (omni_b200_context)."""

    def __init__(self, device=0, lib=None):
        self.lib = lib or library()
        self.handle = C.c_void_p()
        self.lib.check(self.lib.lib.omni_b200_context_create(int(device), C.byref(self.handle)))

    def close(self):
        if self.handle:
            self.lib.lib.omni_b200_context_free(self.handle)
            self.handle = C.c_void_p()

    __del__ = close

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    @property
    def peak_workspace_bytes(self):
        return int(self.lib.lib.omni_b200_context_peak_workspace(self.handle))

    def attention_bhld(self, q, k, v, out, batch, heads, L, head_dim, dtype, out_dtype, lengths=None, block=0,
                       skip_padded_queries=False, scale=0.0):
        """q, k, v, out, lengths: host addresses (ints) or objects with .ctypes.data / .data_ptr()."""
        self.lib.check(self.lib.lib.omni_b200_attention_bhld_host(
            self.handle, _addr(q), _addr(k), _addr(v), _addr(out), batch, heads, L, head_dim, dtype, out_dtype,
            _addr(lengths) if lengths is not None else None, block, int(bool(skip_padded_queries)), float(scale)))

    def vq_argmin(self, x, codebook, ids, rows, dim, codes, profile=BF16, ids_u16=True, cbnorm=None):
        self.lib.check(self.lib.lib.omni_b200_vq_argmin_host(
            self.handle, _addr(x), _addr(codebook), _addr(cbnorm) if cbnorm is not None else None, _addr(ids),
            rows, dim, codes, profile, int(bool(ids_u16))))


def _addr(obj):
    if isinstance(obj, int):
        return obj
    if hasattr(obj, "data_ptr"):
        return obj.data_ptr()
    return obj.ctypes.data


def gelu_(x, stream=None):
    """Ops::gelu in place on a contiguous fp32 or bf16 CUDA tensor."""
    lib = library()
    lib.check(lib.lib.omni_b200_gelu(x.data_ptr(), x.numel(), _dtype_code(x), _stream_ptr(stream)))
    return x


def attention_rows(q, k, v, heads, block=0, valid=None, fused=False, out_dtype=None, stream=None,
                   batch=1, lengths=None, workspace=True):
    """Ops::attention on the reference's row-major layout (CUDA tensors).

    batch > 1: `batch` sequences of q.shape[0] // batch rows each, keys of
    sequence b limited to lengths[b] (a CUDA int32 tensor) when given.
    workspace=False passes only the repacking bytes (no key split scratch)."""
    import torch

    if stream is not None:
        with _on("attention_rows", stream, q):
            return attention_rows(q, k, v, heads, block, valid, fused, out_dtype, None, batch, lengths, workspace)
    rows = q.shape[0]
    n = rows // batch
    d = q.shape[1] // 3 if fused else q.shape[1]
    hd = d // heads
    valid = n if valid is None else valid
    out = torch.empty((rows, d), dtype=out_dtype or q.dtype, device=q.device)
    lib = library()
    if batch == 1 and lengths is None:
        ws_bytes = lib.lib.omni_b200_attention_rows_workspace(n, heads, hd, _dtype_code(q), int(fused))
    else:
        ws_bytes = lib.lib.omni_b200_attention_rows_batch_workspace(n, batch, heads, hd, _dtype_code(q),
                                                                    int(fused))
    if not workspace:
        ws_bytes = 0
        if _dtype_code(q) == 0 or hd % 8 or (3 * d if fused else d) % 8:
            raise ValueError("workspace=False needs rows that are read in place")
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=q.device)
    if batch == 1 and lengths is None:
        lib.check(lib.lib.omni_b200_attention_rows(
            q.data_ptr(), None if fused else k.data_ptr(), None if fused else v.data_ptr(), out.data_ptr(), n,
            heads, hd, block, valid, int(fused), _dtype_code(q), _dtype_code(out), ws.data_ptr(), ws_bytes,
            _stream_ptr(stream)))
    else:
        lib.check(lib.lib.omni_b200_attention_rows_batch(
            q.data_ptr(), None if fused else k.data_ptr(), None if fused else v.data_ptr(), out.data_ptr(), n,
            batch, heads, hd, block, valid, None if lengths is None else lengths.data_ptr(), int(fused),
            _dtype_code(q), _dtype_code(out), ws.data_ptr(), ws_bytes, _stream_ptr(stream)))
    return out


# -------------------------------------------------------- 8-bit layer operators
# A call with one token is over in a few microseconds on the device, so these
# helpers keep the host's part short: every tensor attribute is read once, and the
# device's stream is looked up without building objects or importing per call.
# They work on the current stream of the tensors' device.  stream=s (a torch.cuda.Stream)
# is short for `with torch.cuda.stream(s):` (which a loop of small calls enters once, 8 us of
# the host's time less for each).  As there, the inputs have to be ready on s
# and kept (or recorded on s) until it is done with them, and the outputs are memory of
# s: another stream waits for s before it reads them, and records them when it may
# still read them after they are dropped.
class _Torch:
    """torch's names that the helpers use, looked up at their first call."""

    def __getattr__(self, name):
        import torch

        self.codes = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
        self.e4m3, self.f32, self.bf16, self.i32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.int32
        self.u8, self.f64, self.zeros, self.device = torch.uint8, torch.float64, torch.zeros, torch.device
        self.position_codes = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
        self.empty_like, self.cuda, self.current_device = torch.empty_like, torch.cuda, torch.cuda.current_device
        self.raw_stream = torch._C._cuda_getCurrentRawStream
        if name not in self.__dict__:
            raise AttributeError(name)
        return self.__dict__[name]


_t = _Torch()


def _refuse(message):
    raise NativeError(INVALID_ARGUMENT, message)


def _device_of(what, *tensors):
    """The CUDA device that every given tensor is on."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and (device < 0 or t.get_device() != device):
            _refuse(f"{what}: every tensor must be on the same CUDA device")
    return device


def _row_stride(what, t, shape):
    """Elements between the rows of a matrix with contiguous columns; a single row's
    stride does not matter."""
    if t.is_contiguous():
        return shape[1]
    rows, columns = t.stride()
    if columns != 1 and shape[1] > 1:
        _refuse(f"{what}: columns must be contiguous")
    return rows if shape[0] > 1 else shape[1]


def _call(name, device, stream, *args):
    """Calls an entry point on `device` and on `stream`, or that device's current one."""
    lib = _LIB or library()
    fn = getattr(lib.lib, name)
    s = _t.raw_stream(device) if stream is None else stream.cuda_stream
    if device == _t.current_device():
        status = fn(*args, s)
    else:
        with _t.cuda.device(device):
            status = fn(*args, s)
    if status:
        lib.check(status)


def _matrix(what, t):
    """(shape, type code) of a matrix of one of the element types."""
    code, shape = _t.codes.get(t.dtype), t.shape
    if code is None or len(shape) != 2:
        _refuse(f"{what}: need a [rows, cols] tensor of float32, bfloat16 or float16")
    return shape, code


def _empty_e4m3(x, rows, cols):
    """e4m3 [rows, cols] whose row stride is a multiple of 16, as linear_e4m3 reads it."""
    if cols % 16 == 0:
        if x.is_contiguous():
            return _t.empty_like(x, dtype=_t.e4m3), cols
        return x.new_empty((rows, cols), dtype=_t.e4m3), cols
    pitch = (cols + 15) // 16 * 16
    return x.new_empty((rows, pitch), dtype=_t.e4m3)[:, :cols], pitch


def _norm(what, x, shape, code, weight, residual, residual_out, out, out_stride, scales, eps, out_code,
          stream=None):
    rows, cols = shape
    dtype = x.dtype
    if weight.shape != (cols,) or weight.dtype != dtype or (cols > 1 and weight.stride(0) != 1):
        _refuse(f"{what}: weight must be contiguous [{cols}] of x's type")
    to_ptr = from_ptr = None
    to_stride = from_stride = 0
    if residual is None:
        if residual_out is not None:
            _refuse(f"{what}: residual_out needs a residual")
    else:
        if residual.shape != shape or residual.dtype != dtype:
            _refuse(f"{what}: residual must have x's shape and type")
        if residual_out is None:
            residual_out, to_stride = _t.empty_like(x) if x.is_contiguous() else x.new_empty(shape), cols
        elif residual_out.shape != shape or residual_out.dtype != dtype:
            _refuse(f"{what}: residual_out must have x's shape and type")
        else:
            to_stride = _row_stride(what, residual_out, shape)
        from_stride = _row_stride(what, residual, shape)
        from_ptr, to_ptr = residual.data_ptr(), residual_out.data_ptr()
    device = _device_of(what, x, weight, residual, residual_out, out)
    _call("omni_b200_rms_norm", device, stream, x.data_ptr(), from_ptr, weight.data_ptr(), to_ptr, out.data_ptr(),
          scales, rows, cols, _row_stride(what, x, shape), from_stride, to_stride, out_stride, eps, code, out_code)
    return residual_out


def rms_norm(x, weight, residual=None, eps=1e-6, out=None, residual_out=None, stream=None):
    """Root-mean-square norm of the rows of x [rows, cols] (+ residual).

    Returns (y, h): y = h / sqrt(mean(h^2) + eps) * weight in x's type, h = x + residual
    (None without a residual).  residual_out and out may each be x or residual, not both
    the same one.  stream=s is, here and below, the call inside torch.cuda.stream(s)."""
    if stream is not None and (out is None or (residual is not None and residual_out is None)):
        with _on("rms_norm", stream, x):
            return rms_norm(x, weight, residual, eps, out, residual_out)
    shape, code = _matrix("rms_norm", x)
    if out is None:
        out, out_stride = _t.empty_like(x) if x.is_contiguous() else x.new_empty(shape), shape[1]
    elif out.shape != shape or out.dtype != x.dtype:
        _refuse("rms_norm: out must have x's shape and type")
    else:
        out_stride = _row_stride("rms_norm", out, shape)
    return out, _norm("rms_norm", x, shape, code, weight, residual, residual_out, out, out_stride, None, eps, code,
                      stream)


def rms_norm_e4m3(x, weight, residual=None, eps=1e-6, residual_out=None, stream=None):
    """rms_norm with its output in e4m3 and an fp32 scale for each 128 columns.

    Returns (q, scales, h); q and scales are what linear_e4m3 takes."""
    if stream is not None:
        with _on("rms_norm_e4m3", stream, x):
            return rms_norm_e4m3(x, weight, residual, eps, residual_out)
    shape, code = _matrix("rms_norm_e4m3", x)
    rows, cols = shape
    q, pitch = _empty_e4m3(x, rows, cols)
    scales = x.new_empty((rows, (cols + 127) // 128), dtype=_t.f32)
    return q, scales, _norm("rms_norm_e4m3", x, shape, code, weight, residual, residual_out, q, pitch,
                            scales.data_ptr(), eps, E4M3)


def quantize_e4m3(x, block_rows=1, stream=None):
    """x [rows, cols] in e4m3: (q, scales), a scale for each 128 columns of a row
    (block_rows=1) or each 128 x 128 block (block_rows=128, weights)."""
    if stream is not None:
        with _on("quantize_e4m3", stream, x):
            return quantize_e4m3(x, block_rows)
    shape, code = _matrix("quantize_e4m3", x)
    if block_rows != 1 and block_rows != 128:
        _refuse("quantize_e4m3: block_rows must be 1 or 128")
    rows, cols = shape
    device = _device_of("quantize_e4m3", x)
    stride = _row_stride("quantize_e4m3", x, shape)
    q, pitch = _empty_e4m3(x, rows, cols)
    scales = x.new_empty(((rows + block_rows - 1) // block_rows, (cols + 127) // 128), dtype=_t.f32)
    _call("omni_b200_quantize_e4m3", device, None, x.data_ptr(), q.data_ptr(), scales.data_ptr(), rows, cols, stride,
          pitch, block_rows, code)
    return q, scales


def linear_e4m3(a, a_scales, w, w_scales, bias=None, out_dtype=None, out=None, stream=None):
    """a [m, k] times w [n, k] transposed, both e4m3 with scales (quantize_e4m3 with
    block_rows 1 and 128), plus bias [n]: [m, n] of out_dtype (bfloat16)."""
    if stream is not None and out is None:
        with _on("linear_e4m3", stream, a):
            return linear_e4m3(a, a_scales, w, w_scales, bias, out_dtype, out)
    shape, w_shape = a.shape, w.shape
    if len(shape) != 2 or len(w_shape) != 2 or a.dtype != _t.e4m3 or w.dtype != _t.e4m3 or w_shape[1] != shape[1]:
        _refuse("linear_e4m3: a [m, k] and w [n, k] must be float8_e4m3fn matrices")
    (m, k), n = shape, w_shape[0]
    groups = (k + 127) // 128
    if (a_scales.dtype != _t.f32 or w_scales.dtype != _t.f32 or a_scales.shape != (m, groups)
            or w_scales.shape != ((n + 127) // 128, groups) or not a_scales.is_contiguous()
            or not w_scales.is_contiguous()):
        _refuse(f"linear_e4m3: scales must be contiguous float32 [{m}, {groups}] and [{(n + 127) // 128}, {groups}]")
    if out is None:
        out = a.new_empty((m, n), dtype=_t.bf16 if out_dtype is None else out_dtype)
        stride = n
    elif out.shape != (m, n) or (out_dtype is not None and out.dtype != out_dtype):
        _refuse("linear_e4m3: out must be [m, n] of out_dtype")
    else:
        stride = _row_stride("linear_e4m3", out, (m, n))
    dtype = out.dtype
    code = _t.codes.get(dtype)
    if code is None:
        _refuse("linear_e4m3: the output must be float32, bfloat16 or float16")
    bias_ptr = None
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != dtype or (n > 1 and bias.stride(0) != 1):
            _refuse(f"linear_e4m3: bias must be contiguous [{n}] of the output's type")
        bias_ptr = bias.data_ptr()
    lda, ldw = _row_stride("linear_e4m3", a, shape), _row_stride("linear_e4m3", w, w_shape)
    # A single row counts as one padded to 16.
    if m == 1:
        lda = (k + 15) // 16 * 16
    if n == 1:
        ldw = (k + 15) // 16 * 16
    device = _device_of("linear_e4m3", a, a_scales, w, w_scales, bias, out)
    _call("omni_b200_linear_e4m3", device, stream, a.data_ptr(), a_scales.data_ptr(), w.data_ptr(),
          w_scales.data_ptr(), bias_ptr, out.data_ptr(), m, n, k, lda, ldw, stride, code)
    return out


_STRIDES = C.c_int64 * 12
_INT = 1 << 31


def attention_window(q, k, v, window=0, sinks=0, right=0, lengths=None, q_lengths=None, scale=0.0, out=None,
                     out_dtype=None, stream=None):
    """Sliding-window attention: q [B, H, Lq, D] over k, v [B, Hkv, Lk, D] (any strides
    with contiguous columns), bfloat16 or float16.

    Sequence b holds lengths[b] keys (None: Lk) and q_lengths[b] queries (None: Lq), its
    last ones (CUDA int32 tensors).  The query at position p sees `window` keys up to its
    own (window <= 0: all), the first `sinks` keys, and `right` keys past it.  Rows past a
    sequence's queries are left as they are in `out`, undefined in a new one.  `out` must not
    overlap q, k or v; Lk is at least 1 (an empty cache: lengths of 0)."""
    if stream is not None and out is None:
        with _on("attention_window", stream, q):
            return attention_window(q, k, v, window, sinks, right, lengths, q_lengths, scale, out, out_dtype)
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or v.shape != k_shape:
        _refuse("attention_window: q must be [B, H, Lq, D], k and v [B, Hkv, Lk, D]")
    B, H, Lq, D = q_shape
    Bk, Hkv, Lk, Dk = k_shape
    if Bk != B or Dk != D:
        _refuse("attention_window: q, k and v must agree in batch and head dimension")
    # The entry point takes 32-bit sizes and refuses the rest of what is out of range.
    if not (-_INT < window < _INT and -_INT < right < _INT and -_INT < sinks < _INT
            and max(B, H, Hkv, Lq, Lk, D) < _INT):
        _refuse("attention_window: sizes, window, right and sinks must be below 2^31")
    dtype = q.dtype
    code = _t.codes.get(dtype, F32)
    if code == F32 or k.dtype != dtype or v.dtype != dtype:
        _refuse("attention_window: q, k and v must all be bfloat16, or all float16")
    pointers = [None, None]
    for i, n in enumerate((lengths, q_lengths)):
        if n is not None:
            if n.shape != (B,) or n.dtype != _t.i32 or not n.is_contiguous():
                _refuse("attention_window: lengths and q_lengths must be contiguous int32 [B]")
            pointers[i] = n.data_ptr()
    out_code = code
    if out is None:
        out = q.new_empty(q_shape, dtype=dtype if out_dtype is None else out_dtype)
    elif out.shape != q_shape or (out_dtype is not None and out.dtype != out_dtype):
        _refuse("attention_window: out must have q's shape and out_dtype")
    if out.dtype != dtype:
        if out.dtype != _t.f32:
            _refuse("attention_window: the output's type must be q's, or float32")
        out_code = F32
    device = _device_of("attention_window", q, k, v, lengths, q_lengths, out)
    qb, qh, qt, qd = q.stride()
    kb, kh, kt, kd = k.stride()
    vb, vh, vt, vd = v.stride()
    ob, oh, ot, od = out.stride()
    if qd != 1 or kd != 1 or vd != 1 or od != 1:
        _refuse("attention_window: columns must be contiguous")
    _call("omni_b200_attention_window", device, stream, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H,
          Hkv, Lq, Lk, D, _STRIDES(qb, qh, qt, kb, kh, kt, vb, vh, vt, ob, oh, ot), *pointers, window, right, sinks,
          scale, code, out_code)
    return out


# ------------------------------------- rotary positions and the 4-bit key/value cache
def rotary_axes(sections, interleaved=False):
    """The axis of each pair for rotary(): sections[a] pairs of axis a, one run after the
    other, or dealt out in turn (0, 1, 2, 0, 1, 2, ...) until an axis has none left."""
    left = [int(n) for n in sections]
    if not left or len(left) > 256 or min(left) < 0 or sum(left) == 0:
        _refuse("rotary_axes: need the pairs of each axis")
    if not interleaved:
        return bytes(a for a, n in enumerate(left) for _ in range(n))
    axes = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                axes.append(a)
                left[a] -= 1
    return bytes(axes)


def rotary(q, k, positions, frequencies, axes=None, adjacent=False, inverse=False, q_out=None, k_out=None,
           stream=None):
    """q [B, H, T, D] and k [B, Hkv, T, D] (or None) with rotary positions: (q_out, k_out).

    positions is [axes, B, T], or [B, T] for one axis, int32, int64 or float32 (any strides, 0
    among them); frequencies [pairs], float32 or float64, 2 * pairs <= D.  Pair i is columns
    (i, i + pairs), or (2i, 2i + 1) with adjacent, and turns by positions[axes[i]] *
    frequencies[i]; axes is bytes or a list of numbers (rotary_axes), None: axis 0.  The other
    columns are copied.  inverse turns back: the gradients of q and k are those of q_out
    and k_out with inverse.  q_out and k_out may be q and k."""
    if stream is not None and (q_out is None or (k is not None and k_out is None)):
        with _on("rotary", stream, q):
            return rotary(q, k, positions, frequencies, axes, adjacent, inverse, q_out, k_out)
    shape, dtype = q.shape, q.dtype
    code = _t.codes.get(dtype)
    if code is None or len(shape) != 4:
        _refuse("rotary: q must be [B, H, T, D] of float32, bfloat16 or float16")
    B, H, T, D = shape
    Hkv, k_ptr, k_to = 0, None, None
    if q_out is None:
        q_out = _t.empty_like(q)  # laid out as q is, where q's memory has no gaps
    elif q_out.shape != shape or q_out.dtype != dtype:
        _refuse("rotary: q_out must have q's shape and type")
    qb, qh, qt, qd = q.stride()
    ob, oh, ot, od = q_out.stride()
    ends = qd != 1 or od != 1
    if k is not None:
        Hkv = k.shape[1] if len(k.shape) == 4 else 0
        if k.shape != (B, Hkv, T, D) or Hkv == 0 or k.dtype != dtype:
            _refuse("rotary: k must be [B, Hkv, T, D] of q's type")
        if k_out is None:
            k_out = _t.empty_like(k)
        elif k_out.shape != k.shape or k_out.dtype != dtype:
            _refuse("rotary: k_out must have k's shape and type")
        kb, kh, kt, kd = k.stride()
        lb, lh, lt, ld = k_out.stride()
        ends = ends or kd != 1 or ld != 1
        strides = _STRIDES(qb, qh, qt, ob, oh, ot, kb, kh, kt, lb, lh, lt)
        k_ptr, k_to = k.data_ptr(), k_out.data_ptr()
    else:
        if k_out is not None:
            _refuse("rotary: k_out needs a k")
        strides = _STRIDES(qb, qh, qt, ob, oh, ot)
    if ends and D > 1:
        _refuse("rotary: columns must be contiguous")
    p_shape, p_code = positions.shape, _t.position_codes.get(positions.dtype)
    if p_code is None or (p_shape[1:] if len(p_shape) == 3 else p_shape) != (B, T):
        _refuse("rotary: positions must be [axes, B, T] or [B, T] of int32, int64 or float32")
    A = p_shape[0] if len(p_shape) == 3 else 1
    if len(frequencies.shape) != 1 or frequencies.dtype not in (_t.f32, _t.f64) or not frequencies.is_contiguous():
        _refuse("rotary: frequencies must be contiguous [pairs], float32 or float64")
    pairs = frequencies.shape[0]
    if axes is not None:
        axes = bytes(axes)
        if len(axes) != pairs:
            _refuse("rotary: axes must name an axis for each pair")
    if max(B, H, Hkv, T, D, pairs, A) >= _INT:
        _refuse("rotary: sizes must be below 2^31")
    device = _device_of("rotary", q, k, positions, frequencies, q_out, k_out)
    p_strides = positions.stride()
    _call("omni_b200_rotary", device, stream, q.data_ptr(), q_out.data_ptr(), k_ptr, k_to, positions.data_ptr(),
          frequencies.data_ptr(), axes, B, H, Hkv, T, D, pairs, A, strides,
          _THREE(*p_strides) if len(p_strides) == 3 else _THREE(0, *p_strides), int(adjacent), int(inverse), p_code,
          int(frequencies.dtype == _t.f64), code)
    return q_out, k_out


_THREE, _SIX = C.c_int64 * 3, C.c_int64 * 6


class _CacheE2m1(C.Structure):
    _fields_ = [("data", C.c_void_p), ("table", C.c_void_p), ("pages", C.c_int32), ("page_tokens", C.c_int32),
                ("table_width", C.c_int32), ("page_stride", C.c_int64), ("head_stride", C.c_int64)]


def empty_cache_e2m1(pages, kv_heads, page_tokens, head_dim, device="cuda", stream=None):
    """A cache of keys and values in 4 bits, uint8 [pages, kv_heads, bytes of a page], all
    zeros.  A page holds page_tokens tokens (a multiple of 16) of one key head; head_dim is a
    multiple of 8 up to 128."""
    if stream is not None and (place := _t.device(device)).type == "cuda":
        if place.index is None:  # the stream's, or the current one where it does not say
            place = _t.device("cuda", stream.device_index if hasattr(stream, "device_index") else _t.current_device())
        with _on("empty_cache_e2m1", stream, place.index):
            return empty_cache_e2m1(pages, kv_heads, page_tokens, head_dim, place)
    in_range = 0 <= page_tokens < _INT and 0 <= head_dim < _INT
    size = library().lib.omni_b200_cache_e2m1_bytes(page_tokens, head_dim) if in_range else 0
    if size == 0 or pages <= 0 or kv_heads <= 0:
        _refuse("empty_cache_e2m1: page_tokens must be a multiple of 16 up to 2^30, head_dim a multiple of 8 up to 128")
    return _t.zeros((pages, kv_heads, size), dtype=_t.u8, device=device)


def _cache(what, cache, head_dim, batch, table, lengths, q_lengths):
    """(the entry points' description of a cache, kv_heads, what a sequence's pages hold,
    pointers of lengths and q_lengths)."""
    shape = cache.shape
    if len(shape) != 3 or cache.dtype != _t.u8:
        _refuse(f"{what}: the cache must be uint8 [pages, kv_heads, bytes]")
    pages, kv_heads, size = shape
    block = (head_dim + 31) // 32 * 576
    if head_dim <= 0 or head_dim > 128 or head_dim % 8 or size == 0 or size % block:
        _refuse(f"{what}: a page of {size} bytes is none of head_dim {head_dim} (a multiple of 8 up to 128)")
    page_stride, head_stride, last = cache.stride()
    if last != 1:
        _refuse(f"{what}: the bytes of a page must be contiguous")
    tokens, width, table_ptr = size // block * 16, 1, None
    if table is not None:
        if len(table.shape) != 2 or table.shape[0] != batch or table.dtype != _t.i32 or not table.is_contiguous():
            _refuse(f"{what}: table must be contiguous int32 [B, pages of a sequence]")
        width, table_ptr = table.shape[1], table.data_ptr()
    if max(pages, kv_heads, tokens, width) >= _INT:
        _refuse(f"{what}: sizes must be below 2^31")
    pointers = [None, None]
    for i, n in enumerate((lengths, q_lengths)):
        if n is not None:
            if n.shape != (batch,) or n.dtype != _t.i32 or not n.is_contiguous():
                _refuse(f"{what}: lengths and q_lengths must be contiguous int32 [B]")
            pointers[i] = n.data_ptr()
    return (_CacheE2m1(cache.data_ptr(), table_ptr, pages, tokens, width, page_stride, head_stride), kv_heads,
            tokens * width, pointers)


def _pair_strides(what, a, b):
    ab, ah, at, ad = a.stride()
    bb, bh, bt, bd = b.stride()
    if (ad != 1 or bd != 1) and a.shape[3] > 1:
        _refuse(f"{what}: columns must be contiguous")
    return _SIX(ab, ah, at, bb, bh, bt)


def cache_write_e2m1(k, v, cache, lengths, q_lengths=None, table=None, stream=None):
    """Quantises k and v [B, Hkv, T, D] (bfloat16 or float16, any strides that are multiples of
    8 with contiguous columns) into the cache (empty_cache_e2m1), which it returns.

    Sequence b holds lengths[b] tokens when the call is over; k and v are its last
    q_lengths[b] of them (None: T), from row 0 on.  table [B, pages of a sequence] names the
    pages (None: page b is sequence b); those that are written to stand in it once, and in no
    other call's that may run at the same time.  lengths, q_lengths and table are CUDA int32
    tensors."""
    shape, dtype = k.shape, k.dtype
    code = _t.codes.get(dtype, F32)
    if code == F32 or len(shape) != 4 or v.shape != shape or v.dtype != dtype:
        _refuse("cache_write_e2m1: k and v must be [B, Hkv, T, D], both bfloat16 or both float16")
    B, Hkv, T, D = shape
    what, heads, _, pointers = _cache("cache_write_e2m1", cache, D, B, table, lengths, q_lengths)
    if heads != Hkv or max(B, T) >= _INT:
        _refuse("cache_write_e2m1: k, v and the cache must have the same key heads")
    device = _device_of("cache_write_e2m1", k, v, cache, lengths, q_lengths, table)
    _call("omni_b200_cache_write_e2m1", device, stream, k.data_ptr(), v.data_ptr(), C.byref(what), *pointers, B, Hkv,
          T, D, _pair_strides("cache_write_e2m1", k, v), code)
    return cache


def cache_read_e2m1(cache, head_dim, lengths, rows=None, q_lengths=None, table=None, dtype=None, out=None,
                    stream=None):
    """What the cache stands for: (k, v), the last q_lengths[b] tokens of each sequence (None:
    all rows) from row 0 on.

    out is a pair of tensors [B, Hkv, rows, D] of float32, bfloat16 or float16; without it they
    are made, of dtype (bfloat16) and with `rows` rows (None: as many tokens as a sequence's
    pages hold).  Rows past q_lengths[b] or before a sequence's start stay as they are,
    undefined in new tensors."""
    if stream is not None and out is None:
        with _on("cache_read_e2m1", stream, cache):
            return cache_read_e2m1(cache, head_dim, lengths, rows, q_lengths, table, dtype)
    B = lengths.shape[0] if len(lengths.shape) == 1 else -1
    what, Hkv, capacity, pointers = _cache("cache_read_e2m1", cache, head_dim, B, table, lengths, q_lengths)
    if out is None:
        shape = (B, Hkv, capacity if rows is None else rows, head_dim)
        k, v = (cache.new_empty(shape, dtype=_t.bf16 if dtype is None else dtype) for _ in range(2))
    else:
        k, v = out
        shape = k.shape
        if len(shape) != 4 or shape[0] != B or shape[1] != Hkv or shape[3] != head_dim or v.shape != shape or (
                rows is not None and rows != shape[2]):
            _refuse("cache_read_e2m1: out must be two tensors [B, Hkv, rows, D]")
    code = _t.codes.get(k.dtype)
    if code is None or v.dtype != k.dtype or (dtype is not None and k.dtype != dtype):
        _refuse("cache_read_e2m1: k and v must both be float32, bfloat16 or float16, of dtype")
    if max(B, shape[2]) >= _INT:
        _refuse("cache_read_e2m1: sizes must be below 2^31")
    device = _device_of("cache_read_e2m1", cache, lengths, q_lengths, table, k, v)
    _call("omni_b200_cache_read_e2m1", device, stream, C.byref(what), k.data_ptr(), v.data_ptr(), *pointers, B, Hkv,
          shape[2], head_dim, _pair_strides("cache_read_e2m1", k, v), code)
    return k, v


@functools.lru_cache(maxsize=4096)
def _window_workspace(*sizes):
    """Asked once for the sizes of a call: the question costs as much as a tensor."""
    return library().lib.omni_b200_attention_window_e2m1_workspace(*sizes)


def attention_window_e2m1(q, cache, lengths, q_lengths=None, table=None, window=0, sinks=0, right=0, scale=0.0,
                          kv_len=None, out=None, out_dtype=None, stream=None):
    """attention_window over a cache in 4 bits: q [B, H, T, D] (bfloat16 or float16, strides
    that are multiples of 8), the last q_lengths[b] tokens (None: T) of the lengths[b] that
    sequence b holds, the cache as cache_write_e2m1 left it.

    kv_len is the most tokens that a sequence holds (None: as many as its pages do): what
    work is planned for, and for prompts how large a workspace is (bytes 4 B Hkv kv_len D).
    Rows past a sequence's queries are left as they are in `out`, undefined in a new one."""
    shape, dtype = q.shape, q.dtype
    code = _t.codes.get(dtype, F32)
    if code == F32 or len(shape) != 4:
        _refuse("attention_window_e2m1: q must be [B, H, T, D], bfloat16 or float16")
    B, H, T, D = shape
    what, Hkv, capacity, pointers = _cache("attention_window_e2m1", cache, D, B, table, lengths, q_lengths)
    if kv_len is None:
        kv_len = capacity
    if not (-_INT < window < _INT and -_INT < right < _INT and -_INT < sinks < _INT and 0 <= kv_len < _INT
            and max(B, H, T) < _INT):
        _refuse("attention_window_e2m1: sizes, window, right and sinks must be below 2^31")
    size = _window_workspace(B, H, Hkv, T, kv_len, D, window, right, sinks)
    if stream is not None and (out is None or size):
        with _on("attention_window_e2m1", stream, q):
            return attention_window_e2m1(q, cache, lengths, q_lengths, table, window, sinks, right, scale, kv_len, out,
                                         out_dtype)
    out_code = code
    if out is None:
        out = q.new_empty(shape, dtype=dtype if out_dtype is None else out_dtype)
    elif out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
        _refuse("attention_window_e2m1: out must have q's shape and out_dtype")
    if out.dtype != dtype:
        if out.dtype != _t.f32:
            _refuse("attention_window_e2m1: the output's type must be q's, or float32")
        out_code = F32
    device = _device_of("attention_window_e2m1", q, cache, lengths, q_lengths, table, out)
    workspace = q.new_empty(size, dtype=_t.u8) if size else None
    _call("omni_b200_attention_window_e2m1", device, stream, q.data_ptr(), C.byref(what), out.data_ptr(), *pointers, B,
          H, Hkv, T, kv_len, D, _pair_strides("attention_window_e2m1", q, out), window, right, sinks, scale, code,
          out_code, workspace.data_ptr() if size else None, size)
    return out
