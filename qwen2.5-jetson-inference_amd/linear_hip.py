"""Python binding of the MI355X Linear hot path (``libinfer_linear.so``).

The functions mirror the reference's operator boundary,
``include/infer/cuda_ops.hpp`` (Greedy-cy/qwen2.5-jetson-inference):
same names, same argument order and meaning, raw device pointers plus a
stream.  Each argument may be a device pointer (``int``) or a contiguous
``torch`` CUDA tensor; ``None`` is a null pointer.  A nonzero status from
the C ABI raises :class:`InferError` (the reference throws ``infer::Error``,
``include/infer/common.hpp:66-82``).

There is no fallback: if the library is missing, :func:`load` raises.
"""
from __future__ import annotations

import ctypes
import functools
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
# INFER_HIP_LIBRARY names another build of the same library (the host-only
# sanitizer build the CPU tests load); by default the in-tree build.
LIB_PATH = os.environ.get("INFER_HIP_LIBRARY") or os.path.join(_HERE, "libinfer_linear.so")

OK = 0
INVALID_ARGUMENT = 1
LAUNCH_FAILED = 2
RUNTIME_ERROR = 3

# Every symbol include/infer_linear.h declares.
EXPORTED_SYMBOLS = (
    "infer_hip_last_error",
    "infer_hip_abi_version",
    "infer_hip_gemv_bf16",
    "infer_hip_gemm_bf16",
    "infer_hip_lm_head_bf16",
    "infer_hip_lm_head_bf16_noalloc",
    "infer_hip_lm_head_workspace_entries",
    "infer_hip_gemv_w8a16",
    "infer_hip_gemm_w8a16",
    "infer_hip_w4a16_weight_bytes",
    "infer_hip_w4a16_scale_count",
    "infer_hip_w4a16_pack",
    "infer_hip_gemv_w4a16",
    "infer_hip_gemm_tile_count",
    "infer_hip_gemm_w8a16_tile",
    "infer_hip_gemm_bf16_tile",
    "infer_hip_gemm_workspace_bytes",
    "infer_hip_gemm_w8a16_ws",
    "infer_hip_gemm_bf16_ws",
    "infer_hip_w8a16_gemv_plan_create",
    "infer_hip_w8a16_gemv_plan_launch",
    "infer_hip_w8a16_gemv_plan_bytes",
    "infer_hip_w8a16_gemv_plan_destroy",
    "infer_hip_gemm_plan_create",
    "infer_hip_gemm_plan_launch",
    "infer_hip_gemm_plan_flops",
    "infer_hip_gemm_plan_destroy",
    "infer_hip_gemm_plan_timeline",
)


class W8A16GemvDesc(ctypes.Structure):
    """infer_hip_w8a16_gemv_desc: the arguments of one gemv_w8a16 call."""
    _fields_ = [
        ("weight", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("group_size", ctypes.c_int),
        ("bias", ctypes.c_void_p),
        ("input", ctypes.c_void_p),
        ("output", ctypes.c_void_p),
        ("out_features", ctypes.c_int),
        ("in_features", ctypes.c_int),
    ]


class GemmDesc(ctypes.Structure):
    """infer_hip_gemm_desc: the arguments of one gemm_w8a16 / gemm_bf16 call."""
    _fields_ = [
        ("w8a16", ctypes.c_int),
        ("weight", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("group_size", ctypes.c_int),
        ("bias", ctypes.c_void_p),
        ("input", ctypes.c_void_p),
        ("output", ctypes.c_void_p),
        ("tokens", ctypes.c_int),
        ("out_features", ctypes.c_int),
        ("in_features", ctypes.c_int),
    ]


class InferError(RuntimeError):
    """A nonzero status from the C ABI, with the library's message."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


_lib = None


def _hip_runtimes_mapped():
    try:
        with open("/proc/self/maps") as f:
            return sorted({line.split()[-1] for line in f
                           if "libamdhip64" in line and "/" in line})
    except OSError:
        return []


def load() -> ctypes.CDLL:
    """Load the HIP library (raises if it has not been built).

    torch (when installed) is imported first: its wheel ships its own HIP
    runtime, whose soname (libamdhip64.so.7) the library's dependency then
    resolves to, so the process holds one HIP runtime.  Two runtimes in one
    process cannot share the GPU; that case raises instead of running."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise InferError(RUNTIME_ERROR,
                         f"{LIB_PATH} is missing: run __graft_entry__.build()")
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(LIB_PATH)
    runtimes = _hip_runtimes_mapped()
    if len(runtimes) > 1:
        raise InferError(RUNTIME_ERROR,
                         "two HIP runtimes are loaded in this process: " + ", ".join(runtimes))
    p, i = ctypes.c_void_p, ctypes.c_int
    lib.infer_hip_last_error.restype = ctypes.c_char_p
    lib.infer_hip_abi_version.restype = i
    sigs = {
        "infer_hip_gemv_bf16": [p, p, p, p, i, i, p],
        "infer_hip_gemm_bf16": [p, p, p, p, i, i, i, p],
        "infer_hip_lm_head_bf16": [p, p, p, p, p, p, p, i, i, p],
        "infer_hip_lm_head_bf16_noalloc": [p, p, p, p, p, i, i, p],
        "infer_hip_gemv_w8a16": [p, p, i, p, p, p, i, i, p],
        "infer_hip_gemm_w8a16": [p, p, i, p, p, p, i, i, i, p],
        "infer_hip_gemv_w4a16": [p, p, i, p, p, p, i, i, i, p],
        "infer_hip_w4a16_pack": [p, p, i, i, i, p, p],
        "infer_hip_gemm_w8a16_tile": [p, p, i, p, p, p, i, i, i, i, p],
        "infer_hip_gemm_bf16_tile": [p, p, p, p, i, i, i, i, p],
        "infer_hip_gemm_w8a16_ws": [p, p, i, p, p, p, i, i, i, p, ctypes.c_size_t, p],
        "infer_hip_gemm_bf16_ws": [p, p, p, p, i, i, i, p, ctypes.c_size_t, p],
    }
    for name, args in sigs.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = i
    lib.infer_hip_w4a16_weight_bytes.argtypes = [i, i]
    lib.infer_hip_w4a16_weight_bytes.restype = ctypes.c_size_t
    lib.infer_hip_w4a16_scale_count.argtypes = [i, i, i]
    lib.infer_hip_w4a16_scale_count.restype = ctypes.c_size_t
    lib.infer_hip_gemm_tile_count.argtypes = []
    lib.infer_hip_gemm_tile_count.restype = i
    lib.infer_hip_gemm_workspace_bytes.argtypes = [i, i, i]
    lib.infer_hip_gemm_workspace_bytes.restype = ctypes.c_size_t
    lib.infer_hip_lm_head_workspace_entries.argtypes = [i, i]
    lib.infer_hip_lm_head_workspace_entries.restype = ctypes.c_size_t
    lib.infer_hip_w8a16_gemv_plan_create.argtypes = [p, i, ctypes.POINTER(p)]
    lib.infer_hip_w8a16_gemv_plan_create.restype = i
    lib.infer_hip_w8a16_gemv_plan_launch.argtypes = [p, p]
    lib.infer_hip_w8a16_gemv_plan_launch.restype = i
    lib.infer_hip_w8a16_gemv_plan_bytes.argtypes = [p]
    lib.infer_hip_w8a16_gemv_plan_bytes.restype = ctypes.c_double
    lib.infer_hip_w8a16_gemv_plan_destroy.argtypes = [p]
    lib.infer_hip_w8a16_gemv_plan_destroy.restype = i
    lib.infer_hip_gemm_plan_create.argtypes = [p, i, ctypes.POINTER(p)]
    lib.infer_hip_gemm_plan_create.restype = i
    lib.infer_hip_gemm_plan_launch.argtypes = [p, p]
    lib.infer_hip_gemm_plan_launch.restype = i
    lib.infer_hip_gemm_plan_flops.argtypes = [p]
    lib.infer_hip_gemm_plan_flops.restype = ctypes.c_double
    lib.infer_hip_gemm_plan_destroy.argtypes = [p]
    lib.infer_hip_gemm_plan_destroy.restype = i
    lib.infer_hip_gemm_plan_timeline.argtypes = [p, p, i, ctypes.POINTER(i), p]
    lib.infer_hip_gemm_plan_timeline.restype = i
    _lib = lib
    return lib


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise InferError(INVALID_ARGUMENT, "tensor must live on the GPU")
    if not t.is_contiguous():
        raise InferError(INVALID_ARGUMENT, "tensor must be contiguous")
    return t.data_ptr()


# torch's handle of a device's current stream and the current device, without the
# Stream object that torch.cuda.current_stream() makes (0.2 us against 2.8); None
# until its HIP state exists, or if it has no such functions.
_raw_stream = _raw_device = None


def _current_device():
    """The current GPU's index; without one, an index that no tensor has."""
    import torch
    return torch.cuda.current_device() if torch.cuda.is_available() else -2


def _stream(stream):
    global _raw_stream, _raw_device
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(_raw_device())
        import torch
        current = torch.cuda.current_stream().cuda_stream
        _raw_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return current
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _check(status: int) -> None:
    if status != OK:
        msg = load().infer_hip_last_error().decode("utf-8", "replace")
        raise InferError(status, msg)


def gemv_bf16(weight, bias, input, output, out_features, in_features,
              stream=None):
    """cuda_ops.hpp:24-26."""
    _check(load().infer_hip_gemv_bf16(_ptr(weight), _ptr(bias), _ptr(input),
                                      _ptr(output), out_features, in_features,
                                      _stream(stream)))


def gemm_bf16(weight, bias, input, output, tokens, out_features, in_features,
              stream=None):
    """cuda_ops.hpp:32-35."""
    _check(load().infer_hip_gemm_bf16(_ptr(weight), _ptr(bias), _ptr(input),
                                      _ptr(output), tokens, out_features,
                                      in_features, _stream(stream)))


def lm_head_workspace_entries(vocab: int, in_features: int) -> int:
    return int(load().infer_hip_lm_head_workspace_entries(vocab, in_features))


def lm_head_bf16(weight, bias, input, logits, block_max_value,
                 block_max_index, argmax, vocab, in_features, stream=None):
    """cuda_ops.hpp:42-45 (argmax over FP32 sums, ties to the lowest index)."""
    _check(load().infer_hip_lm_head_bf16(
        _ptr(weight), _ptr(bias), _ptr(input), _ptr(logits),
        _ptr(block_max_value), _ptr(block_max_index), _ptr(argmax), vocab,
        in_features, _stream(stream)))


def lm_head_bf16_noalloc(weight, bias, input, logits, argmax, vocab, in_features,
                         stream=None):
    """lm_head_bf16 with the library's static device scratch instead of a
    workspace (infer_hip_lm_head_bf16_noalloc; vocab <= 1048576)."""
    _check(load().infer_hip_lm_head_bf16_noalloc(
        _ptr(weight), _ptr(bias), _ptr(input), _ptr(logits), _ptr(argmax), vocab,
        in_features, _stream(stream)))


def gemv_w8a16(weight, scales, group_size, bias, input, output, out_features,
               in_features, stream=None):
    """cuda_ops.hpp:47-50."""
    _check(load().infer_hip_gemv_w8a16(_ptr(weight), _ptr(scales), group_size,
                                       _ptr(bias), _ptr(input), _ptr(output),
                                       out_features, in_features,
                                       _stream(stream)))


def gemm_w8a16(weight, scales, group_size, bias, input, output, tokens,
               out_features, in_features, stream=None):
    """cuda_ops.hpp:51-55."""
    _check(load().infer_hip_gemm_w8a16(_ptr(weight), _ptr(scales), group_size,
                                       _ptr(bias), _ptr(input), _ptr(output),
                                       tokens, out_features, in_features,
                                       _stream(stream)))


def quantize_w4a16(weight, group_size: int = 64):
    """FP32 weights [N, K] (numpy) -> (int8 values in [-7, 7], BF16 scale words
    [N, K / group_size]) as the W8A16 exporter quantises: s = max|w| / 7 of a
    row's group in FP32 (0 -> 1), values rint(w / s), s stored as BF16."""
    import numpy as np

    import synthetic
    w = np.ascontiguousarray(weight, dtype=np.float32)
    if w.ndim != 2 or group_size not in (32, 64, 128) or w.shape[1] % group_size or not w.size:
        raise InferError(INVALID_ARGUMENT,
                         f"quantize_w4a16: {w.shape} in groups of {group_size} (32, 64 or 128, "
                         "dividing K)")
    if not np.isfinite(w).all():
        raise InferError(INVALID_ARGUMENT, "quantize_w4a16: weights must be finite")
    blocks = w.reshape(w.shape[0], -1, group_size)
    s = (np.abs(blocks).max(axis=2) / np.float32(7)).astype(np.float32)
    s = np.where(s == 0, np.float32(1), s)
    q = np.clip(np.rint(blocks / s[:, :, None]), -7, 7).astype(np.int8).reshape(w.shape)
    return q, synthetic.float32_to_bf16_bits(s)


def pack_w4a16(values, scales, group_size: int):
    """Row-major int8 values in [-8, 7] [N, K] and BF16 scale words
    [N, K / group_size] (numpy) -> the packed (weight bytes, scale words) that
    gemv_w4a16 takes (infer_hip_w4a16_pack; host only)."""
    import numpy as np
    values = np.ascontiguousarray(values)
    scales = np.ascontiguousarray(scales)
    if values.dtype != np.int8 or values.ndim != 2 or scales.dtype != np.uint16:
        raise InferError(INVALID_ARGUMENT, "pack_w4a16: int8 values [N, K] and uint16 scale words")
    n, k = values.shape
    lib = load()
    count = lib.infer_hip_w4a16_scale_count(n, k, group_size)
    if count == 0 or scales.shape != (n, k // group_size):
        raise InferError(INVALID_ARGUMENT,
                         f"pack_w4a16: values {values.shape}, scales {scales.shape}, group "
                         f"{group_size} (32, 64 or 128, dividing K)")
    packed = np.empty(lib.infer_hip_w4a16_weight_bytes(n, k), np.uint8)
    tiled = np.empty(count, np.uint16)
    _check(lib.infer_hip_w4a16_pack(values.ctypes.data, scales.ctypes.data, group_size, n, k,
                                    packed.ctypes.data, tiled.ctypes.data))
    return packed, tiled


@functools.lru_cache(maxsize=1024)
def _w4a16_bytes(group_size, tokens, n, k):
    """Bytes of weight, scales, bias, input and output (0: a shape that the C ABI
    refuses)."""
    lib = load()
    tiled = 2 * lib.infer_hip_w4a16_scale_count(n, k, group_size)
    if tiled == 0 or tokens < 1:
        return 0, 0, 0, 0, 0
    return lib.infer_hip_w4a16_weight_bytes(n, k), tiled, 2 * n, 2 * tokens * k, 2 * tokens * n


def _w4a16_ptr(t, types, least, device, name):
    """Pointer of a contiguous tensor of at least `least` bytes on the current GPU;
    addresses are taken as they are."""
    if t is None or type(t) is int:
        return t
    if t.nbytes >= least and t.dtype in types and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    if t.nbytes < least or t.dtype not in types:
        raise InferError(INVALID_ARGUMENT,
                         f"gemv_w4a16: {name} of {t.nbytes} bytes of {t.dtype}: {least} bytes of "
                         f"{' or '.join(str(x) for x in types)} needed")
    if t.is_cuda and t.get_device() != device:
        raise InferError(INVALID_ARGUMENT, f"gemv_w4a16: {name} is not on the current GPU")
    return _ptr(t)


_words = _bytes = None  # types of 16-bit words and of bytes


def gemv_w4a16(weight, scales, group_size, bias, input, output, tokens, out_features,
               in_features, stream=None):
    """1 to 16 tokens by packed 4-bit weights (infer_hip_gemv_w4a16).  weight is uint8
    and scales BF16 (or words) as pack_w4a16 lays them out, the rest BF16 (or words);
    buffers may be longer than the shape needs."""
    global _words, _bytes
    if _words is None:
        import torch
        _bytes = torch.uint8, torch.int8
        _words = torch.bfloat16, torch.int16, torch.uint16
    w, s, b, x, y = _w4a16_bytes(group_size, tokens, out_features, in_features)
    device = _current_device() if _raw_device is None else _raw_device()
    status = (_lib or load()).infer_hip_gemv_w4a16(
        _w4a16_ptr(weight, _bytes, w, device, "weight"),
        _w4a16_ptr(scales, _words, s, device, "scales"), group_size,
        _w4a16_ptr(bias, _words, b, device, "bias"), _w4a16_ptr(input, _words, x, device, "input"),
        _w4a16_ptr(output, _words, y, device, "output"), tokens, out_features, in_features,
        _stream(stream) if stream is not None or _raw_stream is None else _raw_stream(device))
    if status:
        _check(status)


# MFMA workgroup tiles (rows x columns of Y) of the explicit-tile entries.
GEMM_TILES = ("128x128", "128x64", "64x128", "64x64", "32x128", "256x128")


def gemm_tile_count() -> int:
    return int(load().infer_hip_gemm_tile_count())


def gemm_w8a16_tile(weight, scales, group_size, bias, input, output, tokens,
                    out_features, in_features, tile, stream=None):
    """gemm_w8a16 with the MFMA workgroup tile named (-1 = automatic)."""
    _check(load().infer_hip_gemm_w8a16_tile(_ptr(weight), _ptr(scales), group_size,
                                            _ptr(bias), _ptr(input), _ptr(output),
                                            tokens, out_features, in_features, tile,
                                            _stream(stream)))


def gemm_bf16_tile(weight, bias, input, output, tokens, out_features,
                   in_features, tile, stream=None):
    """gemm_bf16 with the MFMA workgroup tile named (-1 = automatic)."""
    _check(load().infer_hip_gemm_bf16_tile(_ptr(weight), _ptr(bias), _ptr(input),
                                           _ptr(output), tokens, out_features,
                                           in_features, tile, _stream(stream)))


def gemm_workspace_bytes(max_tokens, out_features, in_features) -> int:
    """Workspace bytes of gemm_*_ws for every token count up to max_tokens
    (0: no such call needs or uses one); the largest of several Linears'
    serves them all."""
    return int(load().infer_hip_gemm_workspace_bytes(max_tokens, out_features, in_features))


def _ws_args(workspace):
    """(pointer, bytes) of a workspace tensor (or None)."""
    if workspace is None:
        return None, 0
    return _ptr(workspace), workspace.numel() * workspace.element_size()


def gemm_w8a16_ws(weight, scales, group_size, bias, input, output, tokens, out_features,
                  in_features, workspace, stream=None):
    """gemm_w8a16 with a caller workspace (a zeroed device tensor of at
    least gemm_workspace_bytes bytes): long-K calls split over K."""
    wp, wb = _ws_args(workspace)
    _check(load().infer_hip_gemm_w8a16_ws(_ptr(weight), _ptr(scales), group_size, _ptr(bias),
                                          _ptr(input), _ptr(output), tokens, out_features,
                                          in_features, wp, wb, _stream(stream)))


def gemm_bf16_ws(weight, bias, input, output, tokens, out_features, in_features, workspace,
                 stream=None):
    """gemm_bf16 with a caller workspace (see gemm_w8a16_ws)."""
    wp, wb = _ws_args(workspace)
    _check(load().infer_hip_gemm_bf16_ws(_ptr(weight), _ptr(bias), _ptr(input), _ptr(output),
                                         tokens, out_features, in_features, wp, wb,
                                         _stream(stream)))


class W8A16GemvPlan:
    """A grouped W8A16 GEMV plan: ``calls`` is a sequence of
    ``(weight, scales, group_size, bias, input, output, out_features,
    in_features)`` tuples, each the arguments of one independent
    :func:`gemv_w8a16` call.  The tensors must outlive the plan."""

    def __init__(self, calls):
        calls = list(calls)
        arr = (W8A16GemvDesc * len(calls))()
        for d, c in zip(arr, calls):
            w, s, g, b, x, y, n, k = c
            d.weight, d.scales, d.group_size = _ptr(w), _ptr(s), g
            d.bias, d.input, d.output = _ptr(b), _ptr(x), _ptr(y)
            d.out_features, d.in_features = n, k
        handle = ctypes.c_void_p()
        _check(load().infer_hip_w8a16_gemv_plan_create(
            ctypes.cast(arr, ctypes.c_void_p) if calls else None, len(calls),
            ctypes.byref(handle)))
        self._handle = handle
        self.count = len(calls)

    @property
    def bytes(self) -> float:
        """Compulsory bytes one launch moves."""
        return float(load().infer_hip_w8a16_gemv_plan_bytes(self._handle))

    def launch(self, stream=None) -> None:
        _check(load().infer_hip_w8a16_gemv_plan_launch(self._handle, _stream(stream)))

    def close(self) -> None:
        if self._handle:
            _check(load().infer_hip_w8a16_gemv_plan_destroy(self._handle))
            self._handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class GemmPlan:
    """A grouped GEMM plan: ``calls`` is a sequence of W8A16 tuples
    ``(weight, scales, group_size, bias, input, output, tokens,
    out_features, in_features)`` (the arguments of :func:`gemm_w8a16`) or of
    BF16 tuples ``(weight, bias, input, output, tokens, out_features,
    in_features)`` (:func:`gemm_bf16`); all of one kind.  The tensors must
    outlive the plan."""

    def __init__(self, calls):
        calls = list(calls)
        arr = (GemmDesc * len(calls))()
        for d, c in zip(arr, calls):
            if len(c) == 9:
                w, s, g, b, x, y, m, n, k = c
                d.w8a16, d.scales, d.group_size = 1, _ptr(s), g
            else:
                w, b, x, y, m, n, k = c
                d.w8a16, d.scales, d.group_size = 0, None, 0
            d.weight, d.bias, d.input, d.output = _ptr(w), _ptr(b), _ptr(x), _ptr(y)
            d.tokens, d.out_features, d.in_features = m, n, k
        handle = ctypes.c_void_p()
        _check(load().infer_hip_gemm_plan_create(
            ctypes.cast(arr, ctypes.c_void_p) if calls else None, len(calls),
            ctypes.byref(handle)))
        self._handle = handle
        self.count = len(calls)

    @property
    def flops(self) -> float:
        return float(load().infer_hip_gemm_plan_flops(self._handle))

    def launch(self, stream=None) -> None:
        _check(load().infer_hip_gemm_plan_launch(self._handle, _stream(stream)))

    def workgroups(self) -> int:
        """Timeline entries of the plan's GEMM launch: its workgroups (raises on
        plans with fewer than 256 tokens in some GEMM)."""
        n = ctypes.c_int(0)
        _check(load().infer_hip_gemm_plan_timeline(self._handle, None, 0, ctypes.byref(n), None))
        return n.value

    TIMELINE_WORDS = 16

    def launch_timeline(self, stamps, stream=None) -> None:
        """One launch that also writes each workgroup's 16 timeline words
        (int64 device tensor of 16 * workgroups() entries, zeroed)."""
        n = ctypes.c_int(0)
        _check(load().infer_hip_gemm_plan_timeline(
            self._handle, _ptr(stamps), stamps.numel() // self.TIMELINE_WORDS, ctypes.byref(n),
            _stream(stream)))

    def close(self) -> None:
        if self._handle:
            _check(load().infer_hip_gemm_plan_destroy(self._handle))
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
