"""Python binding of the operators of a served batch (include/infer_batch.h):
low-rank adapters of many requests, and each sequence's next token.

Arguments are torch CUDA tensors on the current device.  A nonzero status raises
:class:`linear_hip.InferError`; shapes, types and devices that the C ABI cannot
see are checked here.  No reference counterpart: the reference runs one
sequence of one model (src/qwen2.cpp:597-674,
Greedy-cy/qwen2.5-jetson-inference).
"""
from __future__ import annotations

import ctypes
import struct

import torch

import linear_hip
from linear_hip import INVALID_ARGUMENT, InferError, _check, _flat, _here, _too_large

# Every symbol include/infer_batch.h declares.
EXPORTED_SYMBOLS = (
    "infer_hip_lora_workspace_bytes",
    "infer_hip_lora_bf16",
    "infer_hip_sample_workspace_bytes",
    "infer_hip_sample_bf16",
)

MAX_TARGETS = 3


class _Target(ctypes.Structure):
    """infer_hip_lora_target."""
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("base", ctypes.c_void_p),
                ("output", ctypes.c_void_p), ("out_features", ctypes.c_int),
                ("base_stride", ctypes.c_longlong), ("output_stride", ctypes.c_longlong)]


_lib = None
_BF16, _I32, _F32, _U8 = torch.bfloat16, torch.int32, torch.float32, torch.uint8
# One to three of _Target as bytes: a third of the time that setting its fields takes.
_PACK = [struct.Struct("@" + "PPPPi4xqq" * n).pack for n in range(MAX_TARGETS + 1)]


def load():
    global _lib
    if _lib is not None:
        return _lib
    lib = linear_hip.load()
    p, i, ll, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
    sigs = {
        "infer_hip_lora_workspace_bytes": ([i, i, i], z),
        "infer_hip_lora_bf16": ([p, ll, p, i, i, p, i, i, i, p, p, p, z, p], i),
        "infer_hip_sample_workspace_bytes": ([i, i], z),
        "infer_hip_sample_bf16": ([p, ll, i, i, p, p, p, p, p, p, p, p, z, p], i),
    }
    for name, (args, res) in sigs.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    _lib = lib
    return lib


def _bad(text: str):
    raise InferError(INVALID_ARGUMENT, text)


def _rows(t, rows, columns, index, name):
    """Pointer and row stride of BF16 [rows, columns] with contiguous rows."""
    if t.dtype is _BF16 and t.get_device() == index and t.shape == (rows, columns):
        if t.is_contiguous():
            return t.data_ptr(), columns
    else:
        _bad(f"{name} must be bfloat16 [{rows}, {columns}] on GPU {index} (got {list(t.shape)} "
             f"{t.dtype} on {t.device})")
    stride, inner = t.stride()
    if inner != 1 and columns > 1:
        _bad(f"{name}: rows must be contiguous")
    return t.data_ptr(), stride if rows > 1 else columns


def lora_workspace_bytes(tokens: int, max_rank: int, targets: int) -> int:
    return load().infer_hip_lora_workspace_bytes(tokens, max_rank, targets)


def lora(x, ids, targets, workspace, ranks=None, scales=None, stream=None) -> None:
    """output = base + scales[i] B[i] (A[i] x), with i = ids[t] of each token t
    (infer_hip_lora_bf16): x [tokens, K], ids int32 [tokens], targets one to three
    (a [adapters, max_rank, K], b [adapters, N, max_rank], base [tokens, N] or
    None, output [tokens, N]), ranks int32 and scales float32 [adapters] or
    None, workspace uint8 of lora_workspace_bytes.  output may be base."""
    index, on = _here(x, "x", stream)
    if x.dim() != 2 or not 1 <= len(targets) <= MAX_TARGETS:
        _bad(f"lora: x [tokens, K] and 1 to {MAX_TARGETS} targets (got {list(x.shape)}, "
             f"{len(targets)})")
    tokens, k = x.shape
    xp, xs = _rows(x, tokens, k, index, "x")
    shape = targets[0][0].shape
    if len(shape) != 3 or shape[2] != k:
        _bad(f"a must be [adapters, max_rank, {k}] (got {list(shape)})")
    adapters, rank = shape[0], shape[1]
    made, sizes = [], tokens | k | adapters
    for a, b, base, output in targets:
        n = output.shape[-1]
        sizes |= n
        # contiguous, as a rule: looked at without a call for each
        if (base is not None and a.dtype is _BF16 and a.get_device() == index and a.shape == shape
                and a.is_contiguous() and b.dtype is _BF16 and b.get_device() == index
                and b.shape == (adapters, n, rank) and b.is_contiguous()
                and base.dtype is _BF16 and base.get_device() == index
                and base.shape == (tokens, n) and base.is_contiguous()
                and output.dtype is _BF16 and output.get_device() == index
                and output.dim() == 2 and output.shape[0] == tokens and output.is_contiguous()):
            made += (a.data_ptr(), b.data_ptr(), base.data_ptr(), output.data_ptr(), n, n, n)
            continue
        if a.shape != shape or b.shape != (adapters, n, rank):
            _bad(f"a must be {list(shape)} and b {[adapters, n, rank]} (got {list(a.shape)}, "
                 f"{list(b.shape)})")
        op, os_ = _rows(output, tokens, n, index, "output")
        bp, bs = (0, 0) if base is None else _rows(base, tokens, n, index, "base")
        made += (_flat(a, _BF16, None, index, "a"), _flat(b, _BF16, None, index, "b"), bp, op, n,
                 bs, os_)
    if sizes >> 31:  # ctypes would pass the low half
        _too_large("lora")
    status = load().infer_hip_lora_bf16(
        xp, xs, _flat(ids, _I32, tokens, index, "ids"), tokens, k, _PACK[len(targets)](*made),
        len(targets), adapters, rank,
        None if ranks is None else _flat(ranks, _I32, adapters, index, "ranks"),
        None if scales is None else _flat(scales, _F32, adapters, index, "scales"),
        _flat(workspace, _U8, None, index, "workspace"), workspace.numel(), on)
    if status:
        _check(status)


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    return load().infer_hip_sample_workspace_bytes(rows, vocab)


def sample(logits, uniform, tokens, workspace, temperature=None, top_k=None, top_p=None,
           min_p=None, probabilities=None, stream=None) -> None:
    """The next token of every row of logits [rows, vocab] (infer_hip_sample_bf16):
    uniform float32 [rows] in [0, 1), tokens int32 [rows] written; temperature,
    top_p and min_p float32 and top_k int32 [rows] or None (off), probabilities
    float32 [rows] written or None, workspace uint8 of
    sample_workspace_bytes."""
    index, on = _here(logits, "logits", stream)
    if logits.dim() != 2:
        _bad(f"logits must be [rows, vocab] (got {list(logits.shape)})")
    rows, vocab = logits.shape
    lp, stride = _rows(logits, rows, vocab, index, "logits")
    if (rows | vocab) >> 31:  # ctypes would pass the low half
        _too_large("sample")

    def setting(t, dtype, name):
        return None if t is None else _flat(t, dtype, rows, index, name)
    _check(load().infer_hip_sample_bf16(
        lp, stride, rows, vocab, setting(temperature, _F32, "temperature"),
        setting(top_k, _I32, "top_k"), setting(top_p, _F32, "top_p"),
        setting(min_p, _F32, "min_p"), _flat(uniform, _F32, rows, index, "uniform"),
        _flat(tokens, _I32, rows, index, "tokens"), setting(probabilities, _F32, "probabilities"),
        _flat(workspace, _U8, None, index, "workspace"), workspace.numel(), on))
