"""Python binding of the paged KV cache (include/infer_paged.h).

:class:`KvPages` holds a pool's page and scale tensors; the functions take it
with a block table, and torch CUDA tensors for everything else.  A nonzero
status raises :class:`linear_hip.InferError`; shapes, types and devices that
the C ABI cannot see are checked here.  No reference counterpart: the
reference keeps one sequence's contiguous cache (include/infer/cuda_ops.hpp:
78-91, Greedy-cy/qwen2.5-jetson-inference).
"""
from __future__ import annotations

import ctypes

import torch

import linear_hip
from linear_hip import INVALID_ARGUMENT, InferError, _check, _flat, _here, _stream, _too_large

# Every symbol include/infer_paged.h declares.
EXPORTED_SYMBOLS = (
    "infer_hip_kv_pages_store",
    "infer_hip_kv_pages_load",
    "infer_hip_attention_paged_decode_workspace_bytes",
    "infer_hip_attention_paged_decode",
    "infer_hip_kv_pages_plan_workspace_bytes",
    "infer_hip_kv_pages_assign",
    "infer_hip_kv_pages_release",
)

FORMATS = {"bf16": 0, "int8": 1, "fp8": 2}


class _Pages(ctypes.Structure):
    """infer_hip_kv_pages."""
    _fields_ = [("format", ctypes.c_int), ("num_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("num_kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("key_pages", ctypes.c_void_p),
                ("value_pages", ctypes.c_void_p), ("key_scales", ctypes.c_void_p),
                ("value_scales", ctypes.c_void_p)]


class _Table(ctypes.Structure):
    """infer_hip_kv_table."""
    _fields_ = [("pages", ctypes.c_void_p), ("num_sequences", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("stride", ctypes.c_int)]


_lib = None
_BF16, _I32, _F32, _U8 = torch.bfloat16, torch.int32, torch.float32, torch.uint8
_I64 = torch.int64


def load():
    global _lib
    if _lib is not None:
        return _lib
    lib = linear_hip.load()
    p, i, ll, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
    pages, table = ctypes.POINTER(_Pages), ctypes.POINTER(_Table)
    sigs = {
        "infer_hip_kv_pages_store": ([pages, table, p, p, i, p, ll, i, p, ll, p, ll, p, i, p, ll,
                                      p], i),
        "infer_hip_kv_pages_load": ([pages, table, p, p, p, i, p], i),
        "infer_hip_attention_paged_decode_workspace_bytes": ([i, i, i, i], z),
        "infer_hip_attention_paged_decode": ([pages, table, p, p, ll, i, p, p, z, p], i),
        "infer_hip_kv_pages_plan_workspace_bytes": ([i], z),
        "infer_hip_kv_pages_assign": ([p, i, i, i, i, p, i, p, p, p, p, p, i, p, p, p, p, p, z, p],
                                      i),
        "infer_hip_kv_pages_release": ([p, i, i, i, i, p, i, p, p, p, p, p, p, z, p], i),
    }
    for name, (args, res) in sigs.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    _lib = lib
    return lib


def _bad(text: str):
    raise InferError(INVALID_ARGUMENT, text)


class KvPages:
    """A pool of KV pages over caller-owned tensors: key and value
    [pages][KV heads][page size][head_dim], contiguous, bfloat16, int8 or
    float8_e4m3fn, with float32 scales [pages][KV heads][page size] for the
    8-bit types (None for bfloat16)."""

    def __init__(self, key, value, key_scales=None, value_scales=None):
        formats = {torch.bfloat16: "bf16", torch.int8: "int8", torch.float8_e4m3fn: "fp8"}
        if key.dtype not in formats or key.dim() != 4:
            _bad(f"KvPages: key must be [pages, heads, page size, head_dim] of bfloat16, int8 or "
                 f"float8_e4m3fn (got {tuple(key.shape)} {key.dtype})")
        self.format = formats[key.dtype]
        scaled = self.format != "bf16"
        if scaled != (key_scales is not None) or scaled != (value_scales is not None):
            _bad(f"KvPages: {self.format} pages " + ("need scales" if scaled else "have no scales"))
        if value.shape != key.shape or value.dtype != key.dtype:
            _bad("KvPages: key and value must have one shape and type")
        tensors = [key, value] + ([key_scales, value_scales] if scaled else [])
        for t in tensors[2:]:
            if t.shape != key.shape[:3] or t.dtype != torch.float32:
                _bad("KvPages: scales must be float32 [pages, heads, page size]")
        if any(not t.is_contiguous() or not t.is_cuda or t.device != key.device for t in tensors):
            _bad("KvPages: pages and scales must be contiguous, on one GPU")
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = key.shape
        self.key, self.value, self.key_scales, self.value_scales = (
            key, value, key_scales, value_scales)
        self.device, self.index = key.device, key.get_device()
        self._struct = _Pages(FORMATS[self.format], self.num_pages, self.page_size,
                              self.num_kv_heads, self.head_dim, key.data_ptr(), value.data_ptr(),
                              key_scales.data_ptr() if scaled else None,
                              value_scales.data_ptr() if scaled else None)
        self._ref = ctypes.byref(self._struct)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 format: str = "bf16", device="cuda"):
        """A pool of its own, zeroed."""
        if format not in FORMATS:
            _bad(f"KvPages: format {format!r} (bf16, int8 or fp8)")
        dtype = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[format]
        shape = (num_pages, num_kv_heads, page_size, head_dim)

        def pages():
            return torch.zeros(shape, dtype=torch.uint8 if format != "bf16" else dtype,
                               device=device).view(dtype)

        def scales():
            return torch.zeros(shape[:3], device=device) if format != "bf16" else None
        return cls(pages(), pages(), scales(), scales())


# The checks below run on every call: they read each tensor as few times as
# they can (an attribute costs 40-110 ns, a launch 3.6 us).


def _at(t, dtype, pages, name):
    """Pointer of a contiguous tensor of a type on the pool's GPU."""
    if t.dtype is dtype and t.get_device() == pages.index and t.is_contiguous():
        return t.data_ptr()
    _bad(f"{name} must be contiguous {dtype} on {pages.device} (got {t.dtype} on {t.device})")


def _table(table, pages):
    """infer_hip_kv_table of an int32 tensor [sequences, pages] whose rows may be
    longer (a slice of a wider table)."""
    if table.dtype is not _I32 or table.dim() != 2 or table.get_device() != pages.index:
        _bad("block table must be int32 [sequences, pages] on the pool's GPU")
    rows, width = table.shape
    stride, inner = table.stride()
    if inner != 1 and width > 1:
        _bad("block table rows must be contiguous")
    return _Table(table.data_ptr(), rows, width, stride if rows > 1 else width)


def _rows(t, shape, pages, name):
    """Pointer and token stride of BF16 [tokens, heads, head_dim] with
    contiguous tokens."""
    if t.dtype is not _BF16 or t.get_device() != pages.index or t.shape != shape:
        _bad(f"{name} must be bfloat16 {list(shape)} on {pages.device} (got {t.dtype} "
             f"{list(t.shape)} on {t.device})")
    stride, between, inner = t.stride()
    if inner != 1 or (between != shape[2] and shape[1] > 1):
        _bad(f"{name}: a token's heads must be contiguous")
    return t.data_ptr(), stride if shape[0] > 1 else shape[1] * shape[2]


def _on(pages, stream):
    """The stream, of the pool's GPU, which must be the current one."""
    # a pool of tensors exists, so torch's HIP state does
    if (linear_hip._raw_device or torch.cuda.current_device)() != pages.index:
        _bad(f"the pool is on {pages.device}, the current device is {torch.cuda.current_device()}")
    if stream is None and linear_hip._raw_stream is not None:
        return linear_hip._raw_stream(pages.index)
    return _stream(stream)


def kv_pages_store(pages, table, positions, query, key, value, query_out=None, rope=None,
                   sequences=None, stream=None) -> None:
    """RoPE of query and key, key and value into the pages
    (infer_hip_kv_pages_store): query / key / value [tokens, heads, head_dim],
    positions int32 [tokens], rope float32 [positions, head_dim / 2, 2],
    sequences int32 [tokens] or None (token t belongs to sequence t).  query
    None: only the cache is written."""
    on = _on(pages, stream)
    tokens, d = positions.numel(), pages.head_dim
    tab = _table(table, pages)
    qp = qo = rp = sp = None
    qs = os_ = heads = rn = 0
    if query is not None:
        if query_out is None or query.dim() != 3:
            _bad("query and query_out must be [tokens, heads, head_dim]")
        heads = query.shape[1]
        shape = (tokens, heads, d)
        qp, qs = _rows(query, shape, pages, "query")
        qo, os_ = (qp, qs) if query_out is query else _rows(query_out, shape, pages, "query_out")
    shape = (tokens, pages.num_kv_heads, d)
    kp, ks = _rows(key, shape, pages, "key")
    vp, vs = _rows(value, shape, pages, "value")
    if rope is not None:
        rn = rope.shape[0]
        if rope.shape != (rn, d // 2, 2):
            _bad("rope must be float32 [positions, head_dim / 2, 2]")
        rp = _at(rope, _F32, pages, "rope")
    if sequences is not None:
        if sequences.numel() != tokens:
            _bad(f"sequences must hold {tokens} tokens")
        sp = _at(sequences, _I32, pages, "sequences")
    _check(load().infer_hip_kv_pages_store(
        pages._ref, tab, sp, _at(positions, _I32, pages, "positions"), tokens, qp, qs, heads, kp,
        ks, vp, vs, rp, rn, qo, os_, on))


def kv_pages_load(pages, table, lengths, key_cache, value_cache, stream=None) -> None:
    """The first lengths[s] positions of every sequence as BF16 into
    key_cache / value_cache [sequences, KV heads, capacity, head_dim]
    (infer_hip_kv_pages_load)."""
    on = _on(pages, stream)
    tab = _table(table, pages)
    shape = key_cache.shape
    if (len(shape) != 4 or value_cache.shape != shape or shape[0] != tab.num_sequences
            or shape[1] != pages.num_kv_heads or shape[3] != pages.head_dim):
        _bad("caches must be [sequences, KV heads, capacity, head_dim]")
    if lengths.numel() != tab.num_sequences:
        _bad(f"lengths must hold {tab.num_sequences} sequences")
    _check(load().infer_hip_kv_pages_load(
        pages._ref, tab, _at(lengths, _I32, pages, "lengths"),
        _at(key_cache, _BF16, pages, "key_cache"), _at(value_cache, _BF16, pages, "value_cache"),
        shape[2], on))


def attention_paged_decode_workspace_bytes(num_sequences: int, num_heads: int,
                                           num_kv_heads: int, head_dim: int) -> int:
    return load().infer_hip_attention_paged_decode_workspace_bytes(num_sequences, num_heads,
                                                                   num_kv_heads, head_dim)


def attention_paged_decode(pages, table, lengths, query, output, workspace, stream=None) -> None:
    """Attention of one new token a sequence: query and output
    [sequences, heads, head_dim], workspace a uint8 tensor of
    attention_paged_decode_workspace_bytes (infer_hip_attention_paged_decode)."""
    on = _on(pages, stream)
    tab = _table(table, pages)
    shape = query.shape
    if len(shape) != 3 or output.shape != shape:
        _bad("query and output must be [sequences, heads, head_dim]")
    if shape[0] != tab.num_sequences or shape[2] != pages.head_dim:
        _bad(f"query of {shape[0]} sequences and head_dim {shape[2]}: the table has "
             f"{tab.num_sequences}, the pool {pages.head_dim}")
    qp, qs = _rows(query, shape, pages, "query")
    if lengths.numel() != tab.num_sequences:
        _bad(f"lengths must hold {tab.num_sequences} sequences")
    _check(load().infer_hip_attention_paged_decode(
        pages._ref, tab, _at(lengths, _I32, pages, "lengths"), qp, qs, shape[1],
        _at(output, _BF16, pages, "output"), _at(workspace, _U8, pages, "workspace"),
        workspace.numel(), on))


def kv_pages_plan_workspace_bytes(num_sequences: int) -> int:
    return load().infer_hip_kv_pages_plan_workspace_bytes(num_sequences)


def _plan_table(table, stream):
    """(GPU, stream, pointer, rows, columns, distance of rows) of a plan's table,
    which may be a slice of a wider one."""
    index, handle = _here(table, "block table", stream)
    if table.dtype is not _I32 or table.dim() != 2:
        _bad("block table must be int32 [sequences, pages]")
    rows, width = table.shape
    stride, inner = table.stride()
    if inner != 1 and width > 1:
        _bad("block table rows must be contiguous")
    return index, handle, table.data_ptr(), rows, width, stride if rows > 1 else width


def kv_pages_assign(table, page_size: int, free, free_count, lengths, added, workspace, positions,
                    sequences=None, slots=None, starts=None, lengths_out=None,
                    free_count_out=None, stream=None) -> None:
    """Pages for added[s] new tokens of every sequence, and the tokens'
    positions (infer_hip_kv_pages_assign): table int32 [sequences, pages], free
    int32 [pages of the pool] with free_count int32 [1] of them unused, lengths
    and added int32 [sequences].  Written: the table's new entries, positions
    and sequences int32 [tokens], slots int64 [tokens], starts int32
    [sequences + 1], lengths_out and free_count_out (None: in place).
    sequences None: token s belongs to sequence s."""
    index, on, tp, n, width, stride = _plan_table(table, stream)
    if lengths_out is None:
        lengths_out = lengths
    if free_count_out is None:
        free_count_out = free_count
    tokens = positions.numel()
    # what every call has, looked at without a call for each
    if not (lengths.dtype is _I32 and lengths.get_device() == index and lengths.numel() == n
            and lengths.is_contiguous() and added.dtype is _I32 and added.get_device() == index
            and added.numel() == n and added.is_contiguous() and lengths_out.dtype is _I32
            and lengths_out.get_device() == index and lengths_out.numel() == n
            and lengths_out.is_contiguous() and positions.dtype is _I32
            and positions.get_device() == index and positions.is_contiguous()
            and free.dtype is _I32 and free.get_device() == index and free.is_contiguous()):
        for t, count, name in ((lengths, n, "lengths"), (added, n, "added"),
                               (lengths_out, n, "lengths_out"), (positions, None, "positions"),
                               (free, None, "free")):
            _flat(t, _I32, count, index, name)
    pool = free.numel()
    if (n | width | stride | pool | tokens) >> 31:  # ctypes would pass the low half
        _too_large("kv_pages_assign")
    status = load().infer_hip_kv_pages_assign(
        tp, n, width, stride, page_size, free.data_ptr(), pool,
        _flat(free_count, _I32, 1, index, "free_count"),
        _flat(free_count_out, _I32, 1, index, "free_count_out"), lengths.data_ptr(),
        added.data_ptr(), lengths_out.data_ptr(), tokens, positions.data_ptr(),
        None if sequences is None else _flat(sequences, _I32, tokens, index, "sequences"),
        None if slots is None else _flat(slots, _I64, tokens, index, "slots"),
        None if starts is None else _flat(starts, _I32, n + 1, index, "starts"),
        _flat(workspace, _U8, None, index, "workspace"), workspace.numel(), on)
    if status:
        _check(status)


def kv_pages_release(table, page_size: int, free, free_count, lengths, finished, workspace,
                     lengths_out=None, free_count_out=None, stream=None) -> None:
    """The pages of the sequences with finished[s] != 0 (int32 [sequences]) back
    onto free (infer_hip_kv_pages_release); the other arguments are
    kv_pages_assign's."""
    index, on, tp, n, width, stride = _plan_table(table, stream)
    if lengths_out is None:
        lengths_out = lengths
    if free_count_out is None:
        free_count_out = free_count
    if not (lengths.dtype is _I32 and lengths.get_device() == index and lengths.numel() == n
            and lengths.is_contiguous() and finished.dtype is _I32
            and finished.get_device() == index and finished.numel() == n
            and finished.is_contiguous() and lengths_out.dtype is _I32
            and lengths_out.get_device() == index and lengths_out.numel() == n
            and lengths_out.is_contiguous() and free.dtype is _I32
            and free.get_device() == index and free.is_contiguous()):
        for t, count, name in ((lengths, n, "lengths"), (finished, n, "finished"),
                               (lengths_out, n, "lengths_out"), (free, None, "free")):
            _flat(t, _I32, count, index, name)
    pool = free.numel()
    if (n | width | stride | pool) >> 31:
        _too_large("kv_pages_release")
    status = load().infer_hip_kv_pages_release(
        tp, n, width, stride, page_size, free.data_ptr(), pool,
        _flat(free_count, _I32, 1, index, "free_count"),
        _flat(free_count_out, _I32, 1, index, "free_count_out"), lengths.data_ptr(),
        finished.data_ptr(), lengths_out.data_ptr(),
        _flat(workspace, _U8, None, index, "workspace"), workspace.numel(), on)
    if status:
        _check(status)
