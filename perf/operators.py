"""Operators of a decode step that serves several sequences: the paged KV
cache (written with RoPE in BF16, INT8 or FP8, read back, attended by one new
token a sequence) and few-token products with 4-bit weights.

Each case is a dict of plain values.  ``prepare`` makes what a program holds
before the call, ``run`` is one pass: with ``own`` false in plain torch in 32
bits, with ``own`` true through the framework's entry points.  ``work`` is what
a pass cannot do without and ``exact`` its result in 64 bits, written from the
definitions.

Shapes (query heads, KV heads, head_dim): 14/2/64 and 12/2/128 as in
``perf/cases.py``, 32/8/128 and 28/4/128 for wider models, 8/8/64 without
shared heads.  Cache layout: pages [page][KV head][slot][head_dim], with a
FP32 scale per row [page][KV head][slot] where elements have 8 bits.  4-bit
weights: tiles of 16 rows by 128 columns, [N/16][K/128][4][16][4] dwords, dword
(b, r, s) holding row r's columns 32 s + 8 b .. + 8 in the nibble order
0 2 4 6 1 3 5 7 as value + 8; scales BF16 [N/16][K/group][16].
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "qwen2.5-jetson-inference_amd")

THETA = 1e6  # RoPE base
LIMIT = {"int8": 127.0, "fp8": 448.0}
ELEMENT = {"bf16": 2, "int8": 1, "fp8": 1}
SHAPES = {"14/2/64": (14, 2, 64), "12/2/128": (12, 2, 128), "32/8/128": (32, 8, 128),
          "28/4/128": (28, 4, 128), "8/8/64": (8, 8, 64)}
NIBBLES = (0, 2, 4, 6, 1, 3, 5, 7)  # column of each nibble of a dword


def listed():
    return [
        # A decode step's cache write for 24 sequences, BF16: pure latency.
        {"name": "store_24_bf16", "kind": "store", "shape": "14/2/64", "format": "bf16",
         "page": 16, "sequences": 24, "longest": 1000},
        # Four prompts written in INT8 and read back as the contiguous cache the
        # prompt's attention wants.
        {"name": "prompt_4x700_int8", "kind": "prompt", "shape": "14/2/64", "format": "int8",
         "page": 16, "sequences": 4, "longest": 700},
        # Long prompts of a wide model in FP8, ragged, larger pages.
        {"name": "prompt_6x5000_fp8", "kind": "prompt", "shape": "32/8/128", "format": "fp8",
         "page": 64, "sequences": 6, "longest": 5000},
        # One conversation taken out of a BF16 pool.
        {"name": "load_1x901_bf16", "kind": "load", "shape": "14/2/64", "format": "bf16",
         "page": 32, "sequences": 1, "longest": 901},
        # Many long sequences read back from INT8 pages.
        {"name": "load_12x9000_int8", "kind": "load", "shape": "28/4/128", "format": "int8",
         "page": 128, "sequences": 12, "longest": 9000},
        # The smallest attention: one sequence, a short context, small pages.
        {"name": "attend_1x101_bf16", "kind": "attend", "shape": "14/2/64", "format": "bf16",
         "page": 16, "sequences": 1, "longest": 101},
        # Ordinary serving: 16 ragged sequences (one slot of the batch empty),
        # INT8 cache.
        {"name": "attend_16x2000_int8", "kind": "attend", "shape": "12/2/128", "format": "int8",
         "page": 16, "sequences": 16, "longest": 2000},
        # A full batch of a wide model: 64 ragged sequences, FP8 cache.
        {"name": "attend_64x4000_fp8", "kind": "attend", "shape": "32/8/128", "format": "fp8",
         "page": 64, "sequences": 64, "longest": 4000},
        # One very long document, BF16: split over its length or idle.
        {"name": "attend_1x131001_bf16", "kind": "attend", "shape": "12/2/128",
         "format": "bf16", "page": 256, "sequences": 1, "longest": 131001},
        # The smallest product: one token by a square 4-bit Linear with bias.
        {"name": "w4_1x896x896", "kind": "w4", "tokens": 1, "n": 896, "k": 896, "group": 64,
         "bias": True},
        # gate and up as one matrix for five sequences, wider model.
        {"name": "w4_5x17920x1536", "kind": "w4", "tokens": 5, "n": 17920, "k": 1536,
         "group": 128, "bias": False},
        # A 4-bit LM head for sixteen sequences, small groups.
        {"name": "w4_16x151936x896", "kind": "w4", "tokens": 16, "n": 151936, "k": 896,
         "group": 32, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "prompt", "load", "attend", "attend", "attend", "w4", "w4"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        k = group * _log(rng, 2048 // group // 4, 8960 // group)
        n = _log(rng, 100, min(100000, 120000000 // k))
        return {"kind": kind, "tokens": rng.choice([1, 1, rng.randint(2, 16)]), "n": n, "k": k,
                "group": group, "bias": rng.random() < 0.4}
    shape = rng.choice(sorted(SHAPES))
    fmt = rng.choice(["bf16", "int8", "fp8"] if kind != "store" else ["bf16"])
    heads, kv, d = SHAPES[shape]
    sequences = 1 if kind != "store" and rng.random() < 0.25 else _log(rng, 2, 64)
    # rows of a KV head per call, by kind
    room = {"store": 64 * 4000, "prompt": 20000, "load": 60000, "attend": 160000}[kind]
    longest = _log(rng, 20, min({"store": 4000, "prompt": 6000}.get(kind, 100000),
                                max(40, room * 8 * 128 // (kv * d) // sequences)))
    return {"kind": kind, "shape": shape, "format": fmt, "page": rng.choice([16, 32, 64, 128, 256]),
            "sequences": sequences, "longest": longest}


# ------------------------------------------------------------- inputs --


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _lengths(case):
    """Ragged lengths of the case: the longest first, then any; a batch of
    eight or more that is read has an empty slot."""
    rng = random.Random(case["longest"] * 1000 + case["sequences"])
    out = [case["longest"]] + [rng.randint(1, case["longest"])
                               for _ in range(case["sequences"] - 1)]
    if case["sequences"] >= 8 and case["kind"] in ("load", "attend"):
        out[3] = 0
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case, seed):
    """Block table [sequences][pages of the longest] over a shuffled pool, -1
    behind a sequence's last page, and the pool's size."""
    lengths, page = _lengths(case), case["page"]
    width = -(-case["longest"] // page)
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + 2
    order = torch.randperm(total, generator=torch.Generator().manual_seed(int(seed) & 0xFFFFFFF))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c].to(torch.int32)
        at += c
    return table.cuda(), total


def _rope(positions_max, d):
    """(cos, sin) of every position, FP32 from 64-bit angles."""
    freq = THETA ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    a = torch.arange(positions_max, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.stack([a.cos(), a.sin()], dim=-1).float().contiguous()


def _pool(case, seed, g, filled):
    """Pages and scales of K and V: rows of N(0, 1), or zeros."""
    _, kv, d = SHAPES[case["shape"]]
    table, total = _table(case, seed)
    shape, fmt = (total, kv, case["page"], d), case["format"]
    pool = {"table": table}
    for name in ("key", "value"):
        if fmt == "bf16":
            pool[name] = _normal(g, shape) if filled else torch.zeros(
                shape, dtype=torch.bfloat16, device="cuda")
            pool[name + "_scales"] = None
            continue
        # rows whose largest element is near 3 standard deviations
        pool[name + "_scales"] = (torch.rand(shape[:3], generator=g, device="cuda") + 2.5) / LIMIT[
            fmt] if filled else torch.zeros(shape[:3], device="cuda")
        if fmt == "int8":
            x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * 42 if filled \
                else torch.zeros(shape, device="cuda", dtype=torch.float16)
            pool[name] = x.round_().clamp_(-127, 127).to(torch.int8)
        else:
            x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * 150 if filled \
                else torch.zeros(shape, device="cuda", dtype=torch.float16)
            pool[name] = x.clamp_(-448, 448).to(torch.float8_e4m3fn)
    return pool


def _kv_inputs(case, seed):
    heads, kv, d = SHAPES[case["shape"]]
    g, lengths = _gen(seed), _lengths(case)
    if case["kind"] in ("load", "attend"):
        s = _pool(case, seed, g, True)
        s["lengths"] = _ints(lengths)
        if case["kind"] == "attend":
            s["query"] = _normal(g, (len(lengths), heads, d), 2.0)
        return s
    s = _pool(case, seed, g, False)
    if case["kind"] == "store":  # one new token a sequence, at its end
        positions, ids = [n - 1 for n in lengths], list(range(len(lengths)))
        s["sequences"] = None  # token i is sequence i's
    else:  # whole prompts, one after the other
        positions = [p for n in lengths for p in range(n)]
        ids = [i for i, n in enumerate(lengths) for _ in range(n)]
        s["sequences"] = _ints(ids)
        s["lengths"] = _ints(lengths)
    # q, k and v are column blocks of one projection's output
    qkv = _normal(g, (len(positions), heads + 2 * kv, d))
    s["query"], s["key_rows"], s["value_rows"] = qkv.split([heads, kv, kv], dim=1)
    s["positions"], s["ids"] = _ints(positions), ids
    s["rope"] = _rope(case["longest"], d)
    return s


def _w4_inputs(case, seed):
    """Weights as a quantiser leaves them (normal, the largest of a group near
    7), activations with a few strong channels."""
    g = _gen(seed)
    n, k, group, t = case["n"], case["k"], case["group"], case["tokens"]
    q = (torch.randn((n, k), generator=g, device="cuda", dtype=torch.float16) * 2.7).round_().clamp_(
        -8, 7).to(torch.int8)
    scales = ((torch.rand((n, k // group), generator=g, device="cuda") + 0.5) * (0.02 / 2.7)).to(
        torch.bfloat16)
    x = _normal(g, (t, k))
    x[:, :: 97] *= 12
    return q, scales, x, _normal(g, (n,), 0.5) if case["bias"] else None


def _pack(q, scales):
    """The tiles and tiled scales of the module's docstring; rows and columns
    past the matrix hold 0 (nibble 8), scales past it 0."""
    n, k = q.shape
    rows, cols = -(-n // 16) * 16, -(-k // 128) * 128
    u = torch.full((rows, cols), 8, dtype=torch.uint8, device=q.device)
    u[:n, :k] = (q + 8).to(torch.uint8)
    u = u.view(rows // 16, 16, cols // 128, 4, 4, 8)[..., list(NIBBLES)]
    u = u.permute(0, 2, 4, 1, 3, 5).contiguous()  # [tile row][tile][b][r][s][nibble]
    packed = (u[..., 0::2] | (u[..., 1::2] << 4)).contiguous().view(-1)
    s = torch.zeros((rows, scales.shape[1]), dtype=torch.bfloat16, device=q.device)
    s[:n] = scales
    return packed, s.view(rows // 16, 16, -1).transpose(1, 2).contiguous()


def _framework():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import linear_hip
    import paged_hip
    return linear_hip, paged_hip


def prepare(case, seed):
    kind = case["kind"]
    if kind == "w4":
        q, scales, x, bias = _w4_inputs(case, seed)
        packed, tiled = _pack(q, scales)
        s = {"case": case, "weight": packed, "scales": tiled, "x": x, "bias": bias,
             "out": torch.empty((case["tokens"], case["n"]), dtype=torch.bfloat16, device="cuda")}
    else:
        heads, kv, d = SHAPES[case["shape"]]
        s = _kv_inputs(case, seed)
        s["case"] = case
        if kind == "attend":
            s["out"] = torch.empty_like(s["query"])
        else:
            if kind != "load":
                s["query_out"] = torch.empty(s["query"].shape, dtype=torch.bfloat16, device="cuda")
            if kind != "store":
                dest = (case["sequences"], kv, case["longest"], d)
                s["key_cache"] = torch.zeros(dest, dtype=torch.bfloat16, device="cuda")
                s["value_cache"] = torch.zeros(dest, dtype=torch.bfloat16, device="cuda")
    if own:
        # the handle of the pool and the attention's workspace, which a program
        # makes once
        s["linear"], s["paged"] = _framework()
        if kind != "w4":
            s["pages"] = s["paged"].KvPages(s["key"], s["value"], s["key_scales"],
                                            s["value_scales"])
        if kind == "attend":
            need = s["paged"].attention_paged_decode_workspace_bytes(case["sequences"], heads, kv, d)
            s["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- run --


def run(state):
    kind = state["case"]["kind"]
    if kind == "w4":
        return _own_w4(state) if own else _plain_w4(state)
    if kind in ("store", "prompt"):
        _own_store(state) if own else _plain_store(state)
        if kind == "store":
            return {"query": state["query_out"], "key": state["key"], "value": state["value"]}
    if kind == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    _own_load(state) if own else _plain_load(state)
    out = {"key": state["key_cache"], "value": state["value_cache"]}
    if kind == "prompt":
        out["query"] = state["query_out"]
    return out


def _own_w4(s):
    c = s["case"]
    s["linear"].gemv_w4a16(s["weight"], s["scales"], c["group"], s["bias"], s["x"], s["out"],
                           c["tokens"], c["n"], c["k"])
    return s["out"]


def _own_store(s):
    s["paged"].kv_pages_store(s["pages"], s["table"], s["positions"], s["query"], s["key_rows"],
                              s["value_rows"], s["query_out"], rope=s["rope"],
                              sequences=s["sequences"])


def _own_load(s):
    s["paged"].kv_pages_load(s["pages"], s["table"], s["lengths"], s["key_cache"],
                             s["value_cache"])


def _own_attend(s):
    s["paged"].attention_paged_decode(s["pages"], s["table"], s["lengths"], s["query"], s["out"],
                                      s["workspace"])
    return s["out"]


def _plain_w4(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    rows, cols = -(-n // 16) * 16, -(-k // 128) * 128
    u = torch.stack([s["weight"] & 15, s["weight"] >> 4], dim=-1)
    u = u.view(rows // 16, cols // 128, 4, 16, 4, 8)
    u = u[..., [NIBBLES.index(i) for i in range(8)]].permute(0, 3, 1, 4, 2, 5).reshape(rows, cols)
    w = u[:n, :k].float() - 8
    scales = s["scales"].transpose(1, 2).reshape(rows, k // group)[:n].float()
    w = (w.view(n, k // group, group) * scales[:, :, None]).view(n, k)
    y = s["x"].float() @ w.t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(torch.bfloat16)


def _plain_rotate(x, cs):
    x, half = x.float(), x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_store(s):
    c, positions = s["case"], s["positions"].long()
    ids = torch.arange(len(positions), device="cuda") if s["sequences"] is None else s["sequences"]
    page = s["table"][ids.long(), positions // c["page"]].long()[:, None]
    slot = (positions % c["page"])[:, None]
    cs = s["rope"][positions]
    s["query_out"].copy_(_plain_rotate(s["query"], cs))
    head = torch.arange(s["key_rows"].shape[1], device="cuda")[None]
    for name, rows in (("key", _plain_rotate(s["key_rows"], cs)), ("value", s["value_rows"].float())):
        if c["format"] == "bf16":
            s[name][page, head, slot] = rows.to(torch.bfloat16)
            continue
        scale = rows.abs().amax(dim=-1) / LIMIT[c["format"]]
        q = rows / torch.where(scale == 0, 1.0, scale)[..., None]
        s[name + "_scales"][page, head, slot] = scale
        if c["format"] == "int8":
            s[name][page, head, slot] = q.round().clamp(-127, 127).to(torch.int8)
        else:
            q = q.clamp(-448, 448).to(torch.float8_e4m3fn)
            s[name].view(torch.uint8)[page, head, slot] = q.view(torch.uint8)


def _plain_gather(s, name):
    """Every sequence's rows in FP32, [sequences][KV heads][pages x page][d]."""
    at = s["table"].long().clamp(min=0)
    x = s[name]
    if x.dtype == torch.float8_e4m3fn:
        x = x.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    else:
        x = x[at].float()
    if s[name + "_scales"] is not None:
        x = x * s[name + "_scales"][at][..., None]
    b, pages, kv, page, d = x.shape
    return x.transpose(1, 2).reshape(b, kv, pages * page, d)


def _plain_load(s):
    longest = s["case"]["longest"]
    live = torch.arange(longest, device="cuda")[None] < s["lengths"][:, None]
    for name in ("key", "value"):
        rows = _plain_gather(s, name)[:, :, :longest].to(torch.bfloat16)
        out = s[name + "_cache"]
        out.copy_(torch.where(live[:, None, :, None], rows, out))


def _plain_attend(s):
    k, v = _plain_gather(s, "key"), _plain_gather(s, "value")
    b, kv, rows, d = k.shape
    q = s["query"].float().view(b, kv, -1, d)
    score = q @ k.transpose(2, 3) / math.sqrt(d)
    live = (torch.arange(rows, device="cuda")[None] < s["lengths"][:, None])[:, None, None]
    score = torch.where(live, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.where(live, (score - top).exp(), 0.0)
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out.view(b, -1, d).to(torch.bfloat16)


# --------------------------------------------------------------- work --


def work(case):
    """Each input read once, each output written once; multiply-adds as two."""
    if case["kind"] == "w4":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": n * k / 2 + 2.0 * n * k / case["group"] + 2.0 * t * k + 2.0 * t * n
                + (2.0 * n if case["bias"] else 0), "flops": 2.0 * t * n * k}
    heads, kv, d = SHAPES[case["shape"]]
    lengths = _lengths(case)
    row = 2 * kv * (d * ELEMENT[case["format"]] + (0 if case["format"] == "bf16" else 4))
    total, b = sum(lengths), case["sequences"]
    tables = 4.0 * sum(-(-n // case["page"]) for n in lengths) + 4 * b
    if case["kind"] == "attend":
        return {"bytes": total * row + 4.0 * b * heads * d + tables, "flops": 4.0 * total * heads * d}
    if case["kind"] == "load":
        return {"bytes": total * (row + 4.0 * kv * d) + tables, "flops": 2.0 * total * kv * d}
    tokens = b if case["kind"] == "store" else total
    angles = 4.0 * d * (tokens if case["kind"] == "store" else case["longest"])
    moved = tokens * (2.0 * (heads + 2 * kv) * d + 2.0 * heads * d + row) + angles + 8.0 * tokens
    if case["kind"] == "prompt":
        moved += 4.0 * total * kv * d + tables
    return {"bytes": moved, "flops": 6.0 * tokens * (heads + kv) * d / 2}


# -------------------------------------------------------------- exact --


def _exact_rope(x, position):
    """Rows [n][heads][d] turned by their positions' angles (the FP32 table is
    the operator's input)."""
    n, _, d = x.shape
    freq = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.as_tensor(position, device="cuda", dtype=torch.float64).view(n, 1, 1) * freq
    z = torch.complex(x[..., :d // 2].double(), x[..., d // 2:].double())
    z = z * torch.complex(angle.cos().float().double(), angle.sin().float().double())
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_held(rows, fmt):
    """The values that rows stand for once they are held in a format."""
    if fmt == "bf16":
        return rows.to(torch.bfloat16).double()
    s = rows.abs().max(dim=-1, keepdim=True).values / LIMIT[fmt]
    q = rows / s
    if fmt == "int8":
        return torch.round(q) * s
    # E4M3: steps of 2^(e - 3) in [2^e, 2^(e + 1)), 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step * s


def _exact_rows(s, case, name, i, n):
    """Sequence i's first n cached rows, [KV heads][n][d]."""
    pages = s["table"][i, :-(-n // case["page"])].tolist()
    take = lambda x: torch.cat([x[p] for p in pages], dim=1)[:, :n]  # noqa: E731
    x = take(s[name]).to(torch.float32).double()
    return x if s[name + "_scales"] is None else x * take(s[name + "_scales"]).double()[..., None]


def exact(case, seed):
    if case["kind"] == "w4":
        q, scales, x, bias = _w4_inputs(case, seed)
        out = []
        for at in range(0, case["n"], 8192):
            w = q[at:at + 8192].double() * scales[at:at + 8192].double().repeat_interleave(
                case["group"], dim=1)
            out.append(x.double() @ w.t())
        y = torch.cat(out, dim=1)
        return y if bias is None else y + bias.double()
    heads, kv, d = SHAPES[case["shape"]]
    s, lengths, fmt = _kv_inputs(case, seed), _lengths(case), case["format"]
    if case["kind"] == "attend":
        out = torch.zeros((len(lengths), heads, d), dtype=torch.float64, device="cuda")
        for i, n in enumerate(lengths):
            if n:
                k, v = (_exact_rows(s, case, name, i, n) for name in ("key", "value"))
                a = torch.softmax(s["query"][i].double().view(kv, -1, d)
                                  @ k.transpose(1, 2).contiguous() / math.sqrt(d), dim=-1)
                out[i] = (a @ v).view(heads, d)
        return out
    if case["kind"] == "load":
        out = {}
        for name in ("key", "value"):
            out[name] = torch.zeros((len(lengths), kv, case["longest"], d), dtype=torch.float64,
                                    device="cuda")
            for i, n in enumerate(lengths):
                if n:
                    out[name][i, :, :n] = _exact_rows(s, case, name, i, n)
        return out
    positions = s["positions"].tolist()
    rows = {"key": _exact_held(_exact_rope(s["key_rows"], positions), fmt),
            "value": _exact_held(s["value_rows"].double(), fmt)}
    out = {"query": _exact_rope(s["query"], positions)}
    if case["kind"] == "store":
        table = s["table"].tolist()
        for name in ("key", "value"):
            out[name] = s[name].double()
            for i, p in enumerate(positions):
                out[name][table[i][p // case["page"]], :, p % case["page"]] = rows[name][i]
        return out
    for name in ("key", "value"):
        out[name] = torch.zeros((len(lengths), kv, case["longest"], d), dtype=torch.float64,
                                device="cuda")
        at = 0
        for i, n in enumerate(lengths):
            out[name][i, :, :n] = rows[name][at:at + n].transpose(0, 1)
            at += n
    return out
