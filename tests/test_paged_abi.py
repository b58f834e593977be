"""The paged KV cache and the 4-bit weights without a GPU: exported symbols,
refusals before any HIP call, and the host packer and quantiser."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import w4_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def paged(hip):
    import paged_hip
    return paged_hip


def test_library_exports_every_paged_symbol(paged):
    lib = paged.load()
    text = open(os.path.join(ROOT, "include", "infer_paged.h")).read()
    declared = sorted(set(re.findall(r"\b(infer_hip_\w+)\s*\(", text)))
    assert declared
    for name in declared:
        assert hasattr(lib, name), name
    assert sorted(paged.EXPORTED_SYMBOLS) == declared


A = 4096  # an aligned address that is never followed


def pool(paged, **change):
    f = dict(format=1, num_pages=8, page_size=16, num_kv_heads=2, head_dim=64, key_pages=A,
             value_pages=A, key_scales=A, value_scales=A)
    f.update(change)
    return paged._Pages(*f.values())


def table(paged, **change):
    f = dict(pages=A, num_sequences=3, max_pages=4, stride=4)
    f.update(change)
    return paged._Table(*f.values())


BAD_POOLS = [(dict(format=3), "format"), (dict(page_size=8), "page_size"),
             (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
             (dict(head_dim=96), "head_dim"), (dict(num_pages=0), "pool"),
             (dict(num_kv_heads=0), "pool"), (dict(key_pages=None), "null"),
             (dict(value_pages=None), "null"), (dict(key_scales=None), "null"),
             (dict(format=2, value_scales=None), "null"), (dict(key_pages=A + 8), "aligned"),
             (dict(value_scales=A + 4), "aligned")]
BAD_TABLES = [(dict(pages=None), "null"), (dict(num_sequences=0), "block table"),
              (dict(num_sequences=65536), "block table"), (dict(max_pages=0), "block table"),
              (dict(stride=3), "block table"),
              (dict(max_pages=1 << 28, stride=1 << 28), "block table")]


def calls(paged, p, t):
    """The three operators with sound arguments but for the pool and table."""
    lib, p, t = paged.load(), ctypes.byref(p), ctypes.byref(t)
    need = lib.infer_hip_attention_paged_decode_workspace_bytes(3, 4, 2, 64)
    yield lambda: lib.infer_hip_kv_pages_store(p, t, A, A, 5, A, 256, 4, A, 128, A, 128, A, 9, A,
                                               256, None)
    yield lambda: lib.infer_hip_kv_pages_load(p, t, A, A, A, 7, None)
    yield lambda: lib.infer_hip_attention_paged_decode(p, t, A, A, 256, 4, A, A, need, None)


@pytest.mark.parametrize("change,why", BAD_POOLS)
def test_bad_pools_are_refused(hip, paged, change, why):
    for call in calls(paged, pool(paged, **change), table(paged)):
        assert call() == hip.INVALID_ARGUMENT
        assert why in paged.load().infer_hip_last_error().decode()


@pytest.mark.parametrize("change,why", BAD_TABLES)
def test_bad_tables_are_refused(hip, paged, change, why):
    for call in calls(paged, pool(paged), table(paged, **change)):
        assert call() == hip.INVALID_ARGUMENT
        assert why in paged.load().infer_hip_last_error().decode()


def test_null_pool_and_table_are_refused(hip, paged):
    lib, p, t = paged.load(), ctypes.byref(pool(paged)), ctypes.byref(table(paged))
    bad = hip.INVALID_ARGUMENT
    assert lib.infer_hip_kv_pages_load(None, t, A, A, A, 7, None) == bad
    assert lib.infer_hip_kv_pages_load(p, None, A, A, A, 7, None) == bad


STORE = dict(sequences=A, positions=A, tokens=5, query=A, query_stride=256, num_heads=4, key=A,
             key_stride=128, value=A, value_stride=128, rope=A, rope_positions=9, query_out=A,
             query_out_stride=256)


@pytest.mark.parametrize("change,why", [
    (dict(tokens=0), "tokens"), (dict(positions=None), "positions"),
    (dict(sequences=None, tokens=4), "tokens"), (dict(query=None), "query"),
    (dict(num_heads=0), "query"), (dict(num_heads=-1), "query"), (dict(query_out=None), "query_out"),
    (dict(query_stride=255), "multiple of 8"), (dict(query_stride=248), "stride"),
    (dict(query_out_stride=0), "stride"), (dict(key=None), "key"), (dict(value=A + 2), "value"),
    (dict(key_stride=120), "stride"), (dict(value_stride=-128), "stride"),
    (dict(rope_positions=0), "rope"), (dict(rope=A + 4), "rope"),
    (dict(tokens=1 << 30), "too many")])
def test_store_refusals(hip, paged, change, why):
    lib = paged.load()
    args = dict(STORE)
    args.update(change)
    rc = lib.infer_hip_kv_pages_store(ctypes.byref(pool(paged)), ctypes.byref(table(paged)),
                                      *args.values(), None)
    assert rc == hip.INVALID_ARGUMENT and why in lib.infer_hip_last_error().decode()


def test_load_and_attention_refusals(hip, paged):
    lib, p, t = paged.load(), ctypes.byref(pool(paged)), ctypes.byref(table(paged))
    bad, f = hip.INVALID_ARGUMENT, lib.infer_hip_kv_pages_load
    err = lambda: lib.infer_hip_last_error().decode()  # noqa: E731
    assert f(p, t, None, A, A, 7, None) == bad
    assert f(p, t, A, None, A, 7, None) == bad
    assert f(p, t, A, A, A + 8, 7, None) == bad and "aligned" in err()
    assert f(p, t, A, A, A, 0, None) == bad and "capacity" in err()
    f = lib.infer_hip_attention_paged_decode
    need = lib.infer_hip_attention_paged_decode_workspace_bytes(3, 4, 2, 64)
    assert need > 0
    assert f(p, t, None, A, 256, 4, A, A, need, None) == bad
    assert f(p, t, A, None, 256, 4, A, A, need, None) == bad
    assert f(p, t, A, A, 252, 4, A, A, need, None) == bad
    assert f(p, t, A, A, 248, 4, A, A, need, None) == bad and "stride" in err()
    assert f(p, t, A, A, 256, 3, A, A, need, None) == bad and "heads" in err()
    assert f(p, t, A, A, 256, 0, A, A, need, None) == bad
    assert f(p, t, A, A, 256, 4, A + 4, A, need, None) == bad
    assert f(p, t, A, A, 256, 4, A, None, need, None) == bad and "workspace" in err()
    assert f(p, t, A, A, 256, 4, A, A + 8, need, None) == bad
    assert f(p, t, A, A, 256, 4, A, A, need - 1, None) == bad and str(need) in err()


@pytest.mark.parametrize("args", [(0, 4, 2, 64), (1, 3, 2, 64), (1, 0, 1, 64), (1, 4, 2, 96),
                                  (65536, 4, 2, 64), (1, 4, 0, 64)])
def test_workspace_of_bad_shapes_is_zero(paged, args):
    assert paged.attention_paged_decode_workspace_bytes(*args) == 0


def test_pool_wrapper_refuses_what_it_cannot_hold(hip, paged):
    with pytest.raises(hip.InferError, match="format"):
        paged.KvPages.allocate(1, 16, 1, 64, "int4", "cpu")
    with pytest.raises(hip.InferError, match="GPU"):
        paged.KvPages.allocate(1, 16, 1, 64, "bf16", "cpu")
    k = torch.zeros((2, 1, 16, 64), dtype=torch.int8)
    s = torch.zeros((2, 1, 16))
    with pytest.raises(hip.InferError, match="need scales"):
        paged.KvPages(k, k)
    with pytest.raises(hip.InferError, match="no scales"):
        paged.KvPages(k.to(torch.bfloat16), k.to(torch.bfloat16), s, s)
    with pytest.raises(hip.InferError, match="one shape"):
        paged.KvPages(k, k[:1], s, s)
    with pytest.raises(hip.InferError, match="float32"):
        paged.KvPages(k, k, s, s[:1])
    with pytest.raises(hip.InferError, match="bfloat16, int8"):
        paged.KvPages(k.float(), k.float())


# --------------------------------------------------------- 4-bit weights --

def bf16_words(t):
    return t.view(torch.int16).numpy().view(np.uint16)


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (17, 96, 32), (33, 192, 64),
                                       (50, 896, 64)])
def test_pack_layout(hip, n, k, group):
    g = torch.Generator().manual_seed(n)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    s = torch.randn((n, k // group), generator=g).to(torch.bfloat16)
    packed, tiled = hip.pack_w4a16(q.numpy(), bf16_words(s), group)
    want, want_s = w4_ref.pack(q, s)
    assert np.array_equal(packed, want.numpy())
    assert np.array_equal(tiled, bf16_words(want_s))


def test_pack_refusals(hip):
    lib = hip.load()
    q = np.zeros((4, 64), np.int8)
    s = np.zeros((4, 1), np.uint16)
    for group, shape in ((16, (4, 64)), (64, (4, 96)), (0, (4, 64)), (128, (4, 64))):
        with pytest.raises(hip.InferError):
            hip.pack_w4a16(np.zeros(shape, np.int8), s, group)
    with pytest.raises(hip.InferError):
        hip.pack_w4a16(q, s[:3], 64)
    with pytest.raises(hip.InferError):
        hip.pack_w4a16(q.astype(np.int16), s, 64)
    for v in (8, -9):
        bad = q.copy()
        bad[3, 63] = v
        with pytest.raises(hip.InferError, match="outside"):
            hip.pack_w4a16(bad, s, 64)
    assert lib.infer_hip_w4a16_pack(None, A, 64, 4, 64, A, A) == hip.INVALID_ARGUMENT
    assert lib.infer_hip_w4a16_weight_bytes(0, 64) == 0
    assert lib.infer_hip_w4a16_weight_bytes(17, 129) == 2 * 2 * 1024
    assert lib.infer_hip_w4a16_scale_count(17, 128, 64) == 2 * 2 * 16
    assert lib.infer_hip_w4a16_scale_count(17, 130, 64) == 0
    # sizes past 32 bits
    assert lib.infer_hip_w4a16_weight_bytes(1 << 20, 1 << 14) == 1 << 33
    assert lib.infer_hip_w4a16_weight_bytes((1 << 31) - 1, 128) == 1024 << 27


def test_quantise(hip):
    w = np.random.default_rng(0).standard_normal((5, 128)).astype(np.float32)
    w[2, :64] = 0
    q, s = hip.quantize_w4a16(w, 64)
    assert q.dtype == np.int8 and np.abs(q).max() == 7 and s.shape == (5, 2)
    scale = np.abs(w.reshape(5, 2, 64)).max(axis=2) / np.float32(7)
    scale[2, 0] = 1
    assert np.array_equal(q.reshape(5, 2, 64), np.rint(w.reshape(5, 2, 64) / scale[..., None]))
    for bad in (w[:, :100], w[0], np.full((1, 64), np.nan, np.float32)):
        with pytest.raises(hip.InferError):
            hip.quantize_w4a16(bad, 64)


W4 = dict(weight=A, scales=A, group=64, bias=None, input=A, output=A, tokens=1, n=8, k=64)


@pytest.mark.parametrize("change,why", [
    (dict(weight=None), "null"), (dict(scales=None), "null"), (dict(input=None), "null"),
    (dict(output=None), "null"), (dict(group=16), "group"), (dict(group=128), "group"),
    (dict(k=0), "group"), (dict(k=-64), "group"), (dict(n=0), "N=0"), (dict(tokens=0), "tokens"),
    (dict(n=(1 << 28) + 1), "over"), (dict(k=(1 << 24) + 64), "over"),
    (dict(tokens=17), "tokens"), (dict(weight=A + 8), "aligned"), (dict(input=A + 2), "aligned"),
    (dict(scales=A + 8), "aligned")])
def test_w4_refusals(hip, change, why):
    args = dict(W4)
    args.update(change)
    rc = hip.load().infer_hip_gemv_w4a16(*args.values(), None)
    assert rc == hip.INVALID_ARGUMENT
    assert why in hip.load().infer_hip_last_error().decode()


def test_cpp_packer():
    # the parts of tests/cpp/test_w4a16.cpp that need no GPU
    cpp = os.path.join(ROOT, "tests", "cpp")
    subprocess.run(["make", "-C", cpp, "test_w4a16"], check=True, capture_output=True, timeout=300)
    out = subprocess.run([os.path.join(cpp, "test_w4a16"), "host"], capture_output=True, text=True,
                         timeout=60)
    assert out.returncode == 0 and "PASSED" in out.stdout, out.stdout + out.stderr
