"""Calls of the paged cache whose grid would have 2^32 threads or more are refused
before the launch (no GPU is touched: the addresses are never followed)."""
import ctypes

import pytest

from test_paged_abi import A, STORE, paged, pool, table  # noqa: F401


# rows a token, 4 or 8 lanes a row: 2^32 threads at the first, just under it before
# the last workgroup is filled up at the second
@pytest.mark.parametrize("d,tokens", [(64, 1 << 27), (64, (1 << 27) - 1), (128, 1 << 26),
                                      (128, (1 << 26) - 1), (64, 1 << 28), (128, 200000000)])
def test_store_of_too_many_rows(hip, paged, d, tokens):
    args = dict(STORE, tokens=tokens, query_stride=4 * d, key_stride=2 * d, value_stride=2 * d,
                query_out_stride=4 * d)
    lib = paged.load()
    rc = lib.infer_hip_kv_pages_store(ctypes.byref(pool(paged, head_dim=d)),
                                      ctypes.byref(table(paged)), *args.values(), None)
    assert rc == hip.INVALID_ARGUMENT and "too many" in lib.infer_hip_last_error().decode()


def test_store_of_more_heads_than_64_bits_of_lanes(hip, paged):
    heads = (1 << 31) - 1
    args = dict(STORE, tokens=(1 << 31) - 1, num_heads=heads, query_stride=heads * 128 + 120,
                query_out_stride=heads * 128 + 120, key_stride=256, value_stride=256)
    lib = paged.load()
    rc = lib.infer_hip_kv_pages_store(ctypes.byref(pool(paged, head_dim=128)),
                                      ctypes.byref(table(paged)), *args.values(), None)
    assert rc == hip.INVALID_ARGUMENT and "too many" in lib.infer_hip_last_error().decode()


@pytest.mark.parametrize("d,capacity", [(64, 1 << 29), (64, (1 << 29) - 31), (128, 1 << 28),
                                        (128, (1 << 28) - 15), (64, 1 << 30), (128, (1 << 31) - 1)])
def test_load_of_too_many_positions(hip, paged, d, capacity):
    wide = dict(max_pages=1 << 22, stride=1 << 22)
    lib = paged.load()
    rc = lib.infer_hip_kv_pages_load(ctypes.byref(pool(paged, head_dim=d, page_size=256)),
                                     ctypes.byref(table(paged, **wide)), A, A, A, capacity, None)
    assert rc == hip.INVALID_ARGUMENT and "too many" in lib.infer_hip_last_error().decode()
