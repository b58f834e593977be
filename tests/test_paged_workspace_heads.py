"""The attention's workspace size of shapes that the attention refuses is zero."""
import ctypes

import pytest

from test_paged_abi import A, paged, pool, table  # noqa: F401


@pytest.mark.parametrize("heads,kv", [(65536, 1), (65536, 65536), (1 << 20, 2), (131070, 65535)])
def test_more_heads_than_a_call_takes(hip, paged, heads, kv):
    assert paged.attention_paged_decode_workspace_bytes(3, heads, kv, 64) == 0
    lib, d = paged.load(), 64
    rc = lib.infer_hip_attention_paged_decode(
        ctypes.byref(pool(paged, num_kv_heads=min(kv, 65535))), ctypes.byref(table(paged)), A, A,
        heads * d, heads, A, A, 1 << 40, None)
    assert rc == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("heads,kv", [(65535, 1), (65535, 65535), (65534, 32767)])
def test_most_heads(paged, heads, kv):
    assert paged.attention_paged_decode_workspace_bytes(3, heads, kv, 64) > 0
