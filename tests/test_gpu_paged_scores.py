"""Attention over the paged cache of finite scores far past where FP32 holds
their fractions."""
import pytest
import torch

from test_gpu_paged import paged, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def attend_rows(paged, dev, fmt, q, k, v, page=16):
    """Attention of q [heads, d] over k, v [kv, n, d] through a pool that the
    store has written."""
    kv, n, d = k.shape
    pages = paged.KvPages.allocate(-(-n // page), page, kv, d, fmt, dev)
    table = torch.arange(pages.num_pages, dtype=torch.int32, device=dev)[None]
    paged.kv_pages_store(pages, table, torch.arange(n, dtype=torch.int32, device=dev), None,
                         k.transpose(0, 1).contiguous().to(dev), v.transpose(0, 1).contiguous().to(dev),
                         sequences=torch.zeros(n, dtype=torch.int32, device=dev))
    out = torch.empty((1,) + tuple(q.shape), dtype=torch.bfloat16, device=dev)
    run_attention(paged, dev, pages, table, [n], q[None].to(dev), out)
    return out[0].cpu(), pages


# 2^31 to past 2^100 in units of a weight's exponent, of both signs
BIG = [(1e4, 1e5), (3e5, 3e5), (-2e5, 2e5), (1e6, 1e6), (1e10, -1e10), (1e15, 1e15), (-7e14, 3e14)]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("qk", BIG)
@pytest.mark.parametrize("d,n", [(64, 1), (128, 1), (64, 7), (128, 40), (64, 700), (128, 3000)])
def test_large_finite_scores(paged, dev, fmt, qk, d, n):
    """Equal keys at every second position, the others at half of them: the
    greater scores are equal, and their weights; the others are nothing next to
    them.  (A score is a sum of at most 2^7 equal products of 16 bits: exact in
    any order, so equal keys have equal scores.)"""
    g = torch.Generator().manual_seed(n + d)
    q = torch.full((4, d), qk[0]).to(torch.bfloat16)
    k = torch.full((1, n, d), qk[1])
    k[:, 1::2] *= 0.5
    k = k.to(torch.bfloat16)
    v = torch.randn((1, n, d), generator=g).to(torch.bfloat16)
    got, pages = attend_rows(paged, dev, fmt, q, k, v)
    wins = slice(0, None, 2) if qk[0] * qk[1] > 0 or n == 1 else slice(1, None, 2)
    held = pages.value.view(torch.uint8).cpu().view(pages.value.dtype).float().double()
    if fmt != "bf16":
        held = held * pages.value_scales.cpu().double()[..., None]
    live = held.transpose(0, 1).reshape(1, -1, d)[:, :n][:, wins]
    exact, big = live.mean(dim=1), live.abs().mean(dim=1)
    # BF16's rounding of the output; weights as BF16; n sums in FP32
    tol = exact.abs() * 2.0 ** -8 + big * (2.0 ** -8 + n * 2.0 ** -24 + 2.0 ** -20)
    assert ((got.double() - exact).abs() <= tol).all(), float((got.double() - exact).abs().max())
