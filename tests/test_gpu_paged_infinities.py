"""Attention over BF16 pages that hold infinite values."""
import math

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import attention_case, paged, run_attention  # noqa: F401
from test_gpu_paged_scores import attend_rows

pytestmark = pytest.mark.gpu


def with_infinities(v, spots):
    v = v.clone()
    for position, dim, value in spots:
        v[:, position, dim] = value
    return v


@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (6, 1, 128), (16, 1, 64), (33, 1, 128)])
@pytest.mark.parametrize("n", [1, 5, 33, 64, 300, 500, 3000, 20000])
def test_infinite_values(paged, dev, heads, kv, d, n):
    """sum p v with an infinity of a positive weight is that infinity, with both
    it is NaN; other dimensions keep their sums."""
    g = torch.Generator().manual_seed(n)
    q = torch.randn((heads, d), generator=g).to(torch.bfloat16)
    k, v = (torch.randn((kv, n, d), generator=g).to(torch.bfloat16) for _ in range(2))
    spots = [(0, 3, math.inf), (n - 1, 20, -math.inf), (n // 2, 21, math.inf), (n // 3, 33, -math.inf),
             (n - 1, 33, -math.inf), (0, d - 1, math.inf), (n - 1, d - 1, math.inf)]
    both = [] if n == 1 else [(0, 40, math.inf), (n - 1, 40, -math.inf)]
    got, _ = attend_rows(paged, dev, "bf16", q, k, with_infinities(v, spots + both))
    exact, mean_abs, big = ref.attend(q, k.double(), v.double())
    tol = ref.attend_tolerance(exact, mean_abs, big, n, d)
    dims = {dim for _, dim, _ in spots + both}
    rest = [i for i in range(d) if i not in dims]
    assert ((got.double() - exact).abs() <= tol)[:, rest].all()
    for _, dim, value in spots:
        assert (got[:, dim] == value).all(), (dim, got[:, dim])
    for _, dim, _ in both:
        assert got[:, dim].isnan().all()


@pytest.mark.parametrize("n", [40, 3000])
def test_infinite_values_without_a_weight(paged, dev, n):
    """A score of -inf has no weight: 0 times an infinite value is NaN, and
    scores that are all -inf give NaN over any values."""
    d, g = 64, torch.Generator().manual_seed(3)
    q = torch.randn((2, d), generator=g).to(torch.bfloat16)
    q[:, 5] = 1.0
    k, v = (torch.randn((1, n, d), generator=g).to(torch.bfloat16) for _ in range(2))
    k[:, 17, 5] = -math.inf
    got, _ = attend_rows(paged, dev, "bf16", q, k, with_infinities(v, [(17, 9, math.inf)]))
    keep = [i for i in range(n) if i != 17]
    exact, mean_abs, big = ref.attend(q, k.double()[:, keep], v.double()[:, keep])
    ok = (got.double() - exact).abs() <= ref.attend_tolerance(exact, mean_abs, big, n, d)
    assert got[:, 9].isnan().all() and ok[:, [i for i in range(d) if i != 9]].all()
    k[:, :, 5] = -math.inf
    assert attend_rows(paged, dev, "bf16", q, k, v)[0].isnan().all()
    assert attend_rows(paged, dev, "bf16", q, k, v * 1e38)[0].isnan().all()


def test_infinite_values_behind_the_length(paged, dev):
    """Rows behind a sequence's length do not count."""
    lengths = [33, 700, 1]
    _, pages, table, q, out, out64 = attention_case(paged, dev, "bf16", 4, 2, 64, 16, lengths, 3,
                                                    poison=False)
    for s, n in enumerate(lengths):
        if n % 16:
            pages.value[int(table[s, n // 16]), :, n % 16:] = math.inf
    run_attention(paged, dev, pages, table, lengths, q, out)
    for s, (exact, mean_abs, big) in enumerate(out64):
        tol = ref.attend_tolerance(exact, mean_abs, big, lengths[s], 64)
        assert ((out[s].cpu().double() - exact).abs() <= tol).all()
