"""4-bit products of activations far larger than the rest, short of overflow: an
output is off by no more than the roundings that include/infer_linear.h states, 2^-24
of 31 |x| each, also in rows whose weight at the large one is 0."""
import pytest
import torch

import w4_ref as ref
from test_gpu_gemv_w4 import check, make, run

pytestmark = pytest.mark.gpu


# a workgroup's waves splitting K (one and two row tiles), and whole row tiles a wave
@pytest.mark.parametrize("n,k,group", [(50, 1024, 64), (70, 4864, 128), (513, 96, 32),
                                       (33000, 1088, 64), (98319, 256, 32)])
@pytest.mark.parametrize("tokens", [1, 4, 16])
@pytest.mark.parametrize("large", [1e3, -1e5, 1e12, 1e30, -1e36])
def test_large_activations(hip, dev, n, k, group, tokens, large):
    q, s, x, b = make(n, k, group, tokens, n + tokens, bias=True)
    at = k // 3
    q[::2, at] = 0
    x[-1, at] = large
    got = run(hip, dev, q, s, group, b, x)
    y, bound = ref.product(q.to(dev), s.to(dev), group, b.to(dev), x.to(dev))
    check(got, y.cpu(), bound.cpu())
