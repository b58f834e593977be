"""Adapters and sampling from their definitions in 64 bits, on CPU tensors: what
tests/test_gpu_lora.py and tests/test_gpu_sample.py compare the kernels with."""
import math

import torch

INF = math.inf


def lora(x, ids, ranks, scales, a, b, base):
    """(output, tolerance) of one target, float64 [tokens, N].

    The tolerance counts half a step of BF16 for the output (2^-8), 2^-16 of each
    h for its two BF16 parts, a rounding (2^-23) for each of the K + 2 operations
    of an h and for each of the 2 R + 2 of an output."""
    tokens, n = x.shape[0], b.shape[1]
    out = base.double().clone() if base is not None else torch.zeros((tokens, n)).double()
    slack = torch.zeros_like(out)
    for i in range(a.shape[0]):
        mine = (ids == i).nonzero()[:, 0]
        r = a.shape[1] if ranks is None else min(max(int(ranks[i]), 0), a.shape[1])
        if not len(mine) or not r:
            continue
        s = 1.0 if scales is None else float(scales[i])
        xs, w, v = x[mine].double(), a[i, :r].double(), b[i, :, :r].double()
        h = s * (xs @ w.t())
        size = abs(s) * (xs.abs() @ w.abs().t())
        out[mine] += h @ v.t()
        each = h.abs() * 2.0 ** -16 + size * ((x.shape[1] + 2) * 2.0 ** -23)
        slack[mine] = (each + h.abs() * ((2 * r + 2) * 2.0 ** -23)) @ v.abs().t()
    big = base.double().abs() if base is not None else 0.0
    return out, out.abs() * 2.0 ** -8 + slack * (1 + 2.0 ** -8) + big * 2.0 ** -23 + 1e-38


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.0):
    """(token, probability) of one row of logits."""
    v = logits.double()
    if any(math.isnan(s) for s in (temperature, top_p, min_p, uniform)) or v.isnan().any():
        return -1, math.nan
    if (v == -INF).all():
        return -1, 0.0
    v, order = v.sort(descending=True, stable=True)
    if not temperature > 0:
        temperature, top_k, top_p, min_p, uniform = 1.0, 1, 1.0, 0.0, 0.0
    if v[0] == INF:
        w = (v == INF).double()
    elif temperature == INF:
        w = (v > -INF).double()
    else:
        w = ((v - v[0]) / temperature).exp()
    w = w[v > -INF]
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        before = w.cumsum(0) - w
        w = w[:max(1, int((before < top_p * w.sum()).sum()))]
    if min_p > 0:
        w = w[:max(1, int((w >= min_p).sum()))]
    sums = w.cumsum(0)
    target = min(max(uniform, 0.0), 1 - 2.0 ** -24) * sums[-1]
    j = min(int((sums <= target).sum()), len(w) - 1)
    return int(order[j]), float(w[j] / sums[-1])
