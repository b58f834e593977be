"""Low-rank adapters (infer_hip_lora_bf16) in every launch form with inputs whose result
is a whole number that each step holds: A x of 15 or 16 bits, of which the first 8 cancel
in B, so that a part of A x that got lost is there in full.  With outputs of their own, in
place and without a base; q, k and v side by side in one row.

x and A hold whole numbers from 1 to 4 (K up to 8960: A x under 2^16, two BF16 numbers),
B holds -1, 0 and 1 and takes each row of A less another one that differs in a few
places: all sums are under 2^24, exact in FP32 in any order, and the only rounding is the
output's."""
import pytest
import torch

from test_gpu_lora import batch, gen, on, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


def whole(shape, g, low, high):
    return torch.randint(low, high + 1, shape, generator=g).to(torch.bfloat16)


def make(tokens, k, outs, rank, adapters, seed, runs=False):
    g = gen(seed)
    ids = torch.randint(-1, adapters, (tokens,), generator=g, dtype=torch.int32)
    s = {"x": whole((tokens, k), g, 1, 4), "ids": ids.sort().values if runs else ids,
         "scales": torch.tensor([1.0, -1.0, 2.0, 0.5])[torch.arange(adapters) % 4], "a": [],
         "b": [], "base": [whole((tokens, n), g, -100, 100) for n in outs]}
    for n in outs:
        a = whole((adapters, rank, k), g, 1, 4)
        a[:, 1::2] = a[:, ::2]
        at = torch.randint(0, k, (3,), generator=g)
        a[:, 1::2, at] = whole((adapters, rank // 2, 3), g, 1, 4)
        b = torch.zeros((adapters, n, rank))
        # three of the pairs in each column
        pair = torch.randint(0, rank // 2, (adapters, n, 3), generator=g)
        sign = torch.randint(0, 2, (adapters, n, 3), generator=g) * 2.0 - 1
        b.scatter_(2, 2 * pair, sign)
        b[:, :, 1::2] = -b[:, :, ::2]
        s["a"].append(a)
        s["b"].append(b.to(torch.bfloat16))
    return s


def exact(s, i, rows=slice(None), base=True):
    """Target i's output for those tokens, rounded once."""
    x, ids = s["x"][rows].double(), s["ids"][rows]
    zeros = torch.zeros((len(x), s["b"][i].shape[1]), dtype=torch.float64)
    out = s["base"][i][rows].double() if base else zeros
    for j in set(ids.tolist()) - {-1}:
        mine = (ids == j).nonzero()[:, 0]
        h = x[mine] @ s["a"][i][j].double().t()
        assert float(h.max()) < 65536
        out[mine] += float(s["scales"][j]) * (h @ s["b"][i][j].double().t())
    return out.to(torch.bfloat16)


FORMS = [
    # one launch, at ranks of 16 and 32; two launches: by tokens and by adapters, one and two
    # tiles of rows of A at a time, several tiles of a unit
    (1, 896, [896], 8, 4), (33, 1536, [200, 40, 24], 16, 40), (40, 1024, [300], 32, 2),
    (5, 8960, [100], 32, 3), (64, 896, [130], 64, 1), (33, 1536, [96, 40, 40], 64, 20),
    (100, 520, [257], 96, 60),
    # K in two and in four parts
    (3, 1544, [100], 40, 2), (128, 3584, [70, 50], 64, 12), (5, 8200, [40, 70], 128, 2),
    (9, 4104, [1030], 24, 3), (256, 4104, [65], 16, 1), (70, 1600, [40, 9, 300], 56, 1),
    # grouped: one tile of rows of A and two; a unit's tiles side by side in fours, in twos
    # and one after the other
    (300, 1536, [40], 16, 5), (700, 1544, [24, 300], 56, 3), (1100, 3000, [136, 17], 128, 33),
    (6000, 264, [700], 16, 3), (9000, 264, [520, 520], 40, 7)]
# beyond 70 and 192 MiB of bases and outputs, rows of both alignments
LARGE = [(2301, 1544, [9000], 32, 5), (2301, 1544, [8999], 72, 5), (6001, 1536, [8960], 32, 6),
         (6001, 1536, [8959], 32, 6), (6001, 1544, [9008], 128, 4),
         (6001, 264, [4500, 4600], 64, 3)]


@pytest.mark.parametrize("where", ["apart", "in place", "no base"])
@pytest.mark.parametrize("tokens,k,outs,rank,adapters", FORMS + LARGE)
def test_whole_numbers_are_exact(batch, dev, tokens, k, outs, rank, adapters, where):  # noqa: F811
    s = make(tokens, k, outs, rank, adapters, tokens + k + rank)
    d = on(s, dev)
    own = [y.clone() if where == "in place" else torch.full_like(y, 7.0) for y in d["base"]]
    base = {"apart": d["base"], "in place": own, "no base": [None] * len(outs)}[where]
    batch.lora(d["x"], d["ids"], list(zip(d["a"], d["b"], base, own)),
               workspace(batch, tokens, rank, len(outs), dev), scales=d["scales"])
    rows = slice(0, tokens, 1 if tokens * sum(outs) < 1 << 23 else 29)
    for i, out in enumerate(own):
        want = exact(s, i, rows, where != "no base")
        assert torch.equal(out[rows].cpu(), want), (out[rows].cpu() - want).abs().max()
        if where == "apart":
            assert torch.equal(d["base"][i].cpu(), s["base"][i])
        if where == "no base":
            assert int((out[d["ids"] < 0] != 0).sum()) == 0


@pytest.mark.parametrize("tokens,rank", [(20, 16), (90, 64), (300, 16), (1500, 64), (5000, 32)])
@pytest.mark.parametrize("pad", [0, 5])
def test_projections_side_by_side_in_place(batch, dev, tokens, rank, pad):  # noqa: F811
    """q, k and v as columns of one row, `pad` more between them and at the end."""
    outs, k = [1536, 256, 256], 1544
    s = make(tokens, k, outs, rank, 6, tokens + pad, runs=True)
    d = on(s, dev)
    width = sum(outs) + 3 * pad
    row = torch.full((tokens, width), 3.0, dtype=torch.bfloat16, device=dev)
    views, at = [], 0
    for n in outs:
        views.append(row[:, at:at + n])
        at += n + pad
    for v, y in zip(views, d["base"]):
        v.copy_(y)
    batch.lora(d["x"], d["ids"], list(zip(d["a"], d["b"], views, views)),
               workspace(batch, tokens, rank, 3, dev), scales=d["scales"])
    for i, v in enumerate(views):
        assert torch.equal(v.cpu(), exact(s, i))
    if pad:
        rest = torch.ones(width, dtype=torch.bool)
        at = 0
        for n in outs:
            rest[at:at + n] = False
            at += n + pad
        assert (row.cpu()[:, rest] == 3).all()
