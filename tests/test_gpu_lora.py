"""Low-rank adapters (infer_hip_lora_bf16) against their definition in 64 bits
(tests/batch_ref.py): tokens from one to thousands, ranks, odd sizes, strides,
several projections, ids out of range, unused rows that hold NaN, outputs in
place, infinities, captured graphs, another stream."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def batch():
    import batch_hip
    batch_hip.load()
    return batch_hip


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(shape, g, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def workspace(batch, tokens, rank, targets, dev):
    need = batch.lora_workspace_bytes(tokens, rank, targets)
    # NaN words: what a workspace holds before a call must not matter
    return torch.full((need,), 255, dtype=torch.uint8, device=dev)


def make(tokens, k, outs, rank, adapters, seed, runs=False):
    g = gen(seed)
    ids = torch.randint(-1, adapters, (tokens,), generator=g, dtype=torch.int32)
    if runs:
        ids = ids.sort().values
    ranks = torch.randint(0, rank + 1, (adapters,), generator=g, dtype=torch.int32)
    ranks[0] = rank
    s = {"x": bf16((tokens, k), g), "ids": ids, "ranks": ranks,
         "scales": torch.rand(adapters, generator=g) * 2 - 0.5,
         "a": [bf16((adapters, rank, k), g, k ** -0.5) for _ in outs],
         "b": [bf16((adapters, n, rank), g, 0.2) for n in outs],
         "base": [bf16((tokens, n), g) for n in outs]}
    for i in range(adapters):  # unused rows and columns
        for a, b in zip(s["a"], s["b"]):
            a[i, ranks[i]:] = float("nan")
            b[i, :, ranks[i]:] = float("nan")
    return s


def on(s, dev):
    return {k: [t.to(dev) for t in v] if isinstance(v, list) else v.to(dev) for k, v in s.items()}


def check(got, s, i, base=True, ranks=True, scales=True):
    want, tol = ref.lora(s["x"], s["ids"], s["ranks"] if ranks else None,
                         s["scales"] if scales else None, s["a"][i], s["b"][i],
                         s["base"][i] if base else None)
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), (float((off / tol).max()), (off > tol).nonzero()[:4].tolist())


CASES = [
    # tokens, k, outs, rank, adapters
    (1, 8, [1], 8, 1), (1, 896, [896], 8, 4), (2, 40, [17], 16, 3), (15, 104, [130], 24, 2),
    (16, 256, [128, 64], 32, 5), (17, 1000, [1000, 24, 24], 40, 3), (33, 1536, [1536, 256, 256], 16, 40),
    (64, 520, [513], 64, 1), (65, 136, [127, 129], 96, 7), (128, 896, [4864, 4864], 128, 6),
    (200, 72, [300], 104, 300), (257, 4864, [896], 48, 9), (1024, 64, [200], 8, 5),
    (1025, 64, [200], 72, 2000), (1100, 328, [136], 16, 33),
    # one launch and two, around ranks of 16, 32 and 64; rows of A beyond four tiles, of
    # several targets in one; K around a chunk's columns
    (3, 1024, [1025], 16, 2), (3, 1032, [1023], 32, 2), (7, 512, [65], 40, 2),
    (256, 520, [70], 32, 1), (256, 2056, [40, 50, 60], 24, 255), (300, 64, [40, 41, 42], 24, 5),
    (700, 1544, [24, 300], 56, 3), (513, 504, [33, 8, 9], 128, 2), (290, 4096, [128], 32, 1),
    (2050, 8, [16], 8, 700),
    # up to 256 tokens in two launches: K in two and four parts, several tiles of a unit one
    # after the other; two and four tiles of rows of A at a time
    (3, 1544, [100], 40, 2), (5, 3080, [40, 70], 128, 2), (9, 4104, [1030], 24, 3),
    (20, 3592, [257], 72, 1), (256, 4104, [65], 16, 1), (70, 1600, [40, 9, 300], 56, 1),
    (60, 128, [40], 80, 60), (100, 72, [40, 50], 64, 90), (120, 64, [20, 21, 22], 120, 119)]


@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("tokens,k,outs,rank,adapters", CASES)
def test_values(batch, dev, tokens, k, outs, rank, adapters, runs):
    s = make(tokens, k, outs, rank, adapters, tokens + k, runs)
    d = on(s, dev)
    out = [torch.full((tokens + 1, n), 7.0, dtype=torch.bfloat16, device=dev) for n in outs]
    batch.lora(d["x"], d["ids"], [(a, b, y, o[:tokens]) for a, b, y, o in
                                  zip(d["a"], d["b"], d["base"], out)],
               workspace(batch, tokens, rank, len(outs), dev), ranks=d["ranks"],
               scales=d["scales"])
    for i, o in enumerate(out):
        check(o[:tokens], s, i)
        assert (o[tokens:] == 7).all()
        none = s["ids"] < 0
        assert torch.equal(o[:tokens].cpu()[none], s["base"][i][none])
        assert torch.equal(d["base"][i].cpu(), s["base"][i])


@pytest.mark.parametrize("tokens,k,n,rank", [(1, 896, 896, 8), (5, 64, 100, 24), (40, 512, 1000, 64)])
def test_in_place_without_base_and_without_settings(batch, dev, tokens, k, n, rank):
    s = make(tokens, k, [n], rank, 3, 5)
    s["ranks"][:] = rank
    g = gen(6)
    s["a"][0], s["b"][0] = bf16((3, rank, k), g, k ** -0.5), bf16((3, n, rank), g, 0.2)
    d, ws = on(s, dev), workspace(batch, tokens, rank, 1, dev)
    a, b, out = d["a"][0], d["b"][0], d["base"][0].clone()
    batch.lora(d["x"], d["ids"], [(a, b, out, out)], ws)
    check(out, s, 0, scales=False)
    out.fill_(float("nan"))
    batch.lora(d["x"], d["ids"], [(a, b, None, out)], ws, scales=d["scales"])
    check(out, s, 0, base=False)
    assert (out.cpu()[s["ids"] < 0] == 0).all()


@pytest.mark.parametrize("tokens,rank", [(20, 16), (200, 64), (1500, 32)])
def test_the_result_is_the_same_every_time(batch, dev, tokens, rank):
    s = make(tokens, 1536, [1000], rank, 5, 7)
    d = on(s, dev)
    ws = workspace(batch, tokens, rank, 1, dev)
    outs = []
    for _ in range(3):
        out = torch.empty_like(d["base"][0])
        batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)], ws,
                   ranks=d["ranks"], scales=d["scales"])
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("shift,pad", [(0, 8), (0, 3), (1, 0), (8, 16), (5, 7)])
def test_strides_and_alignment(batch, dev, shift, pad):
    """Outputs and bases as column blocks of wider rows, x a block of its own."""
    s = make(21, 72, [131, 64], 16, 3, 8)
    d = on(s, dev)
    width = 131 + 64 + shift + pad
    wide = torch.full((21, width), 3.0, dtype=torch.bfloat16, device=dev)
    base = torch.full((21, width), 5.0, dtype=torch.bfloat16, device=dev)
    cuts = [slice(shift, shift + 131), slice(shift + 131, shift + 195)]
    for i, c in enumerate(cuts):
        base[:, c] = d["base"][i]
    x = torch.full((21, 72 + 24), float("nan"), dtype=torch.bfloat16, device=dev)
    x[:, 8:80] = d["x"]
    batch.lora(x[:, 8:80], d["ids"], [(d["a"][i], d["b"][i], base[:, c], wide[:, c])
                                      for i, c in enumerate(cuts)],
               workspace(batch, 21, 16, 2, dev), ranks=d["ranks"], scales=d["scales"])
    for i, c in enumerate(cuts):
        check(wide[:, c], s, i)
    assert (wide[:, :shift] == 3).all() and (wide[:, shift + 195:] == 3).all()


def test_ids_out_of_range_have_no_adapter(batch, dev):
    s = make(20, 64, [40], 8, 3, 9)
    s["ids"][:8] = torch.tensor([3, 4, -1, -2, 2 ** 31 - 1, -2 ** 31, 1000, 2], dtype=torch.int32)
    d, out = on(s, dev), torch.empty((20, 40), dtype=torch.bfloat16, device=dev)
    s["ids"][(s["ids"] < 0) | (s["ids"] > 2)] = -1
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, 20, 8, 1, dev), ranks=d["ranks"], scales=d["scales"])
    check(out, s, 0)


def test_ranks_out_of_range_are_clamped(batch, dev):
    s = make(12, 64, [40], 16, 4, 10)
    g = gen(3)
    s["a"][0], s["b"][0] = bf16((4, 16, 64), g, 0.1), bf16((4, 40, 16), g, 0.2)
    s["ranks"] = torch.tensor([-5, 17, 2 ** 31 - 1, 3], dtype=torch.int32)
    s["ids"] = (torch.arange(12) % 4).to(torch.int32)
    d, out = on(s, dev), torch.empty((12, 40), dtype=torch.bfloat16, device=dev)
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, 12, 16, 1, dev), ranks=d["ranks"], scales=d["scales"])
    check(out, s, 0)


def test_all_tokens_without_an_adapter(batch, dev):
    s = make(50, 64, [200], 8, 3, 11)
    s["ids"][:] = -1
    s["base"][0][0, :3] = torch.tensor([-0.0, float("inf"), float("nan")], dtype=torch.bfloat16)
    d, out = on(s, dev), torch.empty((50, 200), dtype=torch.bfloat16, device=dev)
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, 50, 8, 1, dev), ranks=d["ranks"], scales=d["scales"])
    assert torch.equal(out.cpu().view(torch.int16), s["base"][0].view(torch.int16))


def test_infinities_and_nan_stay_with_their_token(batch, dev):
    s = make(18, 64, [96], 16, 2, 12)
    s["ids"] = (torch.arange(18) % 2).to(torch.int32)
    s["ranks"][:] = 16
    g = gen(4)
    s["a"][0], s["b"][0] = bf16((2, 16, 64), g, 0.1).abs(), bf16((2, 96, 16), g, 0.2).abs()
    s["scales"][:] = 1.0
    clean = {k: v for k, v in s.items()}
    s["x"] = s["x"].clone()
    s["x"][3, 5], s["x"][8, 60], s["x"][9, 0] = float("inf"), float("-inf"), float("nan")
    d, out = on(s, dev), torch.empty((18, 96), dtype=torch.bfloat16, device=dev)
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, 18, 16, 1, dev), ranks=d["ranks"], scales=d["scales"])
    out = out.cpu()
    assert (out[3] == float("inf")).all() and (out[8] == float("-inf")).all()
    assert out[9].isnan().all()
    rest = [i for i in range(18) if i not in (3, 8, 9)]
    want, tol = ref.lora(clean["x"], clean["ids"], None, None, s["a"][0], s["b"][0], s["base"][0])
    assert ((out.double() - want).abs() <= tol)[rest].all()


def test_thousands_of_tokens(batch, dev):
    s = make(5003, 512, [520], 32, 6, 13, runs=True)
    d, out = on(s, dev), torch.empty((5003, 520), dtype=torch.bfloat16, device=dev)
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, 5003, 32, 1, dev), ranks=d["ranks"], scales=d["scales"])
    check(out, s, 0)


@pytest.mark.parametrize("tokens", [2301, 6001])
@pytest.mark.parametrize("n,rank", [(9000, 8), (9001, 64), (8999, 72), (9008, 128), (9008, 64),
                                    (9000, 72)])
def test_outputs_too_large_for_the_caches(batch, dev, n, rank, tokens):
    """Beyond 70 and 192 MiB of bases and outputs; every 37th token is looked at."""
    s = make(tokens, 72, [n], rank, 5, n, runs=True)
    d, out = on(s, dev), torch.empty((tokens, n), dtype=torch.bfloat16, device=dev)
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)],
               workspace(batch, tokens, rank, 1, dev), ranks=d["ranks"], scales=d["scales"])
    some = slice(0, tokens, 37)
    part = dict(s, x=s["x"][some], ids=s["ids"][some], base=[s["base"][0][some]])
    check(out[some], part, 0)
    assert not out.isnan().any()


def test_offsets_past_32_bits(batch, dev):
    """Tokens, and an adapter, whose bytes and elements lie past 2^32."""
    tokens, n, k, rank = 140000, 16384, 64, 8
    g = torch.Generator(device=dev).manual_seed(14)
    out = torch.zeros((tokens, n), dtype=torch.bfloat16, device=dev)  # 4.6 GB
    x = (torch.randn((tokens, k), generator=g, device=dev)).to(torch.bfloat16)
    ids = torch.full((tokens,), -1, dtype=torch.int32, device=dev)
    ids[-5:] = torch.tensor([0, 1, 1, -1, 0], device=dev)
    a = (torch.randn((2, rank, k), generator=g, device=dev) * 0.1).to(torch.bfloat16)
    b = (torch.randn((2, n, rank), generator=g, device=dev) * 0.2).to(torch.bfloat16)
    batch.lora(x, ids, [(a, b, out, out)], workspace(batch, tokens, rank, 1, dev))
    want, tol = ref.lora(x[-5:].cpu(), ids[-5:].cpu(), None, None, a.cpu(), b.cpu(),
                         torch.zeros((5, n), dtype=torch.bfloat16))
    assert ((out[-5:].cpu().double() - want).abs() <= tol).all()
    assert int((out[:-5] != 0).sum()) == 0


def test_an_adapter_past_2_32_elements(batch, dev):
    adapters, rank, k = 4200, 128, 8200
    a = torch.zeros((adapters, rank, k), dtype=torch.bfloat16, device=dev)  # 8.8 GB
    g = torch.Generator(device=dev).manual_seed(15)
    a[-1] = (torch.randn((rank, k), generator=g, device=dev) * 0.01).to(torch.bfloat16)
    b = torch.zeros((adapters, 24, rank), dtype=torch.bfloat16, device=dev)
    b[-1] = (torch.randn((24, rank), generator=g, device=dev) * 0.1).to(torch.bfloat16)
    x = torch.randn((3, k), generator=g, device=dev).to(torch.bfloat16)
    ids = torch.tensor([adapters - 1, 0, adapters - 1], dtype=torch.int32, device=dev)
    out = torch.empty((3, 24), dtype=torch.bfloat16, device=dev)
    batch.lora(x, ids, [(a, b, None, out)], workspace(batch, 3, rank, 1, dev))
    want, tol = ref.lora(x.cpu(), (ids > 0).int().cpu() - 1, None, None, a[-1:].cpu(),
                         b[-1:].cpu(), None)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("tokens,rank", [(30, 16), (100, 64), (400, 16), (60, 128)])
def test_captured_calls_follow_the_ids(batch, dev, tokens, rank):
    k = 1600 if rank == 128 else 256  # in parts
    s = make(tokens, k, [300, 40], rank, 6, 16)
    d = on(s, dev)
    ws = workspace(batch, tokens, rank, 2, dev)
    out = [torch.empty_like(y) for y in d["base"]]
    targets = list(zip(d["a"], d["b"], d["base"], out))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            batch.lora(d["x"], d["ids"], targets, ws, ranks=d["ranks"], scales=d["scales"])
    for step in range(4):
        s["ids"] = torch.randint(-1, 6, (tokens,), generator=gen(step), dtype=torch.int32)
        s["x"] = bf16((tokens, k), gen(step + 50))
        d["ids"].copy_(s["ids"])
        d["x"].copy_(s["x"])
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check(out[i], s, i)
        first = [o.clone() for o in out]
        batch.lora(d["x"], d["ids"], targets, ws, ranks=d["ranks"], scales=d["scales"])
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_another_stream(batch, dev):
    s = make(40, 896, [896], 16, 4, 17)
    d, ws = on(s, dev), workspace(batch, 40, 16, 1, dev)
    out = torch.empty_like(d["base"][0])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    batch.lora(d["x"], d["ids"], [(d["a"][0], d["b"][0], d["base"][0], out)], ws,
               ranks=d["ranks"], scales=d["scales"], stream=stream)
    stream.synchronize()
    check(out, s, 0)
