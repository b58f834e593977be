"""Sampling (infer_hip_sample_bf16) against its definition in 64 bits
(tests/batch_ref.py): tokens exactly, probabilities to FP32's rounding; settings
together and at their ends, ties, masks, infinities and NaN, vocabularies from
one token up, strides, captured graphs, another stream."""
import math

import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def batch():
    import batch_hip
    batch_hip.load()
    return batch_hip


def gen(seed):
    return torch.Generator().manual_seed(seed)


def run(batch, dev, logits, uniform, stream=None, **settings):
    """(tokens, probabilities) of rows of logits (a CPU or GPU tensor)."""
    rows = logits.shape[0]
    d = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).to(dev)
         for k, v in settings.items()}
    ws = torch.zeros(batch.sample_workspace_bytes(*logits.shape), dtype=torch.uint8, device=dev)
    tokens = torch.full((rows + 1,), -7, dtype=torch.int32, device=dev)
    probabilities = torch.full((rows + 1,), -7.0, device=dev)
    u, x = torch.tensor(uniform, dtype=torch.float32).to(dev), logits.to(dev)
    torch.cuda.synchronize()
    batch.sample(x, u, tokens[:rows], ws, probabilities=probabilities[:rows], stream=stream, **d)
    torch.cuda.synchronize()
    assert int(tokens[rows]) == -7 and float(probabilities[rows]) == -7
    return tokens[:rows].tolist(), probabilities[:rows].tolist()


def check(batch, dev, logits, uniform, **settings):
    tokens, chances = run(batch, dev, logits, uniform, **settings)
    f = lambda v: torch.tensor(v, dtype=torch.float32).double().tolist()  # noqa: E731
    for i in range(logits.shape[0]):
        one = {k: v[i] if k == "top_k" else f(v)[i] for k, v in settings.items()}
        token, chance = ref.sample(logits[i].cpu(), uniform=f(uniform)[i], **one)
        assert tokens[i] == token, (i, tokens[i], token, one)
        # rounded once to FP32, from sums in 64 bits
        assert (math.isnan(chance) and math.isnan(chances[i])) or (
            abs(chances[i] - chance) <= chance * (2.0 ** -24 + 1e-12)), (i, chances[i], chance)
    return tokens


def rows_of(rows, vocab, seed, std=2.2):
    """Many low logits and a few far above."""
    g = gen(seed)
    x = torch.randn((rows, vocab), generator=g) * std - 1
    at = torch.randint(0, vocab, (rows, min(vocab, 12)), generator=g)
    x.scatter_(1, at, torch.rand(at.shape, generator=g) * 9 + 4)
    return x.to(torch.bfloat16), torch.rand(rows, generator=g).tolist()


def pick(values, rows, seed):
    at = torch.randint(0, len(values), (rows,), generator=gen(seed)).tolist()
    return [values[i] for i in at]


def settings(rows, seed):
    return {"temperature": pick([0.0, 0.3, 0.7, 1.0, 1.0, 2.5], rows, seed),
            "top_k": pick([0, 0, 1, 2, 20, 50, 1000, 10 ** 6], rows, seed + 1),
            "top_p": pick([1.0, 1.0, 0.1, 0.8, 0.95, 0.999], rows, seed + 2),
            "min_p": pick([0.0, 0.0, 0.001, 0.05, 0.5], rows, seed + 3)}


@pytest.mark.parametrize("rows,vocab", [
    (1, 1), (3, 2), (5, 7), (4, 8), (9, 63), (33, 257), (40, 1000), (64, 4095), (20, 8192),
    (20, 8193), (12, 32003), (7, 65536), (7, 65537), (6, 100000), (24, 151936), (3, 155649),
    (2, 262147), (300, 901),
    (5, 16384), (5, 16385), (5, 32768), (5, 32769), (3, 106497), (3, 155648), (2, 1048576)])
def test_settings_together(batch, dev, rows, vocab):
    logits, uniform = rows_of(rows, vocab, vocab)
    check(batch, dev, logits, uniform, **settings(rows, vocab))


@pytest.mark.parametrize("vocab", [50, 5000, 151936])
def test_without_settings(batch, dev, vocab):
    logits, uniform = rows_of(30, vocab, 1)
    check(batch, dev, logits, uniform)
    # flat: every token near the next
    flat, uniform = (torch.randn((8, vocab), generator=gen(2)) * 0.05).to(torch.bfloat16), uniform[:8]
    check(batch, dev, flat, uniform)
    check(batch, dev, flat, uniform, top_p=[0.999, 0.5, 0.01, 0.7, 0.9, 0.3, 0.99, 1.0])


@pytest.mark.parametrize("vocab", [10, 1000, 70000, 151936])
def test_equal_logits_go_by_index(batch, dev, vocab):
    """All tokens alike, more of them than 16 bits count: sums are whole numbers, and the
    running sum passes u n after floor(u n) + 1 tokens."""
    us = [0.0, 0.25, 0.5, 0.75, 0.9999999]
    for value in (0.0, -3.5, 17.0):
        logits = torch.full((5, vocab), value, dtype=torch.bfloat16)
        got, chances = run(batch, dev, logits, us)
        f = torch.tensor(us, dtype=torch.float32).double()
        assert got == [int(u * vocab) for u in f.tolist()]
        assert chances == [float(torch.tensor(1.0 / vocab, dtype=torch.float32))] * 5
        got, _ = run(batch, dev, logits, us, top_k=[7] * 5)
        assert got == [int(u * min(7, vocab)) for u in f.tolist()]
        got, _ = run(batch, dev, logits, us, top_p=[0.5] * 5)
        kept = -(-vocab // 2)
        assert got == [int(u * kept) for u in f.tolist()]


@pytest.mark.parametrize("vocab", [3000, 140001])
def test_two_values_with_many_tokens_each(batch, dev, vocab):
    g = gen(vocab)
    logits = torch.where(torch.rand((10, vocab), generator=g) < 0.5, 1.5, 0.75).to(torch.bfloat16)
    uniform = torch.rand(10, generator=g).tolist()
    check(batch, dev, logits, uniform, **settings(10, 5))
    check(batch, dev, logits, uniform, top_k=[vocab // 2 + i * 17 for i in range(10)])


def test_both_zeros_are_one_value(batch, dev):
    logits = torch.tensor([[-1.0, -0.0, 0.0, -0.0, 0.0]] * 5).to(torch.bfloat16)
    got, _ = run(batch, dev, logits, [0.1, 0.35, 0.6, 0.85, 0.99], top_k=[4] * 5)
    assert got == [1, 2, 3, 4, 4]


@pytest.mark.parametrize("vocab", [100, 8000, 151936])
def test_masked_tokens_are_never_taken(batch, dev, vocab):
    logits, uniform = rows_of(12, vocab, 3)
    g = gen(4)
    for i, part in enumerate([0.1, 0.5, 0.9, 0.999]):
        logits[i][torch.rand(vocab, generator=g) < part] = -INF
    logits[4] = -INF
    logits[4, vocab - 1] = -8.0  # one token left, the last
    logits[5] = -INF  # none
    logits[6] = -INF
    logits[6, 0] = torch.finfo(torch.bfloat16).min
    logits[7][logits[7] < 0] = torch.finfo(torch.bfloat16).min  # masks of the lowest value
    uniform[:8] = [0.5, 0.9, 0.99, 0.999, 0.99, 0.5, 0.5, 0.99]
    got = check(batch, dev, logits, uniform)
    assert got[4] == vocab - 1 and got[5] == -1 and got[6] == 0
    check(batch, dev, logits, uniform, **settings(12, 6))
    check(batch, dev, logits, uniform, temperature=[1e-30] * 4 + [INF] * 4 + [3e38] * 4)
    check(batch, dev, logits, uniform, top_k=[vocab] * 12, top_p=[0.9] * 12)


@pytest.mark.parametrize("vocab", [9000, 40000, 151936, 300007])
@pytest.mark.parametrize("mask", [-INF, torch.finfo(torch.bfloat16).min, -1e4, -100.0])
def test_masks_by_region(batch, dev, vocab, mask):
    """Masks of half of the row, of its first piece alone, of all but that, of every second
    run, and thin ones that few lanes of a wave see."""
    logits, uniform = rows_of(7, vocab, 13)
    at = torch.arange(vocab)
    logits[0, vocab // 2:] = mask
    logits[1, :4096] = mask
    logits[2, 4096:] = mask
    logits[3, at // 512 % 2 == 0] = mask
    logits[4, at % 512 < 33] = mask
    logits[5, at % 16 == 3] = mask
    logits[6, at % 8 < 7] = mask
    check(batch, dev, logits, uniform)
    check(batch, dev, logits, uniform, **settings(7, vocab))
    check(batch, dev, logits, uniform, temperature=[1e3] * 7)


def test_infinities_and_nan(batch, dev):
    logits, _ = rows_of(10, 3000, 7)
    logits[0, 77] = INF
    logits[1, [5, 900, 2999]] = INF
    logits[2, 2999] = NAN
    logits[3, 0] = -NAN
    logits[4] = INF
    logits[5, 1:] = -INF
    logits[6] = -INF
    logits[6, 7] = NAN
    logits[7, [5, 900]] = INF
    logits[7, 800] = NAN
    u = [0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5]
    assert check(batch, dev, logits, u)[:3] == [77, 900, -1]
    check(batch, dev, logits, u, **settings(10, 8))
    check(batch, dev, logits, u, temperature=[INF] * 10)
    check(batch, dev, logits, u, temperature=[0.0] * 10)


def test_settings_at_their_ends(batch, dev):
    logits, _ = rows_of(1, 5000, 9)
    ends = {"temperature": [1.0, 0.0, -0.0, -1.0, 1e-45, 1e-30, 3e38, INF, -INF, NAN],
            "top_k": [0, 1, -1, 4999, 5000, 5001, 2 ** 31 - 1, -2 ** 31],
            "top_p": [1.0, 0.0, -1.0, 1e-30, 0.9999999, 2.0, INF, -INF, NAN],
            "min_p": [0.0, 1.0, 1.5, INF, -1.0, -INF, 1e-30, 1e-45, 0.9999999, NAN]}
    for name, values in ends.items():
        for uniform in (0.0, 0.6, 0.9999999):
            check(batch, dev, logits.expand(len(values), -1).contiguous(),
                  [uniform] * len(values), **{name: values})
    us = [0.0, -0.5, 1.0, 7.0, INF, -INF, NAN, 0.99999994, 1e-45]
    check(batch, dev, logits.expand(len(us), -1).contiguous(), us)
    check(batch, dev, logits.expand(len(us), -1).contiguous(), us, top_k=[3] * len(us))


def test_values_from_the_smallest_to_the_largest(batch, dev):
    """Every finite BF16 number once, in a shuffled order."""
    words = torch.arange(65536, dtype=torch.int32)
    words = words[((words >> 7) & 255) != 255]
    words = words[torch.randperm(len(words), generator=gen(10))]
    logits = words.to(torch.int16).view(torch.bfloat16).expand(6, -1).contiguous()
    u = [0.0, 0.3, 0.5, 0.7, 0.9, 0.99]
    check(batch, dev, logits, u, temperature=[3e38] * 6)
    check(batch, dev, logits, u, temperature=[1.0] * 6)
    small = (logits.float() * 2.0 ** -125).to(torch.bfloat16)  # values around 0
    check(batch, dev, small, u)
    check(batch, dev, small, u, top_k=[1, 100, 20000, 40000, 60000, 65000])


@pytest.mark.parametrize("vocab,shift,pad", [(1000, 0, 24), (1000, 1, 0), (999, 3, 6),
                                             (8197, 5, 11), (32000, 7, 1), (6, 1, 1)])
def test_rows_of_a_wider_tensor(batch, dev, vocab, shift, pad):
    """Rows at any 2-byte offset; what lies beside them is larger."""
    logits, uniform = rows_of(9, vocab, 11)
    wide = torch.full((9, shift + vocab + pad), 50.0, dtype=torch.bfloat16, device=dev)
    view = wide[:, shift:shift + vocab]
    view.copy_(logits)
    s = settings(9, 12)
    assert run(batch, dev, view, uniform, **s) == run(batch, dev, logits, uniform, **s)
    check(batch, dev, view, uniform, **s)


def test_frequencies(batch, dev):
    """Evenly spread random numbers give each token its share."""
    n = 4096
    row = torch.tensor([2.0, 1.0, 0.0, 1.0]).to(torch.bfloat16)
    got, _ = run(batch, dev, row.expand(n, -1).contiguous(), [(i + 0.5) / n for i in range(n)])
    p = torch.softmax(row.double(), 0)
    for t in range(4):
        assert abs(got.count(t) - float(p[t]) * n) <= 1
    assert got == sorted(got, key=lambda t: (-float(row[t]), t))


def test_captured_calls_follow_their_inputs(batch, dev):
    rows, vocab = 17, 32003
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device=dev)
    u, t = torch.empty(rows, device=dev), torch.empty(rows, device=dev)
    ws = torch.zeros(batch.sample_workspace_bytes(rows, vocab), dtype=torch.uint8, device=dev)
    tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    logits.fill_(0)
    u.fill_(0)
    t.fill_(1)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            batch.sample(logits, u, tokens, ws, temperature=t)
    for step in range(4):
        x, uniform = rows_of(rows, vocab, 20 + step)
        temps = pick([0.0, 0.5, 1.0], rows, step)
        logits.copy_(x)
        u.copy_(torch.tensor(uniform))
        t.copy_(torch.tensor(temps))
        graph.replay()
        torch.cuda.synchronize()
        first = tokens.tolist()
        assert first == check(batch, dev, x, uniform, temperature=temps)
        batch.sample(logits, u, tokens, ws, temperature=t)
        assert tokens.tolist() == first


def test_another_stream(batch, dev):
    logits, uniform = rows_of(5, 4000, 30)
    want, _ = run(batch, dev, logits, uniform)
    got, _ = run(batch, dev, logits, uniform, stream=torch.cuda.Stream())
    assert got == want


def test_a_row_past_2_32_bytes(batch, dev):
    """Three rows of a tensor of which the last begins past 2^32 elements."""
    stride, vocab = (1 << 31) + 24, 2000
    wide = torch.zeros(2 * stride + vocab, dtype=torch.bfloat16, device=dev)  # 8.6 GB
    view = wide.as_strided((3, vocab), (stride, 1))
    logits, uniform = rows_of(3, vocab, 31)
    view.copy_(logits)
    tokens = torch.empty(3, dtype=torch.int32, device=dev)
    ws = torch.zeros(batch.sample_workspace_bytes(3, vocab), dtype=torch.uint8, device=dev)
    batch.sample(view, torch.tensor(uniform).to(dev), tokens, ws)
    assert tokens.tolist() == [ref.sample(logits[i], uniform=float(torch.tensor(
        uniform[i], dtype=torch.float32)))[0] for i in range(3)]
