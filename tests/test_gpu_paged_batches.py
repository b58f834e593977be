"""Attention of large batches over the paged cache: the forms that calls of more
than 64 units (a sequence's KV heads, or blocks of 16 query heads) take, with units
that are cut and joined, and with whole ones; empty sequences around the 64th."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import FORMATS, attention_case, check_attention, gen, paged, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def ragged(count, most, seed, empty):
    lengths = torch.randint(1, most + 1, (count,), generator=gen(seed)).tolist()
    lengths[count // 2] = most
    for i in empty:
        if i < count:
            lengths[i] = 0
    return lengths


AROUND_64 = (0, 61, 63, 64, 65, 100, 127, 128)


# (heads, KV heads, head_dim, page, sequences, longest): the join takes a unit a
# workgroup, its items (query heads x head_dim / 4) in two rows, one, or more than it
# has threads; from 9 tiles on where units are over 512, else from 25
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page,count,most", [
    (14, 2, 64, 16, 70, 1500), (14, 2, 64, 32, 130, 1500), (32, 8, 128, 64, 20, 1000),
    (32, 8, 128, 16, 20, 1600), (33, 1, 128, 16, 40, 1500), (16, 1, 128, 32, 70, 1300),
    (3, 1, 128, 64, 66, 900), (20, 1, 64, 16, 35, 2000), (8, 8, 64, 16, 70, 600),
    (6, 2, 64, 128, 260, 300), (5, 5, 128, 256, 110, 500), (12, 2, 128, 16, 300, 400)])
def test_cut_units_of_large_batches(paged, dev, fmt, heads, kv, d, page, count, most):
    lengths = ragged(count, most, heads + count, AROUND_64)
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, heads, kv, d, page, lengths,
                                                    count + page)
    ws = run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, d)
    again = torch.empty_like(out)
    run_attention(paged, dev, pages, table, lengths, q, again, ws)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page,count,most", [
    (32, 8, 128, 64, 40, 760), (14, 2, 64, 16, 70, 700), (4, 4, 128, 16, 128, 300),
    (24, 1, 64, 16, 66, 600), (16, 2, 128, 32, 90, 250)])
def test_whole_units_of_large_batches(paged, dev, fmt, heads, kv, d, page, count, most):
    lengths = ragged(count, most, heads + count, AROUND_64)
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, heads, kv, d, page, lengths,
                                                    count + page)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, d)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_and_empty_sequences_of_a_large_batch(paged, dev, fmt):
    """One long sequence behind 80 empty ones, and short ones behind it."""
    lengths = [0] * 80 + [9000] + [0] * 30 + [1, 33, 2000, 0, 64]
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, 14, 2, 64, 16, lengths, 8)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, 64)


def test_captured_large_batch_follows_lengths(paged, dev):
    """A captured call of 90 sequences, replayed with other lengths between eager
    calls with the same workspace."""
    heads, kv, d, page = 8, 2, 128, 32
    most = ragged(90, 1200, 5, AROUND_64)
    pool, pages, table, q, out, _ = attention_case(paged, dev, "int8", heads, kv, d, page,
                                                   [1200] * 90, 5, poison=False)
    lengths = torch.tensor(most, dtype=torch.int32, device=dev)
    ws = torch.zeros(paged.attention_paged_decode_workspace_bytes(90, heads, kv, d),
                     dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.attention_paged_decode(pages, table, lengths, q, out, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention_paged_decode(pages, table, lengths, q, out, ws)
    eager, host = torch.empty_like(out), table.cpu()
    for seed in range(4):
        step = ragged(90, (1200, 40, 700, 1)[seed], seed, AROUND_64)
        lengths.copy_(torch.tensor(step, dtype=torch.int32))
        out.fill_(5)
        graph.replay()
        paged.attention_paged_decode(pages, table, lengths, q, eager, ws)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), seed
        exact = [ref.attend(q[s].cpu(), pool.rows(0, host[s], n), pool.rows(1, host[s], n))
                 for s, n in enumerate(step)]
        check_attention(out, exact, step, d)


@pytest.mark.parametrize("fmt,count", [("bf16", 200), ("int8", 400), ("fp8", 400)])
def test_short_sequences_past_the_caches(paged, dev, fmt, count):
    """Tables of 8 tiles with room for more than 96 MiB."""
    lengths = ragged(count, 256, 6, AROUND_64)
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, 8, 4, 128, 64, lengths, count)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, 128)
