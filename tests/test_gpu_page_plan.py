"""Pages of a step (infer_hip_kv_pages_assign, infer_hip_kv_pages_release) against
their definition in Python integers (tests/plan_ref.py): forms, sizes around the
launches' shapes, pools that run out, lengths past the table, padding, bad pages,
buffers in place, captured graphs, and another stream."""
import pytest
import torch

import plan_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    import paged_hip
    paged_hip.load()
    return paged_hip


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32).to(dev)


def workspace(paged, n, dev):
    # what a workspace holds before a call must not matter
    return torch.full((paged.kv_pages_plan_workspace_bytes(n),), 255, dtype=torch.uint8,
                      device=dev)


def state(table, free, count, lengths, dev):
    return {"table": ints(table, dev), "free": ints(free, dev), "free_count": ints([count], dev),
            "lengths": ints(lengths, dev)}


def check_assign(paged, dev, page, table, free, count, lengths, added, tokens, packed,
                 in_place=False, extras=True, stream=None):
    n = len(lengths)
    want = ref.assign(table, page, free, count, lengths, added, tokens, packed)
    s = state(table, free, count, lengths, dev)
    guard = 77  # behind each output
    positions = torch.full((tokens + 4,), guard, dtype=torch.int32, device=dev)
    ids, slots = torch.full_like(positions, guard), torch.full_like(positions, guard).long()
    starts = torch.full((n + 3,), guard, dtype=torch.int32, device=dev)
    lengths_out = s["lengths"] if in_place else torch.full_like(s["lengths"], guard)
    count_out = s["free_count"] if in_place else torch.full_like(s["free_count"], guard)
    more, ws = ints(added, dev), workspace(paged, n, dev)
    torch.cuda.synchronize()
    paged.kv_pages_assign(
        s["table"], page, s["free"], s["free_count"], s["lengths"], more, ws, positions[:tokens],
        sequences=ids[:tokens] if packed else None, slots=slots[:tokens] if extras else None,
        starts=starts[:n + 1] if packed and extras else None, lengths_out=lengths_out,
        free_count_out=count_out, stream=stream)
    torch.cuda.synchronize()
    assert positions[:tokens].tolist() == want["positions"]
    assert positions[tokens:].tolist() == [guard] * 4
    if packed:
        assert ids[:tokens].tolist() == want["sequences"]
        assert ids[tokens:].tolist() == [guard] * 4
    if extras:
        assert slots[:tokens].tolist() == want["slots"]
        assert slots[tokens:].tolist() == [guard] * 4
        if packed:
            assert starts.tolist() == want["starts"] + [guard] * 2
    assert s["table"].tolist() == want["table"]
    assert lengths_out.tolist() == want["lengths"]
    assert count_out.tolist() == [want["free_count"]]
    assert s["free"].tolist() == list(free)
    return want


def case(n, longest, page, form, seed, share=1.0):
    """(table, free, count, lengths, added) of n sequences."""
    g = gen(seed)
    lengths = torch.randint(0, longest, (n,), generator=g).tolist()
    if form == "decode":
        added = (torch.rand(n, generator=g) < 0.8).int().tolist()
    else:
        added = torch.randint(0, longest, (n,), generator=g).tolist()
        for i in range(0, n, 3):  # prompts from nothing, and idle sequences
            lengths[i] = 0
        for i in range(1, n, 5):
            added[i] = 0
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(lengths, added))
    width = -(-2 * longest // page) + 1
    unused = int(need * share) + (4 if share >= 1 else 0)
    table, free = ref.deal(lengths, page, width, unused, g)
    return table, free, unused, lengths, added


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,longest,page", [(1, 40, 16), (24, 1000, 16), (255, 90, 32),
                                            (1024, 64, 64), (1025, 300, 128), (3001, 50, 256)])
def test_decode_form(paged, dev, n, longest, page, in_place):
    table, free, count, lengths, added = case(n, longest, page, "decode", n)
    check_assign(paged, dev, page, table, free, count, lengths, added, n, False, in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,longest,page,pad", [
    (1, 1, 16, 0), (1, 5000, 16, 3), (3, 17, 16, 0), (8, 3000, 32, 13), (64, 70, 64, 1),
    (300, 40, 16, 5), (300, 900, 16, 5), (200, 2000, 32, 0), (257, 3, 16, 1), (1023, 9, 256, 0), (2048, 12, 128, 7), (2049, 12, 16, 2), (5000, 6, 16, 0)])
def test_packed_form(paged, dev, n, longest, page, pad, in_place):
    table, free, count, lengths, added = case(n, longest, page, "packed", n + longest)
    check_assign(paged, dev, page, table, free, count, lengths, added, max(1, sum(added)) + pad,
                 True, in_place)


@pytest.mark.parametrize("n,form,share", [(40, "decode", 0.5), (40, "packed", 0.5),
                                          (2500, "packed", 0.3), (30, "packed", 0.0),
                                          (1500, "decode", 0.7)])
def test_a_pool_that_runs_out_serves_in_order(paged, dev, n, form, share):
    table, free, count, lengths, added = case(n, 100, 16, form, n, share)
    tokens = n if form == "decode" else sum(added) + 2
    want = check_assign(paged, dev, 16, table, free, count, lengths, added, tokens,
                        form == "packed")
    assert want["lengths"] != [a + b for a, b in zip(lengths, added)]


def test_what_does_not_fit_is_not_served(paged, dev):
    # a table of 4 pages of 16: past it, negative, of no use in the decode form, and
    # the largest numbers there are
    top = 2 ** 31 - 1
    lengths = [64, 60, 63, -5, 0, 70, top, 16, -top - 1]
    added = [1, 4, 2, 3, top, 0, top, -7, 1]
    held = [max(0, min(n, 64)) for n in lengths]
    table, free = ref.deal(held, 16, 4, 9, gen(1))
    for tokens in (5, 9, 40):
        check_assign(paged, dev, 16, table, free, 9, lengths, added, tokens, True)
    check_assign(paged, dev, 16, table, free, 9, lengths, added, 9, False)


@pytest.mark.parametrize("tokens", [1, 49, 50, 51, 100, 149, 150])
def test_tokens_that_end_past_the_room(paged, dev, tokens):
    lengths, added = [5, 0, 100, 0, 3], [50, 0, 50, 0, 50]
    table, free = ref.deal(lengths, 16, 12, 20, gen(2))
    check_assign(paged, dev, 16, table, free, 20, lengths, added, tokens, True)


@pytest.mark.parametrize("count", [-3, 0, 1, 11, 500])
def test_counts_outside_the_pool(paged, dev, count):
    table, free = ref.deal([3, 0], 16, 8, 6, gen(3))
    check_assign(paged, dev, 16, table, free, count, [3, 0], [20, 40], 64, True)


def test_pages_outside_the_pool_have_no_slots(paged, dev):
    table, free = ref.deal([40, 16, 0], 16, 8, 6, gen(4))
    table[0][2], table[1][0], free[4] = -1, 10 ** 9, -8
    check_assign(paged, dev, 16, table, free, 6, [40, 16, 0], [30, 30, 30], 90, True)


def test_optional_outputs_and_unaligned_ones(paged, dev):
    table, free, count, lengths, added = case(9, 60, 16, "packed", 5)
    check_assign(paged, dev, 16, table, free, count, lengths, added, sum(added), True,
                 extras=False)
    want = ref.assign(table, 16, free, count, lengths, added, sum(added), True)
    s, n = state(table, free, count, lengths, dev), sum(added)
    a, b = (torch.zeros(n + 1, dtype=torch.int32, device=dev)[1:] for _ in range(2))
    c = torch.zeros(n + 1, dtype=torch.int64, device=dev)[1:]
    paged.kv_pages_assign(s["table"], 16, s["free"], s["free_count"], s["lengths"],
                          ints(added, dev), workspace(paged, 9, dev), a, sequences=b, slots=c)
    assert a.tolist() == want["positions"] and b.tolist() == want["sequences"]
    assert c.tolist() == want["slots"] and s["lengths"].tolist() == want["lengths"]


def test_a_slice_of_a_wider_table(paged, dev):
    table, free, count, lengths, added = case(7, 40, 16, "packed", 6)
    want = ref.assign(table, 16, free, count, lengths, added, sum(added), True)
    s, width = state(table, free, count, lengths, dev), len(table[0])
    wide = torch.full((7, width + 5), 99, dtype=torch.int32, device=dev)
    wide[:, :width] = s["table"]
    positions = torch.empty(sum(added), dtype=torch.int32, device=dev)
    paged.kv_pages_assign(wide[:, :width], 16, s["free"], s["free_count"], s["lengths"],
                          ints(added, dev), workspace(paged, 7, dev), positions,
                          sequences=torch.empty_like(positions))
    assert wide[:, :width].tolist() == want["table"] and (wide[:, width:] == 99).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,longest,page", [(1, 0, 16), (1, 1, 16), (3, 50, 16), (64, 4000, 16),
                                            (1024, 200, 128), (2100, 90, 32), (5, 100000, 16), (4096, 30, 16),
                                            (4097, 30, 16)])
def test_release(paged, dev, n, longest, page, in_place):
    g = gen(n)
    lengths = torch.randint(0, longest + 1, (n,), generator=g).tolist()
    finished = torch.randint(0, 2, (n,), generator=g).tolist()
    finished[0] = -4  # any number that is not 0
    table, free = ref.deal(lengths, page, max(1, -(-longest // page)), 11, g)
    want = ref.release(table, page, free, 11, lengths, finished)
    s = state(table, free, 11, lengths, dev)
    out = {} if in_place else {"lengths_out": torch.empty_like(s["lengths"]),
                               "free_count_out": torch.empty_like(s["free_count"])}
    paged.kv_pages_release(s["table"], page, s["free"], s["free_count"], s["lengths"],
                           ints(finished, dev), workspace(paged, n, dev), **out)
    assert s["free"].tolist() == want["free"] and s["table"].tolist() == table
    assert out.get("lengths_out", s["lengths"]).tolist() == want["lengths"]
    assert out.get("free_count_out", s["free_count"]).tolist() == [want["free_count"]]


def test_release_of_lengths_and_counts_that_cannot_be(paged, dev):
    top = 2 ** 31 - 1
    lengths, finished = [-3, 70, top, 16], [1, 1, 1, 0]
    table = [[1, 2, 3, 4], [5, 6, 7, 0], [4, 3, 2, 1], [0, 0, 0, 0]]
    for count in (-1, 0, 3, 9):
        free = [9, 9, 9, -1, -1, -1, -1, -1]
        want = ref.release(table, 16, free, count, lengths, finished)
        s = state(table, free, count, lengths, dev)
        paged.kv_pages_release(s["table"], 16, s["free"], s["free_count"], s["lengths"],
                               ints(finished, dev), workspace(paged, 4, dev))
        assert s["free"].tolist() == want["free"]
        assert s["free_count"].tolist() == [want["free_count"]]
        assert s["lengths"].tolist() == want["lengths"]


def test_release_restores_what_was_assigned(paged, dev):
    table, free, count, _, added = case(50, 200, 16, "packed", 9)
    lengths = [0] * 50
    table = [[-1] * len(table[0]) for _ in table]
    need = sum(-(-a // 16) for a in added)
    free = torch.randperm(need + 3, generator=gen(10)).tolist()
    s, ws = state(table, free, need + 3, lengths, dev), workspace(paged, 50, dev)
    positions = torch.empty(sum(added), dtype=torch.int32, device=dev)
    args = (s["table"], 16, s["free"], s["free_count"], s["lengths"])
    for _ in range(3):
        paged.kv_pages_assign(*args, ints(added, dev), ws, positions,
                              sequences=torch.empty_like(positions))
        assert s["lengths"].tolist() == added and s["free_count"].tolist() == [3]
        paged.kv_pages_release(*args, torch.ones(50, dtype=torch.int32, device=dev), ws)
        assert s["free"].tolist() == free and s["free_count"].tolist() == [need + 3]


def test_captured_steps_follow_the_state(paged, dev):
    """A captured step grows its sequences in place, replay by replay, with eager
    work between."""
    n, page, steps = 40, 16, 40
    lengths = list(range(n))
    table, free = ref.deal(lengths, page, 8, 200, gen(11))
    s, ws = state(table, free, 200, lengths, dev), workspace(paged, n, dev)
    added = ints([1] * n, dev)
    positions = torch.empty(n, dtype=torch.int32, device=dev)
    slots = torch.empty(n, dtype=torch.int64, device=dev)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            paged.kv_pages_assign(s["table"], page, s["free"], s["free_count"], s["lengths"],
                                  added, ws, positions, slots=slots)
    count = 200
    for step in range(steps):
        more = [int((step + i) % 4 != 0) for i in range(n)]
        added.copy_(ints(more, dev))
        want = ref.assign(table, page, free, count, lengths, more, n, False)
        graph.replay()
        torch.cuda.synchronize()
        assert positions.tolist() == want["positions"] and slots.tolist() == want["slots"]
        table, lengths, count = want["table"], want["lengths"], want["free_count"]
        assert s["table"].tolist() == table and s["lengths"].tolist() == lengths
        assert s["free_count"].tolist() == [count]


def test_another_stream(paged, dev):
    table, free, count, lengths, added = case(30, 300, 16, "packed", 12)
    stream = torch.cuda.Stream()
    check_assign(paged, dev, 16, table, free, count, lengths, added, sum(added), True,
                 stream=stream)


def test_the_largest_batch(paged, dev):
    n = 65535
    table, free, count, lengths, added = case(n, 8, 16, "decode", 13)
    check_assign(paged, dev, 16, table, free, count, lengths, added, n, False)
    added = [int(i % 7 == 0) * 3 for i in range(n)]
    check_assign(paged, dev, 16, table, free, count, lengths, added, sum(added) + 5, True)
