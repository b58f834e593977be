"""The paged KV cache (include/infer_paged.h) against 64-bit restatements of
its operators (tests/paged_ref.py): formats, head layouts, ragged and empty
sequences, garbage behind a length, strides, refused pages, captured graphs,
other streams, offsets past 32 bits, and a run of the three together."""
import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

FORMATS = ("bf16", "int8", "fp8")


@pytest.fixture(scope="module")
def paged():
    import paged_hip
    paged_hip.load()
    return paged_hip


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(shape, g, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def pool_bits(pages):
    out = [pages.key.view(torch.uint8), pages.value.view(torch.uint8)]
    if pages.key_scales is not None:
        out += [pages.key_scales, pages.value_scales]
    return [t.cpu().clone() for t in out]


def workspace(paged, dev, b, heads, kv, d):
    n = paged.attention_paged_decode_workspace_bytes(b, heads, kv, d)
    return torch.zeros(n, dtype=torch.uint8, device=dev)


# ------------------------------------------------------------------ store --

def check_stored(pages, fmt, i, page, slot, rows, exact):
    """Rows [kv, d] of one token: held as the FP32 rows quantise, and near the
    64-bit ones."""
    got = (pages.key, pages.value)[i]
    raw = got.view(torch.uint8)[page, :, slot].cpu() if fmt == "fp8" else got[page, :, slot].cpu()
    if fmt == "bf16":
        assert torch.equal(raw, rows.to(torch.bfloat16))
        value = raw.double()
    else:
        scale = (pages.key_scales, pages.value_scales)[i][page, :, slot].cpu()
        want = rows.abs().amax(dim=-1) / ref.LIMIT[fmt]
        assert torch.equal(scale, want)
        q = rows / torch.where(want == 0, 1.0, want)[:, None]
        if fmt == "int8":
            assert torch.equal(raw, q.round().to(torch.int8))
            value = raw.double() * scale.double()[:, None]
        else:
            assert torch.equal(raw, q.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
            value = raw.view(torch.float8_e4m3fn).float().double() * scale.double()[:, None]
    assert ((value - exact).abs() <= ref.held_error(exact, fmt) + exact.abs() * 2.0 ** -20
            + 2.0 ** -22 * exact.abs().amax()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 16), (12, 2, 128, 64), (1, 1, 64, 256),
                                             (40, 5, 128, 32)])
def test_store_rotates_and_holds(paged, dev, fmt, heads, kv, d, page):
    g = gen(heads * 100 + page)
    lengths = [37, 1, 300, 16]
    table, total = ref.tables(lengths, page, g)
    ids, positions = [], []
    for s, n in enumerate(lengths):
        for p in sorted({0, n // 2, n - 1}):
            ids.append(s)
            positions.append(p)
    order = torch.randperm(len(ids), generator=g).tolist()
    ids, positions = [ids[i] for i in order], [positions[i] for i in order]
    n = len(ids)
    rope = ref.rope_table(max(lengths), d)
    # q, k and v as column blocks of one projection's output
    qkv = bf16((n, heads + 2 * kv, d), g, 2.0)
    qkv[0, heads:] = 0  # a row of zeros has scale 0
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    pages = paged.KvPages.allocate(total, page, kv, d, fmt, dev)
    dq, dk, dv = qkv.to(dev).split([heads, kv, kv], dim=1)
    out = torch.empty((n, heads, d), dtype=torch.bfloat16, device=dev)
    paged.kv_pages_store(pages, table.to(dev), torch.tensor(positions, dtype=torch.int32, device=dev),
                         dq, dk, dv, out, rope=rope.to(dev),
                         sequences=torch.tensor(ids, dtype=torch.int32, device=dev))
    cs = rope[positions]
    exact, big = ref.rotate(q, cs)
    err = (out.cpu().double() - exact).abs()
    assert (err <= exact.abs() * 2.0 ** -8 + big * 2.0 ** -22).all()
    assert torch.equal(out.cpu(), ref.fused_free(q, cs).to(torch.bfloat16))
    k32, k64 = ref.fused_free(k, cs), ref.rotate(k, cs)[0]
    used = set()
    for t in range(n):
        where = int(table[ids[t], positions[t] // page]), positions[t] % page
        used.add(where)
        check_stored(pages, fmt, 0, *where, k32[t], k64[t])
        check_stored(pages, fmt, 1, *where, v[t].float(), v[t].double())
    # nothing else was written
    live = torch.zeros((total, page), dtype=torch.bool)
    for where in used:
        live[where] = True
    for t in pool_bits(pages)[:2]:
        assert (t.transpose(1, 2)[~live] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_store_decode_form_in_place_and_without_query(paged, dev, fmt):
    """Token i is sequence i's; the query rotated where it lies inside the
    projection's output; then the cache alone, unrotated."""
    heads, kv, d, page, n = 14, 2, 64, 16, 5
    g = gen(7)
    lengths = [3, 16, 17, 40, 1]
    table, total = ref.tables(lengths, page, g)
    positions = torch.tensor([x - 1 for x in lengths], dtype=torch.int32)
    rope = ref.rope_table(64, d)
    qkv = bf16((n, heads + 2 * kv, d), g)
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    dqkv = qkv.to(dev)
    dq, dk, dv = dqkv.split([heads, kv, kv], dim=1)
    pages = paged.KvPages.allocate(total, page, kv, d, fmt, dev)
    paged.kv_pages_store(pages, table.to(dev), positions.to(dev), dq, dk, dv, dq,
                         rope=rope.to(dev))
    cs = rope[positions.long()]
    want = torch.cat([ref.fused_free(q, cs).to(torch.bfloat16), k, v], dim=1)
    assert torch.equal(dqkv.cpu(), want)
    plain = paged.KvPages.allocate(total, page, kv, d, fmt, dev)
    paged.kv_pages_store(plain, table.to(dev), positions.to(dev), None, dk, dv)
    for t in range(n):
        where = int(table[t, int(positions[t]) // page]), int(positions[t]) % page
        check_stored(pages, fmt, 0, *where, ref.fused_free(k, cs)[t], ref.rotate(k, cs)[0][t])
        check_stored(plain, fmt, 0, *where, k[t].float(), k[t].double())
        check_stored(plain, fmt, 1, *where, v[t].float(), v[t].double())


@pytest.mark.parametrize("fmt", FORMATS)
def test_store_skips_what_has_no_place(paged, dev, fmt):
    """Padding, positions past the angles or the pages, sequences outside the
    table and pages outside the pool store nothing."""
    heads, kv, d, page = 2, 1, 64, 16
    table = torch.tensor([[0, 1], [2, 99], [-1, 3]], dtype=torch.int32)
    #        padding  past pages  past angles  bad page  bad page  no sequence      kept
    ids = [0, 0, 0, 1, 2, 3, -1, 0]
    positions = [-1, 32, 40, 17, 5, 0, 0, 31]
    g = gen(3)
    qkv = bf16((8, heads + 2 * kv, d), g)
    q, k, v = (x.to(dev) for x in qkv.split([heads, kv, kv], dim=1))
    q = q.contiguous()
    k, v = k.contiguous(), v.contiguous()
    out = torch.full_like(q, 5.0)
    pages = paged.KvPages.allocate(4, page, kv, d, fmt, dev)
    rope = ref.rope_table(40, d)
    paged.kv_pages_store(pages, table.to(dev), torch.tensor(positions, dtype=torch.int32, device=dev),
                         q, k, v, out, rope=rope.to(dev),
                         sequences=torch.tensor(ids, dtype=torch.int32, device=dev))
    for bits in pool_bits(pages):
        rest = bits.clone()
        rest[1, 0, 15] = 0
        assert (rest == 0).all()
    assert (pages.value[1, 0, 15].view(torch.uint8).cpu() != 0).any()
    # queries: those with an angle are rotated, the others left as they were
    cs = rope[[max(0, min(p, 39)) for p in positions]]
    want = ref.fused_free(q.cpu(), cs).to(torch.bfloat16)
    want[0] = want[2] = 5.0
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_rows_that_are_not_finite_read_as_nan(paged, dev, fmt):
    kv, d, page = 2, 64, 16
    k = torch.ones((3, kv, d), dtype=torch.bfloat16)
    k[0, 0, 5], k[1, 1, 63], k[2, 0, 0] = math.inf, math.nan, -math.inf
    pages = paged.KvPages.allocate(1, page, kv, d, fmt, dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    paged.kv_pages_store(pages, table, torch.arange(3, dtype=torch.int32, device=dev), None,
                         k.to(dev), torch.ones_like(k).to(dev),
                         sequences=torch.zeros(3, dtype=torch.int32, device=dev))
    kc = torch.zeros((1, kv, 3, d), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    paged.kv_pages_load(pages, table, torch.tensor([3], dtype=torch.int32, device=dev), kc, vc)
    nan = torch.tensor([[True, False, True], [False, True, False]])
    assert torch.equal(kc[0].isnan().all(dim=-1).cpu(), nan)
    assert torch.equal(kc[0].isnan().any(dim=-1).cpu(), nan)
    assert (kc[0].cpu()[~nan] == 1).all() and (vc == 1).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("size", [3.0e38, 1.2e-38, 2.0e-40])
def test_extreme_rows_stay_in_range(paged, dev, fmt, size):
    """Near the ends of BF16's range, the scale itself subnormal at the lowest:
    an element stays within half a step, or within one of the scale's own
    (2^-149 x the format's limit)."""
    g = gen(11)
    k = (torch.rand((4, 1, 128), generator=g) * 2 - 1).mul(size).to(torch.bfloat16)
    pages = paged.KvPages.allocate(1, 16, 1, 128, fmt, dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    paged.kv_pages_store(pages, table, torch.arange(4, dtype=torch.int32, device=dev), None,
                         k.to(dev), k.to(dev),
                         sequences=torch.zeros(4, dtype=torch.int32, device=dev))
    scale = pages.key_scales[0, 0, :4].cpu().double()
    q = pages.key.cpu().view(torch.uint8 if fmt == "fp8" else torch.int8)[0, 0, :4]
    q = (q.view(torch.float8_e4m3fn) if fmt == "fp8" else q).float().double()
    value, exact = q * scale[:, None], k[:, 0].double()
    assert ((value - exact).abs() <= ref.held_error(exact, fmt)
            + ref.LIMIT[fmt] * 2.0 ** -149).all()


# ------------------------------------------------------------------- load --

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv,d,page,capacity", [(2, 64, 16, 70), (3, 128, 64, 257), (1, 64, 256, 1)])
def test_load_reads_back(paged, dev, fmt, kv, d, page, capacity):
    g = gen(kv + page)
    lengths = [0, 1, capacity, 16, -3, capacity + 40, 15, 17]
    table, total = ref.tables(lengths, page, g)
    pool = ref.Pool(fmt, total, page, kv, d, g)
    pages = pool.to_device(paged, dev)
    kc = torch.full((len(lengths), kv, capacity, d), 9.0, dtype=torch.bfloat16, device=dev)
    vc = torch.full_like(kc, -9.0)
    paged.kv_pages_load(pages, table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev),
                        kc, vc)
    for s, n in enumerate(lengths):
        n = max(0, min(n, capacity))
        for i, (c, fill) in enumerate(((kc, 9.0), (vc, -9.0))):
            got, exact = c[s].cpu(), pool.rows(i, table[s], n)
            assert ((got[:, :n].double() - exact).abs() <= exact.abs() * 2.0 ** -8).all()
            assert (got[:, n:] == fill).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv,d,capacity", [(1, 64, 400003), (2, 128, 100001)])
def test_load_of_much(paged, dev, fmt, kv, d, capacity):
    """Outputs past 96 MiB, of which little is live."""
    page, g, lengths = 64, gen(d), [1, 700, 0, 65]
    table, total = ref.tables(lengths, page, g, width=-(-capacity // page))
    pool = ref.Pool(fmt, total, page, kv, d, g)
    kc = torch.full((len(lengths), kv, capacity, d), 3.0, dtype=torch.bfloat16, device=dev)
    vc = kc.clone()
    paged.kv_pages_load(pool.to_device(paged, dev), table.to(dev),
                        torch.tensor(lengths, dtype=torch.int32, device=dev), kc, vc)
    for i, cache in enumerate((kc, vc)):
        for s, n in enumerate(lengths):
            exact = pool.rows(i, table[s], n)
            assert ((cache[s, :, :n].cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -8).all()
            assert bool((cache[s, :, n:] == 3.0).all())


def test_load_ends_with_the_table_and_marks_bad_pages(paged, dev):
    g = gen(5)
    pool = ref.Pool("int8", 4, 16, 1, 64, g)
    pages = pool.to_device(paged, dev)
    wide = torch.tensor([[0, 1, 2], [3, 7, -5]], dtype=torch.int32, device=dev)
    kc = torch.full((2, 1, 48, 64), 3.0, dtype=torch.bfloat16, device=dev)
    vc = kc.clone()
    paged.kv_pages_load(pages, wide[:, :2], torch.tensor([48, 20], dtype=torch.int32, device=dev),
                        kc, vc)
    got = kc.cpu()
    assert torch.equal(got[0, :, :32], pool.rows(0, [0, 1], 32).to(torch.bfloat16))
    assert (got[0, :, 32:] == 3).all()
    assert torch.equal(got[1, :, :16], pool.rows(0, [3], 16).to(torch.bfloat16))
    assert got[1, :, 16:20].isnan().all() and (got[1, :, 20:] == 3).all()


# -------------------------------------------------------------- attention --

def attention_case(paged, dev, fmt, heads, kv, d, page, lengths, seed, std=1.0, qstd=1.0,
                   poison=True, width=None):
    g = gen(seed)
    table, total = ref.tables(lengths, page, g, width=width)
    pool = ref.Pool(fmt, total, page, kv, d, g, std)
    q = bf16((len(lengths), heads, d), g, qstd)
    out64 = [ref.attend(q[s], pool.rows(0, table[s], n), pool.rows(1, table[s], n))
             for s, n in enumerate(lengths)]
    pages = pool.to_device(paged, dev)
    if poison:  # what no sequence holds must not count
        live = torch.zeros((total, page), dtype=torch.bool)
        for s, n in enumerate(lengths):
            for p in range(max(0, n)):
                live[int(table[s, p // page]), p % page] = True
        dead = (~live).to(dev)
        for t, s in ((pages.key, pages.key_scales), (pages.value, pages.value_scales)):
            if s is None:
                t.transpose(1, 2)[dead] = math.nan
            else:
                s.transpose(1, 2)[dead] = math.nan
                t.view(torch.uint8).transpose(1, 2)[dead] = 0x7F
    out = torch.full((len(lengths), heads, d), 7.0, dtype=torch.bfloat16, device=dev)
    return pool, pages, table.to(dev), q.to(dev), out, out64


def check_attention(out, out64, lengths, d):
    for s, (exact, mean_abs, big) in enumerate(out64):
        got = out[s].cpu().double()
        tol = ref.attend_tolerance(exact, mean_abs, big, max(lengths[s], 0), d)
        bad = ~((got - exact).abs() <= tol)
        assert not bad.any(), (s, lengths[s], float((got - exact).abs().max()), int(bad.sum()))


def run_attention(paged, dev, pages, table, lengths, q, out, ws=None):
    if ws is None:
        ws = workspace(paged, dev, q.shape[0], q.shape[1], pages.num_kv_heads, pages.head_dim)
    paged.attention_paged_decode(pages, table, torch.tensor(lengths, dtype=torch.int32, device=dev),
                                 q, out, ws)
    return ws


RAGGED = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 127, 128, 129, 255, 257, 500, -1]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 16), (12, 2, 128, 16), (8, 8, 64, 32),
                                             (32, 8, 128, 64), (16, 1, 128, 128), (24, 1, 64, 256),
                                             (33, 1, 128, 16), (3, 3, 128, 256)])
def test_attention_of_ragged_sequences(paged, dev, fmt, heads, kv, d, page):
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, heads, kv, d, page, RAGGED,
                                                    heads + page)
    ws = run_attention(paged, dev, pages, table, RAGGED, q, out)
    check_attention(out, out64, RAGGED, d)
    again = torch.empty_like(out)
    run_attention(paged, dev, pages, table, RAGGED, q, again, ws)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page,lengths", [
    (14, 2, 64, 16, [20011]), (12, 2, 128, 64, [33000]), (28, 4, 128, 32, [5000, 3]),
    (8, 8, 64, 256, [9001, 1, 4096, 0]), (6, 1, 128, 16, [1]), (14, 2, 64, 16, [1]),
    (20, 1, 64, 128, [7777, 300])])
def test_attention_split_over_long_sequences(paged, dev, fmt, heads, kv, d, page, lengths):
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, heads, kv, d, page, lengths,
                                                    len(lengths) + page)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, d)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,d,page", [(7, 1, 64, 16), (28, 4, 128, 32), (16, 1, 64, 64),
                                             (24, 2, 128, 16), (40, 2, 64, 128)])
def test_attention_of_tables_with_much_room(paged, dev, fmt, heads, kv, d, page):
    """Short and long sequences under tables for 400000 positions each."""
    lengths = [1, 5000, 0, 33, 1200]
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, heads, kv, d, page, lengths,
                                                    heads + d, width=400000 // page)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, d)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("count", [64, 65, 300, 1500])
def test_attention_of_many_sequences(paged, dev, fmt, count):
    rng = gen(count)
    lengths = torch.randint(0, 90, (count,), generator=rng).tolist()
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, 4, 2, 64, 16, lengths, count)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, 64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_of_far_apart_scores(paged, dev, fmt):
    """Scores up to several hundred apart, so that every weight but a few
    vanishes and the running maximum climbs."""
    lengths = [600, 129, 40]
    _, pages, table, q, out, out64 = attention_case(paged, dev, fmt, 14, 2, 64, 16, lengths, 21,
                                                    std=3.0, qstd=12.0)
    run_attention(paged, dev, pages, table, lengths, q, out)
    check_attention(out, out64, lengths, 64)


def test_attention_scores_below_exponents_range(paged, dev):
    """Every score near -30000: only their differences count."""
    d, n, page = 64, 200, 16
    g = gen(2)
    table, total = ref.tables([n], page, g)
    pool = ref.Pool("bf16", total, page, 1, d, g)
    pool.parts[0][:] = -60.0
    pool.parts[0][..., 0] = (torch.randn(pool.parts[0].shape[:3], generator=g)).to(torch.bfloat16)
    q = torch.full((1, 2, d), 64.0, dtype=torch.bfloat16)
    q[..., 0] = 4.0
    exact = ref.attend(q[0], pool.rows(0, table[0], n), pool.rows(1, table[0], n))
    pages, out = pool.to_device(paged, dev), torch.empty((1, 2, d), dtype=torch.bfloat16, device=dev)
    run_attention(paged, dev, pages, table.to(dev), [n], q.to(dev), out)
    check_attention(out, [exact], [n], d)


def test_attention_bad_pages_give_nan_and_lengths_end_with_the_table(paged, dev):
    heads, kv, d, page = 4, 2, 64, 16
    g = gen(9)
    pool = ref.Pool("int8", 6, page, kv, d, g)
    table = torch.tensor([[0, 1], [2, 77], [-1, 3], [4, 5], [3, -2]], dtype=torch.int32)
    lengths = [1000, 17, 32, 32, 16]  # past the table, two bad ones, whole, bad one not reached
    q = bf16((5, heads, d), g)
    pages, out = pool.to_device(paged, dev), torch.zeros((5, heads, d), dtype=torch.bfloat16,
                                                          device=dev)
    run_attention(paged, dev, pages, table.to(dev), lengths, q.to(dev), out)
    assert out[1].isnan().all() and out[2].isnan().all()
    for s, n in ((0, 32), (3, 32), (4, 16)):
        exact = ref.attend(q[s], pool.rows(0, table[s], n), pool.rows(1, table[s], n))
        check_attention(out[s:s + 1], [exact], [n], d)


def test_attention_infinite_scores(paged, dev):
    """Scores of -inf have no weight; of all -inf, or one +inf, the result is NaN."""
    d, page = 64, 16
    g = gen(8)
    table, total = ref.tables([40, 40, 40], page, g)
    pool = ref.Pool("bf16", total, page, 1, d, g)
    for s, rows, value in ((0, (3, 17, 39), -math.inf), (1, range(40), -math.inf),
                           (2, (20,), math.inf)):
        for p in rows:
            pool.parts[0][int(table[s, p // page]), 0, p % page, 5] = value
    q = bf16((3, 2, d), g)
    q[..., 5] = 1.0
    pages, out = pool.to_device(paged, dev), torch.empty((3, 2, d), dtype=torch.bfloat16, device=dev)
    run_attention(paged, dev, pages, table.to(dev), [40, 40, 40], q.to(dev), out)
    keep = [p for p in range(40) if p not in (3, 17, 39)]
    exact = ref.attend(q[0], pool.rows(0, table[0], 40)[:, keep], pool.rows(1, table[0], 40)[:, keep])
    check_attention(out[:1], [exact], [37], d)
    assert out[1:].isnan().all()


@pytest.mark.parametrize("where", ["query", "key", "value"])
def test_attention_nan_stays_in_its_sequence(paged, dev, where):
    lengths = [100, 700, 64]
    _, pages, table, q, out, out64 = attention_case(paged, dev, "bf16", 4, 2, 64, 16, lengths, 13)
    if where == "query":
        q[1] = math.nan
    else:
        t = pages.key if where == "key" else pages.value
        t[int(table[1, 650 // 16]), :, 650 % 16] = math.nan
    run_attention(paged, dev, pages, table, lengths, q, out)
    assert out[1].isnan().all()
    check_attention(out[0::2], out64[0::2], lengths[0::2], 64)


def test_attention_strided_query_and_table_slice(paged, dev):
    heads, kv, d, page = 6, 2, 128, 32
    lengths = [40, 333, 96]
    _, pages, table, q, out, out64 = attention_case(paged, dev, "fp8", heads, kv, d, page, lengths, 4)
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    qkv = torch.full((3, heads + 2 * kv, d), math.nan, dtype=torch.bfloat16, device=dev)
    qkv[:, :heads] = q
    run_attention(paged, dev, pages, wide[:, :table.shape[1]], lengths, qkv[:, :heads], out)
    check_attention(out, out64, lengths, d)


def test_attention_captured_once_follows_lengths(paged, dev):
    """One captured graph, replayed while lengths grow and shrink, between eager
    calls that share its workspace in turn."""
    heads, kv, d, page = 14, 2, 64, 16
    most = [3000, 41, 700]
    g = gen(17)
    pool, pages, table, q, out, _ = attention_case(paged, dev, "int8", heads, kv, d, page, most, 17,
                                                   poison=False)
    ws = workspace(paged, dev, 3, heads, kv, d)
    lengths = torch.tensor(most, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.attention_paged_decode(pages, table, lengths, q, out, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention_paged_decode(pages, table, lengths, q, out, ws)
    eager = torch.empty_like(out)
    host = table.cpu()
    for step in ([3000, 41, 700], [1, 0, 699], [2999, 40, 33], [64, 41, 512], [0, 0, 0]):
        lengths.copy_(torch.tensor(step, dtype=torch.int32))
        out.fill_(5)
        graph.replay()
        paged.attention_paged_decode(pages, table, lengths, q, eager, ws)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), step
        exact = [ref.attend(q[s].cpu(), pool.rows(0, host[s], n), pool.rows(1, host[s], n))
                 for s, n in enumerate(step)]
        check_attention(out, exact, step, d)


def test_attention_on_other_streams_with_their_own_workspaces(paged, dev):
    lengths = [900, 64]
    cases = [attention_case(paged, dev, f, 14, 2, 64, 16, lengths, 30 + i)
             for i, f in enumerate(FORMATS)]
    ws = [workspace(paged, dev, 2, 14, 2, 64) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    for _ in range(20):
        for (_, pages, table, q, out, _), w, s in zip(cases, ws, streams):
            paged.attention_paged_decode(pages, table, n, q, out, w, stream=s)
    torch.cuda.synchronize()
    for _, _, _, _, out, out64 in cases:
        check_attention(out, out64, lengths, 64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(paged, dev, fmt):
    """A pool whose last pages lie past 2^32 bytes: stored, loaded, attended."""
    kv, d, page, heads = 8, 128, 256, 16
    size = kv * page * d * (2 if fmt == "bf16" else 1)
    total = (1 << 32) // size + 8
    dtype = ref.DTYPE[fmt]
    raw = [torch.empty(total * size, dtype=torch.uint8, device=dev).view(dtype).view(
        total, kv, page, d) for _ in range(2)]
    sc = [None if fmt == "bf16" else torch.empty((total, kv, page), device=dev) for _ in range(2)]
    pages = paged.KvPages(*raw, *sc)
    n = 300
    table = torch.tensor([[total - 1, total - 3]], dtype=torch.int32)
    g = gen(1)
    k, v = bf16((n, kv, d), g), bf16((n, kv, d), g)
    paged.kv_pages_store(pages, table.to(dev), torch.arange(n, dtype=torch.int32, device=dev), None,
                         k.to(dev), v.to(dev), sequences=torch.zeros(n, dtype=torch.int32, device=dev))
    kc = torch.empty((1, kv, n, d), dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    paged.kv_pages_load(pages, table.to(dev), torch.tensor([n], dtype=torch.int32, device=dev), kc, vc)
    for got, rows in ((kc, k), (vc, v)):
        exact = rows.double().transpose(0, 1)
        tol = ref.held_error(exact, fmt) * (1 + 2.0 ** -8) + exact.abs() * 2.0 ** -8
        assert ((got[0].cpu().double() - exact).abs() <= tol).all()
    q = bf16((1, heads, d), g)
    out = torch.empty((1, heads, d), dtype=torch.bfloat16, device=dev)
    run_attention(paged, dev, pages, table.to(dev), [n], q.to(dev), out)
    # over the rows as they were read back: within 2^-8 of the held values
    exact = ref.attend(q[0], kc[0].cpu().double(), vc[0].cpu().double())
    if fmt == "bf16":
        check_attention(out, [exact], [n], d)
    else:  # the read-back's own rounding moves scores by 2^-8 sum |q k|, values by 2^-8
        tol = ref.attend_tolerance(*exact, n, d) + exact[1] * (2 * 2.0 ** -8 * exact[2] + 2.0 ** -8)
        assert ((out[0].cpu().double() - exact[0]).abs() <= tol).all()


# --------------------------------------------------------------- together --

@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_then_decode_steps(paged, dev, fmt):
    """Two prompts written to pages and read back give the prefill attention of
    the contiguous operator; then decode steps, each storing its token and
    attending, captured once and replayed."""
    import model_hip
    heads, kv, d, page = 14, 2, 64, 16
    prompts, steps = [45, 16], 5
    g = gen(40)
    most = [n + steps for n in prompts]
    table, total = ref.tables(most, page, g)
    table = table.to(dev)
    pages = paged.KvPages.allocate(total, page, kv, d, fmt, dev)
    rope = ref.rope_table(max(most), d)
    drope = rope.to(dev)
    ids = torch.tensor([i for i, n in enumerate(prompts) for _ in range(n)], dtype=torch.int32)
    positions = torch.tensor([p for n in prompts for p in range(n)], dtype=torch.int32)
    qkv = bf16((len(ids), heads + 2 * kv, d), g).to(dev)
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    rq = torch.empty((len(ids), heads, d), dtype=torch.bfloat16, device=dev)
    paged.kv_pages_store(pages, table, positions.to(dev), q, k, v, rq, rope=drope,
                         sequences=ids.to(dev))
    capacity = max(most)
    kc = torch.zeros((2, kv, capacity, d), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    paged.kv_pages_load(pages, table, lengths, kc, vc)
    ws = workspace(paged, dev, 2, heads, kv, d)
    at = 0
    for s, n in enumerate(prompts):
        mine = rq[at:at + n].contiguous()
        out = torch.empty_like(mine)
        model_hip.attention_prefill_bf16(mine, kc[s], vc[s], out, n, heads, kv, d, capacity)
        # the prompt's last row is the one-token attention over its pages
        got = torch.empty((2, heads, d), dtype=torch.bfloat16, device=dev)
        both = torch.stack([mine[-1], mine[-1]])
        only = torch.tensor([n if i == s else 0 for i in range(2)], dtype=torch.int32, device=dev)
        paged.attention_paged_decode(pages, table, only, both, got, ws)
        exact = ref.attend(mine[-1].cpu(), kc[s, :, :n].cpu().double(), vc[s, :, :n].cpu().double())
        tol = ref.attend_tolerance(*exact, n, d)
        # the pages' values before the read-back's rounding, in the 8-bit formats
        slack = 0 if fmt == "bf16" else exact[1] * (2 * 2.0 ** -8 * exact[2] + 2.0 ** -8)
        assert ((got[s].cpu().double() - exact[0]).abs() <= tol + slack).all()
        assert ((out[-1].cpu().double() - exact[0]).abs() <= tol).all()
        assert (got[1 - s] == 0).all()
        at += n
    # decode: token, position and length in fixed buffers, one captured step
    step_qkv = torch.empty((2, heads + 2 * kv, d), dtype=torch.bfloat16, device=dev)
    pos, out = lengths.clone(), torch.empty((2, heads, d), dtype=torch.bfloat16, device=dev)
    sq, sk, sv = step_qkv.split([heads, kv, kv], dim=1)

    def step():
        paged.kv_pages_store(pages, table, pos, sq, sk, sv, sq, rope=drope)
        lengths.add_(1)
        paged.attention_paged_decode(pages, table, lengths, sq, out, ws)
        pos.add_(1)

    warm = torch.cuda.Stream()
    step_qkv.zero_()
    keep = pos.clone(), lengths.clone()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    pos.copy_(keep[0])
    lengths.copy_(keep[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    pos.copy_(keep[0])
    lengths.copy_(keep[1])
    for i in range(steps):
        new = bf16((2, heads + 2 * kv, d), g)
        step_qkv.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for s in range(2):
            n = prompts[s] + i + 1
            one_k = torch.zeros((2, kv, n, d), dtype=torch.bfloat16, device=dev)
            one_v = torch.zeros_like(one_k)
            paged.kv_pages_load(pages, table, torch.tensor([n, n], dtype=torch.int32, device=dev),
                                one_k, one_v)
            cs = rope[n - 1:n]
            turned = ref.fused_free(new[s:s + 1, :heads], cs).to(torch.bfloat16)[0]
            assert torch.equal(step_qkv[s, :heads].cpu(), turned)
            last = ref.rotate(new[s:s + 1, heads:heads + kv], cs)[0][0]
            err = (one_k[s, :, n - 1].cpu().double() - last).abs()
            assert (err <= ref.held_error(last, fmt) * (1 + 2.0 ** -8) + last.abs() * 2.0 ** -8
                    + last.abs().amax() * 2.0 ** -20).all()
            exact = ref.attend(turned, one_k[s].cpu().double(), one_v[s].cpu().double())
            tol = ref.attend_tolerance(*exact, n, d)
            slack = 0 if fmt == "bf16" else exact[1] * (2 * 2.0 ** -8 * exact[2] + 2.0 ** -8)
            assert ((out[s].cpu().double() - exact[0]).abs() <= tol + slack).all()
