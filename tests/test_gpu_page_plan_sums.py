"""Sums of pages past 31 bits: which of more released pages than a list has room for are
kept, by the definition of infer_hip_kv_pages_release in Python integers."""
import pytest
import torch

from test_gpu_page_plan import ints, paged, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("last", [2 ** 30, 100, 16 * 700])
def test_more_pages_back_than_31_bits_count(paged, dev, in_place, last):  # noqa: F811
    """33 sequences of up to 2^26 pages (8.9 GB of table), all ended: 2^31 pages and more go
    back to a pool of 1000, in which the last of them come to lie."""
    n, width, page, pool, count = 33, 1 << 26, 16, 1000, 7
    table = torch.arange(width, dtype=torch.int32, device=dev).repeat(n, 1)
    table += torch.arange(n, dtype=torch.int32, device=dev)[:, None]
    lengths = [width * page] * (n - 1) + [last]
    want, place = list(range(-pool, 0)), count
    for s in reversed(range(n)):  # from the last page on, as far as there is room
        pages = -(-lengths[s] // page)
        for j in reversed(range(max(0, pages - pool), pages)):
            if place < pool:
                want[place] = j + s
                place += 1
    free, free_count = ints(range(-pool, 0), dev), ints([count], dev)
    d = ints(lengths, dev)
    out = {} if in_place else {"lengths_out": torch.empty_like(d),
                               "free_count_out": torch.empty_like(free_count)}
    paged.kv_pages_release(table, page, free, free_count, d,
                           torch.ones(n, dtype=torch.int32, device=dev),
                           workspace(paged, n, dev), **out)
    assert free.tolist() == want
    assert out.get("free_count_out", free_count).tolist() == [pool]
    assert out.get("lengths_out", d).tolist() == [0] * n
