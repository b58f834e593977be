"""Pages of a step from their definition, in Python integers: what
tests/test_gpu_page_plan.py compares the kernels with."""
import torch


def assign(table, page, free, count, lengths, added, tokens, packed):
    """Lists in, a dict of lists out; table is changed in a copy."""
    table = [list(row) for row in table]
    room, pages = len(table[0]) * page, len(free)
    count = min(max(count, 0), pages)
    out = {"positions": [-1] * tokens, "sequences": [-1] * tokens, "slots": [-1] * tokens,
           "starts": [0], "lengths": [], "table": table}
    start = ends = used = 0
    for s, (kept, more) in enumerate(zip(lengths, added)):
        n, more = max(kept, 0), max(more, 0)
        held = -(-n // page)
        fits = n + more <= room and (packed or more <= 1)
        need = -(-(n + more) // page) - held if fits else 0
        before = ends
        ends += need
        served = fits and (need == 0 or ends <= count)
        if packed and more and start + more > tokens:
            served = False
        if served:
            used += need
            for j in range(need):
                table[s][held + j] = free[count - 1 - before - j]
            for i in range(more):
                p = n + i
                t = start + i if packed else s
                at = table[s][p // page]
                out["positions"][t], out["sequences"][t] = p, s
                out["slots"][t] = at * page + p % page if 0 <= at < pages else -1
        out["lengths"].append(n + more if served else kept)
        start += more
        out["starts"].append(min(start, 2 ** 31 - 1))
    out["free_count"] = count - used
    return out


def release(table, page, free, count, lengths, finished):
    free, pages = list(free), len(free)
    count = min(max(count, 0), pages)
    gone = []
    for row, n, over in zip(table, lengths, finished):
        if over:
            gone += row[:min(-(-max(n, 0) // page), len(row))]
    for i, p in enumerate(gone):
        place = count + len(gone) - 1 - i
        if place < pages:
            free[place] = p
    return {"free": free, "free_count": min(count + len(gone), pages),
            "lengths": [0 if over else n for n, over in zip(lengths, finished)]}


def deal(lengths, page, width, unused, g):
    """A table whose sequences hold their pages, dealt at random from a pool, and
    the list of the unused ones (padded with -1 to the pool's size)."""
    held = [-(-max(n, 0) // page) for n in lengths]
    total = sum(held) + unused
    order = torch.randperm(max(1, total), generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    free = order[at:at + unused] if total else []
    return table, free + [-1] * (max(1, total) - len(free))
