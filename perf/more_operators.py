"""Operators around a step that serves several requests: the pages that its new
tokens need and the positions they get, low-rank adapters beside a shared
projection, and the choice of each sequence's next token.

Each case is a dict of plain values.  ``prepare`` makes what a program holds
before the call, ``run`` is one pass: with ``own`` false in plain torch, with
``own`` true through the framework's entry points.  ``work`` is what a pass
cannot do without and ``exact`` its result in 64 bits, written from the
definitions.

Pages: a pool's unused pages are the first ``free_count`` entries of ``free``,
the last of them handed out first.  Each sequence holds ``lengths`` positions
and gets ``added`` more; new pages go to the sequences in order, and one whose
pages do not all fit gets none and stays as it is.  A token's slot is page *
page size + position % page size.

Adapters: out = base + scale[id] * B[id] (A[id] x) for each token's id (-1:
none), A [adapters][largest rank][K], B [adapters][N][largest rank], the first
ranks[id] of them in use, for one to three projections of one x.

Sampling: a row's tokens in descending order of logit (ties: lowest index
first), weighted by exp((logit - largest) / temperature); the first top_k of
them, of those the shortest run with top_p of their weight, of those the ones
with at least min_p of the largest weight; the first token whose running weight
passes uniform * total.  Temperature 0 takes the first token.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "qwen2.5-jetson-inference_amd")


def listed():
    return [
        # A decode step of 24 sequences, some slots idle: pure latency.
        {"name": "assign_24_decode", "kind": "assign", "form": "decode", "sequences": 24,
         "longest": 1000, "page": 16, "short": False},
        # Eight prompts that arrive together.
        {"name": "assign_8x6000_prompts", "kind": "assign", "form": "prompts", "sequences": 8,
         "longest": 6000, "page": 16, "short": False},
        # A very large batch of prompts and continuations, more than the pool has
        # pages for.
        {"name": "assign_2000x3000_mixed", "kind": "assign", "form": "mixed", "sequences": 2000,
         "longest": 3000, "page": 32, "short": True},
        # A batch in which half of the sequences have ended.
        {"name": "release_64x4000", "kind": "release", "sequences": 64, "longest": 4000,
         "page": 16},
        # A pool that is nearly emptied at once.
        {"name": "release_1500x20000", "kind": "release", "sequences": 1500, "longest": 20000,
         "page": 16},
        # The smallest adapter call: one token, rank 8, a square projection.
        {"name": "lora_1x896_r8", "kind": "lora", "tokens": 1, "k": 896, "outs": "896", "rank": 8,
         "adapters": 4, "layout": "mixed"},
        # A decode step's q, k and v for 33 requests with adapters of their own.
        {"name": "lora_33x1536_qkv_r16", "kind": "lora", "tokens": 33, "k": 1536,
         "outs": "1536+256+256", "rank": 16, "adapters": 40, "layout": "mixed"},
        # A large batch's gate and up with high ranks: the adapters' bytes.
        {"name": "lora_128x3584_gate_up_r64", "kind": "lora", "tokens": 128, "k": 3584,
         "outs": "18944+18944", "rank": 64, "adapters": 12, "layout": "mixed"},
        # Prompts, each with one adapter.
        {"name": "lora_6001x1536_prompts_r32", "kind": "lora", "tokens": 6001, "k": 1536,
         "outs": "8960", "rank": 32, "adapters": 6, "layout": "prompts"},
        # One sequence's next token.
        {"name": "sample_1x151936", "kind": "sample", "rows": 1, "vocab": 151936},
        # A small batch, an odd vocabulary.
        {"name": "sample_17x32003", "kind": "sample", "rows": 17, "vocab": 32003},
        # A full batch over a large vocabulary.
        {"name": "sample_256x151936", "kind": "sample", "rows": 256, "vocab": 151936},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["assign", "assign", "release", "lora", "lora", "lora", "sample", "sample",
                       "sample"])
    if kind in ("assign", "release"):
        case = {"kind": kind, "sequences": _log(rng, 1, 4000),
                "page": rng.choice([16, 32, 64, 128, 256])}
        if kind == "release":
            return dict(case, longest=_log(rng, 20, min(100000, 30000000 // case["sequences"])))
        form = rng.choice(["decode", "prompts", "mixed"])
        room = {"decode": 16000000, "mixed": 6000000, "prompts": 1400000}[form]
        return dict(case, form=form, longest=_log(rng, 20, min(60000, room // case["sequences"])),
                    short=rng.random() < 0.3)
    if kind == "sample":
        rows = _log(rng, 1, 300)
        return {"kind": kind, "rows": rows,
                "vocab": _log(rng, 900, min(260000, 256 * 151936 // rows))}
    layout = rng.choice(["mixed", "mixed", "prompts"])
    k = 8 * _log(rng, 64, 1120)
    outs = [_log(rng, 100, 19000) for _ in range(rng.randint(1, 3))]
    if rng.random() < 0.7:
        outs = [-(-n // 8) * 8 for n in outs]
    rank = rng.choice([8, 16, 24, 32, 64, 128])
    room = 6001 * (1536 + 2 * 8960) // (k + 2 * sum(outs))  # tokens and adapters by bytes
    held = max(2, 35000000 // (rank * (k * len(outs) + sum(outs))))
    return {"kind": kind, "tokens": _log(rng, 1, min(300, room)) if layout == "mixed"
            else _log(rng, 20, max(30, room)), "k": k, "outs": "+".join(map(str, outs)),
            "rank": rank, "adapters": _log(rng, 1, min(40, held)), "layout": layout}


# ------------------------------------------------------------- inputs --


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sizes(case):
    """(cached, added) of each sequence."""
    rng = random.Random(case["longest"] * 1000 + case["sequences"])
    cached, added = [], []
    for _ in range(case["sequences"]):
        form = case["form"]
        if form == "mixed":  # one in four is a prompt or a later piece of one
            form = rng.choice(["decode", "decode", "decode", "prompts"])
        if form == "decode":
            cached.append(rng.randint(0, case["longest"] - 1))
            added.append(int(rng.random() < 0.9))
        else:
            n = rng.randint(1, case["longest"])
            held = rng.randint(0, n - 1) if rng.random() < 0.3 else 0
            cached.append(held)
            added.append(n - held)
    return cached, added


def _plan_inputs(case, seed):
    """Pages dealt at random: the sequences' own into the table, the rest
    unused."""
    page, rng = case["page"], random.Random(case["longest"] + 7 * case["sequences"])
    if case["kind"] == "assign":
        cached, added = _sizes(case)
    else:
        cached = [rng.randint(0, case["longest"]) for _ in range(case["sequences"])]
        added = [0] * len(cached)
    held = [-(-n // page) for n in cached]
    need = sum(-(-(n + m) // page) - h for n, m, h in zip(cached, added, held))
    unused = need * 4 // 5 if case.get("short") else need + 5
    total = sum(held) + unused
    g = torch.Generator().manual_seed(int(seed) & 0xFFFFFFF)
    order = torch.randperm(max(1, total), generator=g).to(torch.int32)
    width = max(1, -(-case["longest"] // page))
    table = torch.full((len(cached), width), -1, dtype=torch.int32)
    counts = torch.tensor(held)
    mine = torch.arange(width)[None] < counts[:, None]
    table[mine] = order[:sum(held)]
    free = torch.full((max(1, total),), -1, dtype=torch.int32)
    free[:unused] = order[sum(held):total]
    s = {"table": table.cuda(), "free": free.cuda(), "free_count": _ints([unused]),
         "lengths": _ints(cached)}
    if case["kind"] == "assign":
        s["added"] = _ints(added)
    else:  # half of the sequences have ended, nearly all of a very large batch
        part = 0.5 if len(cached) < 500 else 0.9
        s["finished"] = (torch.rand(len(cached), generator=g) < part).to(torch.int32).cuda()
    return s, sum(added)


def _lora_ids(case, seed):
    """Each token's adapter: any, one in ten none; or runs of one adapter, one
    of four or more without."""
    rng, t = random.Random(seed), case["tokens"]
    if case["layout"] == "mixed":
        ids = [-1 if rng.random() < 0.1 else rng.randrange(case["adapters"]) for _ in range(t)]
        return [rng.randrange(case["adapters"])] + ids[1:]
    runs = min(t, case["adapters"])
    cuts = sorted(rng.sample(range(1, t), runs - 1)) + [t]
    names = list(range(runs))
    rng.shuffle(names)
    if runs >= 4:
        names[rng.randrange(runs)] = -1
    ids = []
    for name, end in zip(names, cuts):
        ids += [name] * (end - len(ids))
    return ids


def _ranks(case):
    rng, r = random.Random(case["rank"] * 100 + case["adapters"]), case["rank"]
    return [r] + [rng.choice([r, r, r // 2, r * 3 // 4]) for _ in range(case["adapters"] - 1)]


def _outs(case):
    return [int(n) for n in case["outs"].split("+")]


def _lora_inputs(case, seed):
    """Activations with a few strong channels, adapters as training leaves them
    (A near its start, B small), a projection's output of the same size."""
    g, t, k, r, m = _gen(seed), case["tokens"], case["k"], case["rank"], case["adapters"]

    def normal(shape, std):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)
    x = normal((t, k), 1.0)
    x[:, :: 101] *= 8
    return {"x": x, "ids": _ints(_lora_ids(case, seed)), "ranks": _ints(_ranks(case)),
            "scales": torch.rand(m, generator=g, device="cuda") * 1.5 + 0.5,
            "a": [normal((m, r, k), k ** -0.5) for _ in _outs(case)],
            "b": [normal((m, n, r), 0.1) for n in _outs(case)],
            "base": [normal((t, n), 1.0) for n in _outs(case)]}


def _sample_inputs(case, seed):
    """Logits of a trained model's shape: many low ones, a few far above; every
    request with settings of its own."""
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.2 - 1.0
    at = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    high = torch.rand((rows, 24), generator=g, device="cuda") * 9 + 6
    logits.scatter_(1, at, high)
    rng = random.Random(seed)
    pick = lambda values: [rng.choice(values) for _ in range(rows)]  # noqa: E731

    def floats(values):
        return torch.tensor(values, dtype=torch.float32, device="cuda")
    first = rng.choice([0.6, 0.8, 1.0])
    return {"logits": logits.to(torch.bfloat16),
            "uniform": torch.rand(rows, generator=g, device="cuda"),
            "temperature": floats([first] + pick([0.0, 0.3, 0.7, 0.8, 1.0, 1.0, 1.3])[1:]),
            "top_k": _ints(pick([0, 0, 1, 20, 50, 64, 1000])),
            "top_p": floats(pick([1.0, 1.0, 0.8, 0.9, 0.95])),
            "min_p": floats(pick([0.0, 0.0, 0.0, 0.02, 0.1]))}


def _framework():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import batch_hip
    import paged_hip
    return batch_hip, paged_hip


def prepare(case, seed):
    kind = case["kind"]
    if kind == "lora":
        s = _lora_inputs(case, seed)
        s["out"] = [torch.empty_like(y) for y in s["base"]]
    elif kind == "sample":
        s = _sample_inputs(case, seed)
        s["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        s["probabilities"] = torch.empty(case["rows"], device="cuda")
    else:
        s, tokens = _plan_inputs(case, seed)
        if kind == "assign":
            # room for some padding, as a captured step of a fixed size has
            room = case["sequences"] if case["form"] == "decode" else tokens + 13
            s["positions"] = torch.empty(room, dtype=torch.int32, device="cuda")
            s["slots"] = torch.empty(room, dtype=torch.int64, device="cuda")
            if case["form"] != "decode":
                s["sequences"] = torch.empty_like(s["positions"])
                s["starts"] = torch.empty(case["sequences"] + 1, dtype=torch.int32, device="cuda")
        s["lengths_out"] = torch.empty_like(s["lengths"])
        s["free_count_out"] = torch.empty_like(s["free_count"])
    s["case"] = case
    if own:
        # the workspaces, which a program makes once
        s["batch"], s["paged"] = _framework()
        if kind == "lora":
            need = s["batch"].lora_workspace_bytes(case["tokens"], case["rank"], len(s["a"]))
        elif kind == "sample":
            need = s["batch"].sample_workspace_bytes(case["rows"], case["vocab"])
        else:
            need = s["paged"].kv_pages_plan_workspace_bytes(case["sequences"])
        s["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- run --


def run(state):
    kind = state["case"]["kind"]
    if kind == "lora":
        _own_lora(state) if own else _plain_lora(state)
        return state["out"]
    if kind == "sample":
        _own_sample(state) if own else _plain_sample(state)
        return {"tokens": state["tokens"], "probabilities": state["probabilities"]}
    if kind == "release":
        _own_release(state) if own else _plain_release(state)
        return {"free": state["free"], "free_count": state["free_count_out"],
                "lengths": state["lengths_out"]}
    _own_assign(state) if own else _plain_assign(state)
    out = {"table": state["table"], "positions": state["positions"], "slots": state["slots"],
           "lengths": state["lengths_out"], "free_count": state["free_count_out"]}
    if state["case"]["form"] != "decode":
        out["sequences"], out["starts"] = state["sequences"], state["starts"]
    return out


def _own_assign(s):
    s["paged"].kv_pages_assign(
        s["table"], s["case"]["page"], s["free"], s["free_count"], s["lengths"], s["added"],
        s["workspace"], s["positions"], sequences=s.get("sequences"), slots=s["slots"],
        starts=s.get("starts"), lengths_out=s["lengths_out"], free_count_out=s["free_count_out"])


def _own_release(s):
    s["paged"].kv_pages_release(
        s["table"], s["case"]["page"], s["free"], s["free_count"], s["lengths"], s["finished"],
        s["workspace"], lengths_out=s["lengths_out"], free_count_out=s["free_count_out"])


def _own_lora(s):
    s["batch"].lora(s["x"], s["ids"], list(zip(s["a"], s["b"], s["base"], s["out"])),
                    s["workspace"], ranks=s["ranks"], scales=s["scales"])


def _own_sample(s):
    s["batch"].sample(s["logits"], s["uniform"], s["tokens"], s["workspace"],
                      temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"], probabilities=s["probabilities"])


def _plain_assign(s):
    page, table = s["case"]["page"], s["table"]
    old, added = s["lengths"].long(), s["added"].long()
    held = (old + page - 1) // page
    need = (old + added + page - 1) // page - held
    ends = need.cumsum(0)
    served = (need == 0) | (ends <= s["free_count"])
    s["lengths_out"].copy_(torch.where(served, old + added, old))
    used = torch.where(served, need, 0).sum()
    s["free_count_out"].copy_(s["free_count"] - used)
    # the token t of the call, its sequence and its position there
    t = torch.arange(len(s["positions"]), device="cuda")
    if "starts" in s:
        starts = torch.cat([added.new_zeros(1), added.cumsum(0)])
        s["starts"].copy_(starts)
        seq = torch.searchsorted(starts[1:], t, right=True).clamp(max=len(old) - 1)
        live = t < starts[-1]
    else:
        seq, starts = t, t
        live = added > 0
    pos = old[seq] + t - starts[seq]
    live = live & served[seq]
    entry = (pos // page).clamp(max=table.shape[1] - 1)
    fresh = live & (pos // page >= held[seq])
    at = s["free_count"].long() - 1 - (ends - need)[seq] - (pos // page - held[seq])
    new = s["free"][at.clamp(0, len(s["free"]) - 1)]
    own_page = torch.where(fresh, new, table[seq, entry])
    where = torch.where(fresh, seq * table.shape[1] + entry, table.numel())
    wide = torch.cat([table.view(-1), table.new_zeros(1)])
    wide[where] = own_page
    table.copy_(wide[:-1].view(table.shape))
    s["positions"].copy_(torch.where(live, pos, -1))
    s["slots"].copy_(torch.where(live, own_page.long() * page + pos % page, -1))
    if "sequences" in s:
        s["sequences"].copy_(torch.where(live, seq, -1))


def _plain_release(s):
    page, table = s["case"]["page"], s["table"]
    out = s["finished"] != 0
    held = torch.where(out, (s["lengths"].long() + page - 1) // page, 0)
    total = held.sum()
    column = torch.arange(table.shape[1], device="cuda")[None]
    gone = column < held[:, None]
    # the i-th page released becomes the i-th from the end of the unused ones
    place = s["free_count"] + total - 1 - ((held.cumsum(0) - held)[:, None] + column)
    wide = torch.cat([s["free"], s["free"].new_zeros(1)])
    wide[torch.where(gone, place, len(s["free"]))] = table
    s["free"].copy_(wide[:-1])
    s["free_count_out"].copy_(s["free_count"] + total)
    s["lengths_out"].copy_(torch.where(out, 0, s["lengths"]))


def _plain_lora(s):
    m, r, k = s["a"][0].shape
    mine = s["ids"][:, None] == torch.arange(m, device="cuda")
    live = torch.arange(r, device="cuda")[None] < s["ranks"][:, None]
    factor = (mine[:, :, None] & live) * s["scales"][:, None]
    x = s["x"].float()
    for a, b, base, out in zip(s["a"], s["b"], s["base"], s["out"]):
        h = (x @ a.float().view(m * r, k).t()) * factor.view(-1, m * r)
        out.copy_(base.float() + h @ b.float().transpose(1, 2).reshape(m * r, -1))


def _plain_sample(s):
    rows, vocab = s["logits"].shape
    values, order = s["logits"].double().sort(dim=1, descending=True, stable=True)
    greedy = s["temperature"] == 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    w = ((values - values[:, :1]) / t).exp()
    place = torch.arange(vocab, device="cuda")[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)
    keep = place < torch.where(greedy, 1, k)[:, None]
    total = torch.where(keep, w, 0.0).cumsum(1)
    p = s["top_p"].double()[:, None]
    # a token stays while those before it hold less than top_p of the weight
    keep = keep & ((p >= 1) | (total - w < p * total[:, -1:]) | (place == 0))
    keep = keep & (w >= s["min_p"].double()[:, None])
    w = torch.where(keep, w, 0.0)
    total = w.cumsum(1)
    target = s["uniform"].double()[:, None] * total[:, -1:]
    first = (total <= target).sum(dim=1, keepdim=True).clamp(max=vocab - 1)
    s["tokens"].copy_(order.gather(1, first)[:, 0])
    s["probabilities"].copy_((w.gather(1, first) / total[:, -1:])[:, 0])


# --------------------------------------------------------------- work --


def work(case):
    """Each input read once, each output written once; multiply-adds as two."""
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2.0 * n + 28.0 * case["rows"], "flops": 2.0 * n}
    if case["kind"] == "lora":
        ids, ranks, k, outs = _lora_ids(case, 1), _ranks(case), case["k"], _outs(case)
        used = sum(ranks[i] for i in set(ids) if i >= 0)
        each = sum(ranks[i] for i in ids if i >= 0)
        t, n, c = case["tokens"], sum(outs), len(outs)
        return {"bytes": 2.0 * t * k + 4.0 * t * n + 2.0 * used * (c * k + n) + 4.0 * t
                + 8.0 * case["adapters"], "flops": 2.0 * each * (c * k + n)}
    page, n = case["page"], case["sequences"]
    if case["kind"] == "release":
        rng = random.Random(case["longest"] + 7 * n)
        pages = sum(-(-rng.randint(0, case["longest"]) // page) for _ in range(n))
        part = 0.5 if n < 500 else 0.9
        return {"bytes": 8.0 * part * pages + 12.0 * n, "flops": 1.0 * n}
    cached, added = _sizes(case)
    fresh = sum(-(-(c + m) // page) + (-c // page) for c, m in zip(cached, added))
    tokens = sum(added)
    return {"bytes": tokens * (12.0 if case["form"] == "decode" else 16.0) + 8.0 * fresh
            + (12.0 if case["form"] == "decode" else 16.0) * n + 4.0 * tokens / page,
            "flops": 1.0 * (tokens + n)}


# -------------------------------------------------------------- exact --


def _exact_assign(case, seed):
    s, tokens = _plan_inputs(case, seed)
    page, table, free = case["page"], s["table"].cpu(), s["free"].tolist()
    count, cached, added = int(s["free_count"]), s["lengths"].tolist(), s["added"].tolist()
    decode = case["form"] == "decode"
    room = case["sequences"] if decode else tokens + 13
    positions = torch.full((room,), -1, dtype=torch.int64)
    slots, ids = positions.clone(), positions.clone()
    starts, at, asked, left = [0], 0, 0, count
    lengths = list(cached)
    for i, (n, m) in enumerate(zip(cached, added)):
        held = -(-n // page)
        more = -(-(n + m) // page) - held
        if more == 0 or asked + more <= count:
            for j in range(more):
                table[i, held + j] = free[count - 1 - asked - j]
            left -= more
            lengths[i] = n + m
            where = i if decode else at
            p = torch.arange(n, n + m)
            positions[where:where + m] = p
            slots[where:where + m] = table[i, p // page].long() * page + p % page
            ids[where:where + m] = i
        asked += more
        at += m
        starts.append(at)
    out = {"table": table, "positions": positions.int(), "slots": slots,
           "lengths": torch.tensor(lengths, dtype=torch.int32),
           "free_count": torch.tensor([left], dtype=torch.int32)}
    if not decode:
        out["sequences"] = ids.int()
        out["starts"] = torch.tensor(starts, dtype=torch.int32)
    return out


def _exact_release(case, seed):
    s, _ = _plan_inputs(case, seed)
    gone, lengths = [], s["lengths"].tolist()
    table = s["table"].cpu()
    for i, over in enumerate(s["finished"].tolist()):
        if over:
            gone.append(table[i, :-(-lengths[i] // case["page"])])
            lengths[i] = 0
    gone = torch.cat(gone).flip(0) if gone else torch.zeros(0, dtype=torch.int32)
    free, count = s["free"].cpu(), int(s["free_count"])
    free[count:count + len(gone)] = gone
    return {"free": free, "free_count": torch.tensor([count + len(gone)], dtype=torch.int32),
            "lengths": torch.tensor(lengths, dtype=torch.int32)}


def _exact_lora(case, seed):
    s, ranks = _lora_inputs(case, seed), _ranks(case)
    ids = s["ids"].long()
    out = [y.double() for y in s["base"]]
    for i in sorted(set(ids.tolist()) - {-1}):
        mine = (ids == i).nonzero()[:, 0]
        for y, a, b in zip(out, s["a"], s["b"]):
            h = s["x"][mine].double() @ a[i, :ranks[i]].double().t()
            y[mine] += s["scales"][i].double() * (h @ b[i, :, :ranks[i]].double().t())
    return out


def _exact_sample(case, seed):
    """By the distinct values of a row, largest first, and how many hold each."""
    s = _sample_inputs(case, seed)
    tokens, chances = [], []
    for i in range(case["rows"]):
        row = s["logits"][i]
        values, counts = torch.unique(row.double(), return_counts=True)
        values, counts = values.flip(0), counts.flip(0).double()
        t, k = float(s["temperature"][i]), int(s["top_k"][i])
        if t == 0:
            k, t = 1, 1.0
        before = counts.cumsum(0) - counts
        if k > 0:  # of the value at the border, only those that still fit
            counts = torch.minimum(counts, (k - before).clamp(min=0))
        w = ((values - values[0]) / t).exp()
        mass = counts * w
        sums = mass.cumsum(0)
        p = float(s["top_p"][i])
        if p < 1:
            lacking = (p * sums[-1] - (sums - mass)) / w
            counts = torch.minimum(counts, lacking.ceil().clamp(min=0))
            counts[0] = counts[0].clamp(min=1)
        counts = torch.where(w >= float(s["min_p"][i]), counts, 0.0)
        mass = counts * w
        sums = mass.cumsum(0)
        target = float(s["uniform"][i]) * sums[-1]
        j = int((sums <= target).sum())
        nth = int(((target - (sums[j] - mass[j])) / w[j]).floor())
        nth = min(nth, int(counts[j]) - 1)
        tokens.append((row.double() == values[j]).nonzero()[nth, 0])
        chances.append(w[j] / sums[-1])
    return {"tokens": torch.stack(tokens).int(), "probabilities": torch.stack(chances)}


def exact(case, seed):
    return {"assign": _exact_assign, "release": _exact_release, "lora": _exact_lora,
            "sample": _exact_sample}[case["kind"]](case, seed)
