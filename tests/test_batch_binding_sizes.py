"""Sizes past 32 bits, which the C ABI takes as int: the bindings of page plans, adapters
and sampling refuse them (ctypes would pass what is left of them).  Tensors without
memory, and a library that takes every call."""
import pytest
import torch


class Accepts:
    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def modules(hip, monkeypatch):
    import batch_hip
    import paged_hip
    for module in (batch_hip, paged_hip):
        monkeypatch.setattr(module, "load", Accepts)
        monkeypatch.setattr(module, "_here", lambda t, name, stream: (t.get_device(), 0))
    return batch_hip, paged_hip


def t(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


BIG = [2 ** 31, 2 ** 32 + 9]


@pytest.mark.parametrize("big", BIG)
@pytest.mark.parametrize("which", ["none", "free", "positions", "rows", "columns", "stride"])
def test_page_plans(hip, modules, which, big):
    paged = modules[1]
    n = big if which == "rows" else 3
    tokens = big if which == "positions" else 7
    table = (t(n, big if which == "columns" else 4) if which != "stride"
             else t(1).as_strided((3, 4), (big, 1)))
    pool = (table, 16, t(big if which == "free" else 9), t(1), t(n), t(n),
            t(64, dtype=torch.uint8))
    calls = [(lambda: paged.kv_pages_assign(*pool, t(tokens), sequences=t(tokens)),
              which == "none"),
             (lambda: paged.kv_pages_release(*pool), which in ("none", "positions"))]
    for call, sound in calls:
        if sound:
            call()
            continue
        with pytest.raises(hip.InferError):
            call()


@pytest.mark.parametrize("big", BIG)
@pytest.mark.parametrize("which", ["none", "tokens", "k", "adapters", "n"])
def test_adapters(hip, modules, which, big):
    batch = modules[0]
    size = {"tokens": 5, "k": 64, "adapters": 2, "n": 40}
    if which != "none":
        size[which] = big

    def w(*shape):
        return t(*shape, dtype=torch.bfloat16)
    args = (w(size["tokens"], size["k"]), t(size["tokens"]),
            [(w(size["adapters"], 8, size["k"]), w(size["adapters"], size["n"], 8),
              w(size["tokens"], size["n"]), w(size["tokens"], size["n"]))],
            t(64, dtype=torch.uint8))
    if which == "none":
        batch.lora(*args)
        return
    with pytest.raises(hip.InferError):
        batch.lora(*args)


@pytest.mark.parametrize("big", BIG)
@pytest.mark.parametrize("which", ["none", "rows", "vocab"])
def test_sampling(hip, modules, which, big):
    batch = modules[0]
    rows, vocab = big if which == "rows" else 3, big if which == "vocab" else 50
    args = (t(rows, vocab, dtype=torch.bfloat16), t(rows, dtype=torch.float32), t(rows),
            t(64, dtype=torch.uint8))
    if which == "none":
        batch.sample(*args)
        return
    with pytest.raises(hip.InferError):
        batch.sample(*args)
