"""Adapters, sampling and page plans without a GPU: exported symbols and refusals
before any HIP call."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 4096  # an aligned address that is never followed


@pytest.fixture(scope="module")
def batch(hip):
    import batch_hip
    return batch_hip


@pytest.fixture(scope="module")
def paged(hip):
    import paged_hip
    return paged_hip


def test_library_exports_every_batch_symbol(batch):
    lib = batch.load()
    text = open(os.path.join(ROOT, "include", "infer_batch.h")).read()
    declared = sorted(set(re.findall(r"\b(infer_hip_\w+)\s*\(", text)))
    assert declared
    for name in declared:
        assert hasattr(lib, name), name
    assert sorted(batch.EXPORTED_SYMBOLS) == declared
    assert batch.MAX_TARGETS == int(re.search(r"INFER_HIP_LORA_TARGETS (\d+)", text).group(1))


# --------------------------------------------------------------- page plans --

ASSIGN = dict(table=A, num_sequences=3, max_pages=4, stride=4, page_size=16, free_pages=A,
              num_pages=9, free_count=A, free_count_out=A, lengths=A, added=A, lengths_out=A,
              tokens=7, positions=A, sequences=A, slots=A, starts=A, workspace=A,
              workspace_bytes=1 << 20)
RELEASE = dict(table=A, num_sequences=3, max_pages=4, stride=4, page_size=16, free_pages=A,
               num_pages=9, free_count=A, free_count_out=A, lengths=A, finished=A, lengths_out=A,
               workspace=A, workspace_bytes=1 << 20)
BOTH = [(dict(table=None), "null"), (dict(num_sequences=0), "block table"),
        (dict(num_sequences=65536), "block table"), (dict(max_pages=0), "block table"),
        (dict(stride=3), "block table"), (dict(max_pages=(1 << 26) + 1, stride=1 << 27),
                                          "block table"),
        (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"),
        (dict(page_size=512), "page_size"), (dict(page_size=0), "page_size"),
        (dict(free_pages=None), "null"), (dict(num_pages=0), "pages"),
        (dict(num_pages=(1 << 30) + 1), "pages"), (dict(free_count=None), "null"),
        (dict(free_count_out=None), "null"), (dict(lengths=None), "null"),
        (dict(lengths_out=None), "null"), (dict(workspace=None), "workspace"),
        (dict(workspace=A + 8), "workspace"), (dict(workspace_bytes=16), "workspace")]


def refused(hip, lib, fn, args, why):
    assert fn(*args.values(), None) == hip.INVALID_ARGUMENT
    assert why in lib.infer_hip_last_error().decode()


@pytest.mark.parametrize("change,why", BOTH)
def test_plan_refusals(hip, paged, change, why):
    lib = paged.load()
    refused(hip, lib, lib.infer_hip_kv_pages_assign, {**ASSIGN, **change}, why)
    refused(hip, lib, lib.infer_hip_kv_pages_release, {**RELEASE, **change}, why)


@pytest.mark.parametrize("change,why", [
    (dict(added=None), "null"), (dict(positions=None), "null"), (dict(tokens=0), "tokens"),
    (dict(tokens=(1 << 30) + 1), "tokens"), (dict(sequences=None, starts=None), "tokens"), (dict(sequences=None, tokens=3), "starts")])
def test_assign_refusals(hip, paged, change, why):
    lib = paged.load()
    refused(hip, lib, lib.infer_hip_kv_pages_assign, {**ASSIGN, **change}, why)


def test_release_refusals(hip, paged):
    lib = paged.load()
    refused(hip, lib, lib.infer_hip_kv_pages_release, {**RELEASE, "finished": None}, "null")


def test_plan_workspace(paged):
    size = paged.kv_pages_plan_workspace_bytes
    assert size(0) == size(-1) == size(65536) == 0
    assert 0 < size(1) <= size(2) <= size(65535) and size(65535) % 16 == 0


def test_plan_binding_refuses_cpu_tensors(hip, paged):
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    with pytest.raises(hip.InferError, match="GPU"):
        paged.kv_pages_assign(i(2, 3), 16, i(9), i(1), i(2), i(2), i(4), i(5), sequences=i(5))
    with pytest.raises(hip.InferError, match="GPU"):
        paged.kv_pages_release(i(2, 3), 16, i(9), i(1), i(2), i(2), i(4))


# ----------------------------------------------------------------- adapters --

TARGET = dict(a=A, b=A, base=A, output=2 * A, out_features=40, base_stride=40, output_stride=40)
LORA = dict(x=A, x_stride=64, ids=A, tokens=5, in_features=64, targets=None, num_targets=1,
            adapters=3, max_rank=16, ranks=A, scales=A, workspace=A, workspace_bytes=1 << 20)


def lora_args(batch, target=(), **change):
    t = (batch._Target * 3)(*[batch._Target(*{**TARGET, **dict(target)}.values())] * 3)
    return {**LORA, "targets": ctypes.cast(t, ctypes.c_void_p).value, **change}, t


@pytest.mark.parametrize("change,why", [
    (dict(x=None), "null"), (dict(x=A + 8), "aligned"), (dict(x_stride=63), "stride"),
    (dict(x_stride=68), "stride"), (dict(x_stride=56), "stride"), (dict(x_stride=-64), "stride"),
    (dict(ids=None), "null"), (dict(tokens=0), "tokens"), (dict(tokens=(1 << 20) + 1), "tokens"),
    (dict(in_features=0), "in_features"), (dict(in_features=60), "in_features"),
    (dict(in_features=1 << 23), "in_features"), (dict(targets=None), "null"),
    (dict(num_targets=0), "targets"), (dict(num_targets=4), "targets"),
    (dict(adapters=0), "adapters"), (dict(adapters=(1 << 20) + 1), "adapters"),
    (dict(max_rank=0), "rank"), (dict(max_rank=12), "rank"), (dict(max_rank=136), "rank"),
    (dict(workspace=None), "workspace"), (dict(workspace=A + 4), "workspace"),
    (dict(workspace_bytes=100), "workspace")])
def test_lora_refusals(hip, batch, change, why):
    args, keep = lora_args(batch, **change)
    lib = batch.load()
    refused(hip, lib, lib.infer_hip_lora_bf16, args, why)
    del keep


@pytest.mark.parametrize("target,why", [
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(output=None), "null"),
    (dict(a=A + 2), "aligned"), (dict(b=A + 8), "aligned"), (dict(out_features=0), "out_features"),
    (dict(out_features=1 << 23, output_stride=1 << 23, base_stride=1 << 23), "out_features"),
    (dict(output_stride=39), "stride"), (dict(base_stride=39), "stride"),
    (dict(output=A, output_stride=48), "base")])
def test_lora_target_refusals(hip, batch, target, why):
    lib = batch.load()
    for n in (1, 3):
        args, keep = lora_args(batch, target, num_targets=n)
        refused(hip, lib, lib.infer_hip_lora_bf16, args, why)
        del keep


def test_lora_targets_are_packed_as_the_structure(batch):
    fields = [1 << 40, 2, 3, 4, 5, 6, 1 << 41]
    for n in (1, 2, 3):
        want = bytes((batch._Target * n)(*[batch._Target(*fields)] * n))
        assert batch._PACK[n](*fields * n) == want


def test_lora_workspace(batch):
    size = batch.lora_workspace_bytes
    for bad in ((0, 16, 1), (1, 0, 1), (1, 12, 1), (1, 136, 1), (1, 16, 0), (1, 16, 4),
                ((1 << 20) + 1, 16, 1)):
        assert size(*bad) == 0
    assert 0 < size(1, 8, 1) <= size(2, 8, 1) <= size(2, 128, 3)


def test_lora_binding_refuses_cpu_tensors(hip, batch):
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(hip.InferError, match="GPU"):
        batch.lora(x, torch.zeros(2, dtype=torch.int32), [(x, x, x, x)], x)


# ----------------------------------------------------------------- sampling --

SAMPLE = dict(logits=A, stride=100, rows=3, vocab=100, temperature=A, top_k=A, top_p=A, min_p=A,
              uniform=A, tokens=A, probabilities=A, workspace=A, workspace_bytes=1 << 30)


@pytest.mark.parametrize("change,why", [
    (dict(logits=None), "null"), (dict(logits=A + 1), "aligned"), (dict(stride=99), "stride"),
    (dict(stride=-100), "stride"), (dict(rows=0), "rows"), (dict(rows=(1 << 20) + 1), "rows"),
    (dict(vocab=0), "tokens"), (dict(vocab=(1 << 20) + 1, stride=1 << 25), "tokens"),
    (dict(uniform=None), "null"), (dict(tokens=None), "null"),
    (dict(workspace=None), "workspace"), (dict(workspace=A + 8), "workspace"),
    (dict(workspace_bytes=0), "workspace")])
def test_sample_refusals(hip, batch, change, why):
    lib = batch.load()
    refused(hip, lib, lib.infer_hip_sample_bf16, {**SAMPLE, **change}, why)


def test_sample_workspace(batch):
    size = batch.sample_workspace_bytes
    assert size(0, 5) == size(5, 0) == size(1 << 21, 5) == size(5, 1 << 21) == 0
    assert 0 < size(1, 1) <= size(1, 151936) <= size(64, 151936)


def test_sample_binding_refuses_cpu_tensors(hip, batch):
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(hip.InferError, match="GPU"):
        batch.sample(x, torch.zeros(2), torch.zeros(2, dtype=torch.int32), x)


@pytest.mark.parametrize("rank,targets", [(8, 1), (40, 2), (128, 3)])
def test_a_workspace_serves_calls_of_fewer_tokens(batch, rank, targets):
    bytes_of = [batch.lora_workspace_bytes(t, rank, targets) for t in
                (1, 2, 16, 255, 256, 257, 300, 1024, 1025, 5000, 1 << 20)]
    assert bytes_of[0] > 0 and bytes_of == sorted(bytes_of)


# ------------------------------------------------------------------ bindings --

class Accepts:
    """In the library's place: every call is taken."""
    def __getattr__(self, name):
        return lambda *args: 0


def bound_calls(batch, paged, dev):
    """(binding, arguments) of sound calls whose tensors are on `dev`."""
    def i(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=dev)

    def f(*shape):
        return torch.zeros(shape, dtype=torch.float32, device=dev)

    def w(*shape):
        return torch.zeros(shape, dtype=torch.bfloat16, device=dev)

    u8 = torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    yield paged.kv_pages_assign, dict(
        table=i(3, 4), page_size=16, free=i(9), free_count=i(1), lengths=i(3), added=i(3),
        workspace=u8, positions=i(7), sequences=i(7), slots=i(7).long(), starts=i(4),
        lengths_out=i(3), free_count_out=i(1))
    yield paged.kv_pages_release, dict(
        table=i(3, 4), page_size=16, free=i(9), free_count=i(1), lengths=i(3), finished=i(3),
        workspace=u8, lengths_out=i(3), free_count_out=i(1))
    yield batch.sample, dict(
        logits=w(3, 50), uniform=f(3), tokens=i(3), workspace=u8, temperature=f(3), top_k=i(3),
        top_p=f(3), min_p=f(3), probabilities=f(3))

    def lora(x, ids, a, b, base, output, workspace, ranks, scales):
        batch.lora(x, ids, [(a, b, base, output)], workspace, ranks=ranks, scales=scales)
    yield lora, dict(x=w(5, 64), ids=i(5), a=w(2, 8, 64), b=w(2, 40, 8), base=w(5, 40),
                     output=w(5, 40), workspace=u8, ranks=i(2), scales=f(2))


def test_bindings_refuse_other_types_counts_and_strides(hip, batch, paged, monkeypatch):
    for module in (batch, paged):
        monkeypatch.setattr(module, "load", Accepts)
        monkeypatch.setattr(module, "_here", lambda t, name, stream: (t.get_device(), 0))
    for call, args in bound_calls(batch, paged, "cpu"):
        call(**args)
        for name, t in args.items():
            if not isinstance(t, torch.Tensor):
                continue
            bad = [t.short(), t.double()]
            if name not in ("free", "positions", "workspace"):  # their size is the call's
                bad.append(torch.cat([t, t]))
            if t.numel() > 1:  # every second element
                bad.append(torch.cat([t, t], dim=-1)[..., ::2])
            if name == "table":  # any shape of two dimensions
                bad = [t.short(), t.double(), t[0], torch.cat([t, t], dim=-1)[..., ::2]]
            for k, other in enumerate(bad):
                with pytest.raises(hip.InferError):
                    call(**{**args, name: other})
                    pytest.fail(f"{call.__name__}: {name}, {k}")


def test_bindings_refuse_numbers_of_targets(hip, batch, monkeypatch):
    monkeypatch.setattr(batch, "load", Accepts)
    monkeypatch.setattr(batch, "_here", lambda t, name, stream: (t.get_device(), 0))

    def w(*shape):
        return torch.zeros(shape, dtype=torch.bfloat16)
    target = (w(2, 8, 64), w(2, 40, 8), w(5, 40), w(5, 40))
    args = (w(5, 64), torch.zeros(5, dtype=torch.int32))
    for targets in ([], [target] * 4, [target, (w(2, 16, 64), w(2, 40, 16)) + target[2:]]):
        with pytest.raises(hip.InferError):
            batch.lora(*args, targets, torch.zeros(64, dtype=torch.uint8))


@pytest.mark.gpu
def test_bindings_refuse_tensors_of_the_host(hip, batch, paged, dev):
    """After every other check of theirs has passed without a GPU."""
    for call, args in bound_calls(batch, paged, dev):
        for name, t in args.items():
            if isinstance(t, torch.Tensor):
                with pytest.raises(hip.InferError):
                    call(**{**args, name: t.cpu()})
