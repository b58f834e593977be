"""A served batch's operators one after the other, as a step uses them: pages and
positions for the new tokens, adapters beside a projection, the cache written and
attended, the next tokens drawn, ended sequences' pages given back; the decode
steps as one captured graph over state that changes in place."""
import math

import pytest
import torch

import batch_ref
import paged_ref
import plan_ref

pytestmark = pytest.mark.gpu

HEADS, KV, D, PAGE, VOCAB, K = 4, 2, 64, 16, 3000, 256


class Step:
    """Weights and the operators' calls of one layer and a head."""

    def __init__(self, dev, sequences, adapters, seed):
        import batch_hip
        import linear_hip
        import paged_hip
        self.batch, self.linear, self.paged = batch_hip, linear_hip, paged_hip
        g = torch.Generator().manual_seed(seed)
        n = (HEADS + 2 * KV) * D

        def bf16(shape, std):
            return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)
        self.cpu = {"embed": bf16((VOCAB, K), 1.0), "qkv": bf16((n, K), K ** -0.5),
                    "a": bf16((adapters, 8, K), K ** -0.5), "b": bf16((adapters, n, 8), 0.3),
                    "head": bf16((VOCAB, HEADS * D), 0.4)}
        self.w = {k: v.to(dev) for k, v in self.cpu.items()}
        self.rope = paged_ref.rope_table(200, D)
        self.dev_rope = self.rope.to(dev)
        self.dev, self.n = dev, n
        self.ids = torch.randint(-1, adapters, (sequences,), generator=g, dtype=torch.int32)
        self.dev_ids = self.ids.to(dev)

    def scratch(self, tokens, attended):
        d = {"device": self.dev}
        b = self.batch
        return {"x": torch.empty((tokens, K), dtype=torch.bfloat16, **d),
                "qkv": torch.empty((tokens, self.n), dtype=torch.bfloat16, **d),
                "q": torch.empty((tokens, HEADS, D), dtype=torch.bfloat16, **d),
                "out": torch.empty((attended, HEADS, D), dtype=torch.bfloat16, **d),
                "logits": torch.empty((attended, VOCAB), dtype=torch.bfloat16, **d),
                "positions": torch.empty(tokens, dtype=torch.int32, **d),
                "lora": torch.empty(b.lora_workspace_bytes(tokens, 8, 1), dtype=torch.uint8, **d),
                "sample": torch.empty(b.sample_workspace_bytes(attended, VOCAB),
                                      dtype=torch.uint8, **d),
                "attend": torch.empty(self.paged.attention_paged_decode_workspace_bytes(
                    attended, HEADS, KV, D), dtype=torch.uint8, **d)}

    def project(self, s, tokens, ids):
        self.linear.gemm_bf16(self.w["qkv"], None, s["x"], s["qkv"], tokens, self.n, K) \
            if tokens > 1 else self.linear.gemv_bf16(self.w["qkv"], None, s["x"], s["qkv"],
                                                     self.n, K)
        self.batch.lora(s["x"], ids, [(self.w["a"], self.w["b"], s["qkv"], s["qkv"])], s["lora"])
        return s["qkv"].view(tokens, HEADS + 2 * KV, D).split([HEADS, KV, KV], dim=1)


def close(got, want, size):
    return ((got.double().cpu() - want).abs() <= size).all()


def test_prompts_then_captured_steps_then_release(dev):
    sequences, steps = 6, 5
    m = Step(dev, sequences, 3, 1)
    g = torch.Generator().manual_seed(2)
    prompt = [5, 0, 17, 33, 1, 16]  # sequence 1 stays idle
    total = sum(prompt)
    pages = m.paged.KvPages.allocate(24, PAGE, KV, D, "bf16", dev)
    order = torch.randperm(24, generator=g).tolist()
    table = [[-1] * 5 for _ in range(sequences)]
    state = {"table": torch.tensor(table, dtype=torch.int32, device=dev),
             "free": torch.tensor(order, dtype=torch.int32, device=dev),
             "count": torch.tensor([24], dtype=torch.int32, device=dev),
             "lengths": torch.zeros(sequences, dtype=torch.int32, device=dev)}
    plan_ws = torch.empty(m.paged.kv_pages_plan_workspace_bytes(sequences), dtype=torch.uint8,
                          device=dev)

    # The prompts, packed; the caller's padding of three tokens stores nothing.
    tokens = total + 3
    s = m.scratch(tokens, sequences)
    added = torch.tensor(prompt, dtype=torch.int32, device=dev)
    ids = torch.empty(tokens, dtype=torch.int32, device=dev)
    m.paged.kv_pages_assign(state["table"], PAGE, state["free"], state["count"], state["lengths"],
                            added, plan_ws, s["positions"], sequences=ids)
    want = plan_ref.assign(table, PAGE, order, 24, [0] * sequences, prompt, tokens, True)
    assert s["positions"].tolist() == want["positions"] and ids.tolist() == want["sequences"]
    words = torch.randint(0, VOCAB, (tokens,), generator=g)
    s["x"].copy_(m.cpu["embed"][words])
    token_ids = torch.where(ids >= 0, m.dev_ids[ids.clamp(min=0).long()], -1).to(torch.int32)
    q, k, v = m.project(s, tokens, token_ids)
    base = m.cpu["embed"][words].double() @ m.cpu["qkv"].double().t()
    exact, tol = batch_ref.lora(m.cpu["embed"][words], token_ids.cpu(), None, None, m.cpu["a"],
                                m.cpu["b"], base)
    # the projection's own rounding before the adapters', half a step of it
    assert close(s["qkv"], exact, tol + base.abs() * 2.0 ** -8 + 1e-4)
    m.paged.kv_pages_store(pages, state["table"], s["positions"], q, k, v, s["q"],
                           rope=m.dev_rope, sequences=ids)
    cached = [[] for _ in range(sequences)]  # (key, value) rows of each sequence
    kr = paged_ref.fused_free(k.cpu(), m.rope[s["positions"].cpu().clamp(min=0).long()])
    for t in range(total):
        cached[want["sequences"][t]].append((kr[t].to(torch.bfloat16), v[t].cpu()))

    # Decode steps: one graph, replayed; the random numbers and idle sequences change.
    d = m.scratch(sequences, sequences)
    one = torch.tensor([int(n > 0) for n in prompt], dtype=torch.int32, device=dev)
    uniform = torch.empty(sequences, device=dev)
    last = torch.tensor([int(words[max(0, e - 1)]) for e in want["starts"][1:]],
                        dtype=torch.int32, device=dev)
    temperature = torch.tensor([0.0, 1.0, 0.7, 1.0, 1.3, 1.0], device=dev)
    top_k = torch.tensor([0, 0, 50, 0, 7, 0], dtype=torch.int32, device=dev)
    top_p = torch.tensor([1.0, 1.0, 1.0, 0.9, 0.95, 1.0], device=dev)

    def step():
        m.paged.kv_pages_assign(state["table"], PAGE, state["free"], state["count"],
                                state["lengths"], one, plan_ws, d["positions"])
        d["x"].copy_(m.w["embed"][last.long()])
        q, k, v = m.project(d, sequences, m.dev_ids)
        m.paged.kv_pages_store(pages, state["table"], d["positions"], q, k, v, d["q"],
                               rope=m.dev_rope)
        m.paged.attention_paged_decode(pages, state["table"], state["lengths"], d["q"], d["out"],
                                       d["attend"])
        m.linear.gemm_bf16(m.w["head"], None, d["out"].view(sequences, HEADS * D), d["logits"],
                           sequences, VOCAB, HEADS * D)
        m.batch.sample(d["logits"], uniform, last, d["sample"], temperature=temperature,
                       top_k=top_k, top_p=top_p)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    table, lengths, count = want["table"], want["lengths"], want["free_count"]
    for i in range(steps):
        us = torch.rand(sequences, generator=g)
        uniform.copy_(us)
        before = last.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = plan_ref.assign(table, PAGE, order, count, lengths, one.tolist(), sequences, False)
        table, lengths, count = want["table"], want["lengths"], want["free_count"]
        assert d["positions"].tolist() == want["positions"]
        assert state["table"].tolist() == table and state["lengths"].tolist() == lengths
        assert state["count"].tolist() == [count]
        x = m.cpu["embed"][before.cpu().long()]
        base = x.double() @ m.cpu["qkv"].double().t()
        exact, tol = batch_ref.lora(x, m.ids, None, None, m.cpu["a"], m.cpu["b"], base)
        assert close(d["qkv"], exact, tol + base.abs() * 2.0 ** -8 + 1e-4)
        q, k, v = d["qkv"].cpu().view(sequences, -1, D).split([HEADS, KV, KV], dim=1)
        kr = paged_ref.fused_free(k, m.rope[d["positions"].cpu().clamp(min=0).long()])
        for n in range(sequences):
            if not prompt[n]:
                assert (d["out"][n] == 0).all()
                continue
            cached[n].append((kr[n].to(torch.bfloat16), v[n]))
            keys = torch.stack([r[0] for r in cached[n]], dim=1).double()
            values = torch.stack([r[1] for r in cached[n]], dim=1).double()
            out, mean, big = paged_ref.attend(d["q"][n].cpu(), keys, values)
            # the output's rounding, and softmax's of 32-bit scores of size `big`
            assert close(d["out"][n], out, out.abs() * 2.0 ** -8 + mean * (
                2.0 ** -18 * (1 + big)) + 1e-6)
        for n in range(sequences):
            token, _ = batch_ref.sample(
                d["logits"][n].cpu(), float(temperature[n]), int(top_k[n]),
                float(top_p[n].double()), 0.0, float(us[n].double()))
            assert int(last[n]) == token

    # Two sequences end; what they held can be handed out again.
    finished = torch.tensor([0, 0, 1, 0, 1, 0], dtype=torch.int32, device=dev)
    back = plan_ref.release(table, PAGE, order, count, lengths, finished.tolist())
    m.paged.kv_pages_release(state["table"], PAGE, state["free"], state["count"],
                             state["lengths"], finished, plan_ws)
    assert state["free"].tolist()[:back["free_count"]] == back["free"][:back["free_count"]]
    assert state["count"].tolist() == [back["free_count"]]
    assert state["lengths"].tolist() == back["lengths"]
    held = {p for row, n in zip(table, back["lengths"]) for p in row[:-(-n // PAGE)]}
    assert held.isdisjoint(back["free"][:back["free_count"]])
    assert len(held) + back["free_count"] == 24 and not math.isnan(float(d["out"].sum()))
