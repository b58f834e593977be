"""Sampling (infer_hip_sample_bf16) of rows in which few values have most of the
tokens, against its definition in 64 bits (tests/batch_ref.py)."""
import pytest
import torch

from test_gpu_sample import batch, check, gen, rows_of, settings  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [155649, 200000, 262147, 1048576])
@pytest.mark.parametrize("zeros", [65536, 70001, 131072])
def test_rows_that_begin_with_zeros(batch, dev, vocab, zeros):  # noqa: F811
    """More of them than a workgroup takes at a time of a row that it reads twice; in the
    last rows negative zeros and the smallest number among them."""
    logits, uniform = rows_of(4, vocab, vocab + zeros)
    logits[:, :zeros] = 0.0
    logits[2, 5:zeros:2] = -0.0
    logits[3, 3:zeros:1000] = 2.0 ** -133
    check(batch, dev, logits, uniform)
    check(batch, dev, logits, uniform, **settings(4, vocab))
    check(batch, dev, logits, uniform, top_k=[1000, 30000, 60000, 100000])


LOWEST = torch.finfo(torch.bfloat16).min


def masked(vocab, mask, seed):
    """Rows of a finite mask with lower values in a few places: one -infinity anywhere, some
    in every piece, a padded end, most of the row unmasked ahead of both; the other way
    round; and both masks by halves and mixed."""
    logits, uniform = rows_of(9, vocab, seed)
    g = gen(seed + 1)
    at = torch.arange(vocab)
    rare = torch.rand(vocab, generator=g) < 0.005
    keep = at % 400 == 7
    for row in logits[:4]:
        row[~keep] = mask
    logits[0, vocab // 3] = -float("inf")
    logits[1, rare] = -float("inf")
    logits[2, -300:] = -float("inf")
    logits[3, 10:310] = -float("inf")
    logits[4, vocab // 4:] = mask
    logits[4, rare & (at > vocab // 4)] = -float("inf")
    logits[5, ~keep] = -float("inf")
    logits[5, rare] = mask
    logits[6, 600:vocab // 2], logits[6, vocab // 2:] = mask, -float("inf")
    logits[7, ~keep] = mask
    logits[7, (torch.rand(vocab, generator=g) < 0.45) & ~keep] = -float("inf")
    logits[8, ~keep] = mask
    logits[8, ::7] = -float("inf")
    return logits, uniform


@pytest.mark.parametrize("vocab", [30000, 151936, 262147])
@pytest.mark.parametrize("mask", [LOWEST, -1e4, -30.0])
def test_a_finite_mask_beside_minus_infinity(batch, dev, vocab, mask):  # noqa: F811
    logits, uniform = masked(vocab, mask, vocab)
    check(batch, dev, logits, uniform)
    check(batch, dev, logits, uniform, **settings(9, 3))
    check(batch, dev, logits, uniform, temperature=[1e3] * 9)


@pytest.mark.parametrize("vocab,many", [(40000, 20000), (40000, 35000), (151936, 20000),
                                        (151936, 60000), (151936, 140000), (262147, 200000)])
def test_one_value_above_the_lowest_with_many_tokens(batch, dev, vocab, many):  # noqa: F811
    """Zeros, a positive and a negative number with lower ones beneath; a number and its
    opposite; three numbers of the lot."""
    logits, uniform = rows_of(6, vocab, many)
    g = gen(many)
    for i, value in enumerate([0.0, 3.0, -2.0]):
        logits[i, torch.randperm(vocab, generator=g)[:many]] = value
    at = torch.randperm(vocab, generator=g)
    logits[3, at[:many // 2]], logits[3, at[many // 2:many]] = 1.5, -1.5
    logits[4, at[:many // 2]], logits[4, at[many // 2:many]] = 0.0, -0.0
    third = many // 3
    for k in range(3):
        logits[5, at[k * third:(k + 1) * third]] = k - 1.0
    check(batch, dev, logits, uniform)
    check(batch, dev, logits, uniform, **settings(6, 4))
    check(batch, dev, logits, uniform, top_k=[many // 2, many - 1, many, many + 1, 7, vocab])


def test_a_rare_lower_value_beside_a_mask_costs_little(batch, dev):  # noqa: F811
    """A finite mask is counted as fast with a -infinity beside it as without; where its
    counts did not fit, the row would be read again some hundred times."""
    logits, uniform = rows_of(16, 151936, 5)
    logits[:, 3000:] = -1e4
    d = {"uniform": torch.tensor(uniform).to(dev),
         "tokens": torch.empty(16, dtype=torch.int32, device=dev),
         "workspace": torch.zeros(batch.sample_workspace_bytes(16, 151936), dtype=torch.uint8,
                                  device=dev)}

    def least(x):
        x, times = x.to(dev), []
        for _ in range(12):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                batch.sample(x, **d)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    alone = least(logits)
    for places in ([5000], [151935], range(4000, 4300), range(3000, 151936, 200)):
        beside = logits.clone()
        beside[:, list(places)] = -float("inf")
        assert least(beside) < 4 * alone, places
