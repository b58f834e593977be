"""Low-rank adapters (infer_hip_lora_bf16) of numbers that FP32 holds and BF16 does not."""
import pytest
import torch

from test_gpu_lora import batch, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,k,rank", [(3, 64, 8), (20, 64, 32), (64, 64, 64), (5, 1600, 40),
                                           (9, 4104, 128), (300, 64, 16), (900, 64, 104)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_numbers_past_the_largest_of_bf16(batch, dev, tokens, k, rank, sign):  # noqa: F811
    """A x of 2^127 (2 - 2^-9), a number of FP32 that lies nearer to 2^128 than to the
    largest of BF16; times 2^-120 it is 255.75, of which the base takes 255 away."""
    x = torch.zeros((tokens, k), dtype=torch.bfloat16)
    x[:, 0], x[:, k - 1] = 2.0 ** 63, 2.0 ** 63
    a = torch.zeros((1, rank, k), dtype=torch.bfloat16)
    a[0, rank - 1, 0], a[0, rank - 1, k - 1] = 2.0 ** 64 * (2 - 2 ** -7), 2.0 ** 64 * 1.5 * 2 ** -8
    a *= sign
    b = torch.full((1, 40, rank), 2.0 ** -120).to(torch.bfloat16)
    base = torch.full((tokens, 40), -255.0 * sign).to(torch.bfloat16)
    ids = torch.zeros(tokens, dtype=torch.int32)
    out = torch.empty((tokens, 40), dtype=torch.bfloat16, device=dev)
    ws = workspace(batch, tokens, rank, 1, dev)
    batch.lora(x.to(dev), ids.to(dev), [(a.to(dev), b.to(dev), base.to(dev), out)], ws)
    assert (out == 0.75 * sign).all()
    # by the scale; and infinite where FP32 is
    a = (a.float() * 2.0 ** -100).to(torch.bfloat16)
    batch.lora(x.to(dev), ids.to(dev), [(a.to(dev), b.to(dev), base.to(dev), out)], ws,
               scales=torch.tensor([2.0 ** 100], device=dev))
    assert (out == 0.75 * sign).all()
    batch.lora(x.to(dev), ids.to(dev), [(a.to(dev), b.to(dev), base.to(dev), out)], ws,
               scales=torch.tensor([2.0 ** 101], device=dev))
    assert (out == sign * float("inf")).all()
