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
