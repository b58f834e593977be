"""infer_hip_gemv_w4a16 against 64 bits: group sizes, token counts, rows that
do not fill a tile, columns that do not fill one, values at the ends of their
range, activations that are huge, infinite or NaN, captured graphs."""
import math
import os
import subprocess

import pytest
import torch

import w4_ref as ref

pytestmark = pytest.mark.gpu


def make(n, k, group, tokens, seed, bias=False):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    s = ((torch.rand((n, k // group), generator=g) + 0.1) * 0.02).to(torch.bfloat16)
    s[::3] *= -1  # nothing asks scales to be positive
    x = torch.randn((tokens, k), generator=g).to(torch.bfloat16)
    b = torch.randn(n, generator=g).to(torch.bfloat16) if bias else None
    return q, s, x, b


def run(hip, dev, q, s, group, b, x, spare=3):
    n, k = q.shape
    tokens = x.shape[0]
    packed, tiled = ref.pack(q, s)
    out = torch.full((tokens + spare, n), 5.0, dtype=torch.bfloat16, device=dev)
    hip.gemv_w4a16(packed.to(dev), tiled.to(dev), group, None if b is None else b.to(dev),
                   x.to(dev), out, tokens, n, k)
    got = out.cpu()
    assert (got[tokens:] == 5).all()
    return got[:tokens]


def check(got, y, bound):
    err = (got.double() - y).abs()
    assert (err <= y.abs() * 2.0 ** -8 + bound * (1 + 2.0 ** -8)).all(), float(err.max())


@pytest.mark.parametrize("n,k,group", [
    (1, 32, 32), (15, 32, 32), (16, 64, 64), (17, 96, 32), (33, 128, 128), (100, 192, 64),
    (257, 160, 32), (896, 896, 64), (896, 896, 128), (130, 4864, 64), (896, 4864, 128),
    (70, 8960, 32), (1000, 1088, 64), (4864, 896, 32), (5000, 1536, 128), (513, 9088, 64),
    (20, 33 * 128, 128), (48, 20480, 64)])
@pytest.mark.parametrize("tokens", [1, 2, 5, 16])
def test_product(hip, dev, n, k, group, tokens):
    q, s, x, b = make(n, k, group, tokens, n + k + tokens, bias=tokens % 2 == 1)
    check(run(hip, dev, q, s, group, b, x), *ref.product(q, s, group, b, x))


@pytest.mark.parametrize("tokens", list(range(1, 17)))
def test_every_token_count(hip, dev, tokens):
    q, s, x, b = make(50, 384, 64, tokens, tokens, bias=True)
    check(run(hip, dev, q, s, 64, b, x), *ref.product(q, s, 64, b, x))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_rows(hip, dev, group):
    """As many rows as a vocabulary, not a multiple of anything."""
    q, s, x, b = make(151931, 256, group, 3, group)
    check(run(hip, dev, q, s, group, b, x), *ref.product(q, s, group, b, x))


# Whole row tiles a wave (65536 rows up; 32768 for 9 tokens up and long K): one token,
# a few, sixteen; groups that end inside a column tile; rows that end inside a tile or
# a 4-row piece; LDS for three, two and one workgroup a CU, and too little.  Pairs of
# row tiles (24576 rows up; 16384 for 9 tokens up) with one and several column tiles a
# wave, for up to 4, 8 and 16 tokens.
@pytest.mark.parametrize("n,k,group,tokens", [
    (33001, 160, 32, 16), (32773, 1088, 64, 1), (40008, 4096, 128, 16), (33000, 96, 32, 2),
    (34567, 2432, 64, 9), (50001, 1536, 64, 4), (32768, 32, 32, 1), (33000, 8960, 64, 16),
    (20001, 384, 64, 12), (18000, 4864, 128, 16), (17001, 3168, 32, 9), (20003, 2048, 32, 8),
    (98305, 160, 32, 1), (98319, 1088, 64, 4), (98306, 96, 32, 3), (99001, 416, 32, 8),
    (100004, 128, 128, 16), (24577, 1088, 64, 5), (24580, 96, 32, 1), (30001, 2432, 32, 4),
    (33001, 160, 32, 8), (33017, 1184, 32, 16), (26011, 192, 64, 7), (65537, 1504, 32, 2), (65600, 64, 64, 1)])
def test_product_of_many_rows(hip, dev, n, k, group, tokens):
    q, s, x, b = make(n, k, group, tokens, n + k, bias=tokens % 2 == 0)
    got = run(hip, dev, q, s, group, b, x)
    y, bound = ref.product(q.to(dev), s.to(dev), group, None if b is None else b.to(dev), x.to(dev))
    check(got, y.cpu(), bound.cpu())


@pytest.mark.parametrize("tokens", [1, 16])
def test_weights_past_32_bits(hip, dev, tokens):
    """The last rows of more than 2^32 bytes of weights."""
    n, k, group, last = (1 << 18) + 4800, 32768, 64, 48
    g = torch.Generator(device=dev).manual_seed(3)
    packed = torch.randint(0, 256, (n * k // 2,), generator=g, dtype=torch.uint8, device=dev)
    scales = (torch.rand(n * (k // group), generator=g, device=dev) * 0.02).to(torch.bfloat16)
    assert packed.numel() > 1 << 32
    x = torch.randn((tokens, k), generator=g, device=dev).to(torch.bfloat16)
    out = torch.empty((tokens, n), dtype=torch.bfloat16, device=dev)
    hip.gemv_w4a16(packed, scales, group, None, x, out, tokens, n, k)
    for at in (0, n - last):
        q = ref.unpack(packed[at * k // 2:(at + last) * k // 2].cpu(), last, k)
        s = scales[at * (k // group):(at + last) * (k // group)].cpu().view(last // 16, -1, 16)
        s = s.transpose(1, 2).reshape(last, -1)
        check(out[:, at:at + last].cpu(), *ref.product(q, s, group, None, x.cpu()))


@pytest.mark.parametrize("tokens", [1, 3, 16])
@pytest.mark.parametrize("n", [32805, 98341])
def test_infinities_in_many_rows(hip, dev, n, tokens):
    """The forms for many rows: the last token has an infinity and a NaN apart."""
    k, group = 256, 64
    q, s, x, b = make(n, k, group, tokens, 77, bias=True)
    x[-1, 200] = math.inf
    got = run(hip, dev, q, s, group, b, x).double()
    if tokens > 1:
        check(got[:-1], *ref.product(q, s, group, b, x[:-1]))
    want = math.inf * (q[:, 200].double() * s[:, 200 // group].double())
    assert torch.equal(got[-1].isnan(), want.isnan())
    assert torch.equal(got[-1][~want.isnan()], want[~want.isnan()])
    x[-1, 3] = math.nan
    assert run(hip, dev, q, s, group, b, x)[-1].isnan().all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_value_at_every_column(hip, dev, group):
    """One-hot activations read single weights back: exact."""
    n, k = 40, 256
    q = ((torch.arange(n)[:, None] * 5 + torch.arange(k)[None] * 3) % 16 - 8).to(torch.int8)
    s = torch.exp2(torch.arange(n * (k // group)).view(n, -1) % 7 - 3.0).to(torch.bfloat16)
    want = q.double() * s.double().repeat_interleave(group, dim=1)
    for at in range(0, k, 16):
        x = torch.zeros((16, k), dtype=torch.bfloat16)
        x[torch.arange(16), at + torch.arange(16)] = 1
        got = run(hip, dev, q, s, group, None, x)
        assert torch.equal(got.double(), want[:, at:at + 16].t())


@pytest.mark.parametrize("value", [-8, 7, 0])
def test_constant_weights(hip, dev, value):
    q = torch.full((37, 512), value, dtype=torch.int8)
    _, s, x, _ = make(37, 512, 64, 4, 1)
    check(run(hip, dev, q, s, 64, None, x), *ref.product(q, s, 64, None, x))


@pytest.mark.parametrize("special", [math.inf, -math.inf, math.nan, 3.0e38, -3.3e38])
@pytest.mark.parametrize("tokens", [1, 3])
def test_activations_at_the_ends_of_their_range(hip, dev, special, tokens):
    """The last token holds one such value: as the sum's definition in FP32
    says, and the other tokens are not touched."""
    q, s, x, b = make(50, 1024, 64, tokens, 8, bias=True)
    q[:20, 700] = torch.arange(20, dtype=torch.int8) % 16 - 8
    x[-1, 700] = special
    got = run(hip, dev, q, s, 64, b, x).double()
    if tokens > 1:
        y, bound = ref.product(q, s, 64, b, x[:-1])
        check(got[:-1], y, bound)
    w = q[:, 700].double() * s[:, 700 // 64].double()
    if math.isfinite(special):
        y = ref.product(q, s, 64, b, x)[0][-1]
        # sums of exact products: the large one's rounding is 2^-24 of it
        tol = y.abs() * 2.0 ** -8 + abs(special) * w.abs() * 2.0 ** -20 + 1.0
        assert ((got[-1] - y).abs() <= tol).all()
        return
    want = special * w  # 0 x inf is NaN
    assert torch.equal(got[-1].isnan(), want.isnan())
    assert torch.equal(got[-1][~want.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("n,k,group", [(50, 96, 32), (70, 1088, 64), (25000, 160, 32)])
@pytest.mark.parametrize("tokens", [1, 5, 9])
@pytest.mark.parametrize("special", [math.inf, 3.0e38])
def test_column_tiles_that_end_before_their_last_group(hip, dev, n, k, group, tokens, special):
    """Nothing of a token's first columns comes in for columns past K."""
    q, s, x, b = make(n, k, group, tokens, 21, bias=True)
    q[0, 0], q[1, 0] = 0, 5
    x[0, 0] = special
    got = run(hip, dev, q, s, group, b, x).double()
    if tokens > 1:
        check(got[1:], *ref.product(q, s, group, b, x[1:]))
    w = q[:, 0].double() * s[:, 0].double()
    if math.isfinite(special):
        y, bound = ref.product(q, s, group, b, x[:1])
        # q s x in FP32, of sums whose terms are as large as the first
        check(got[:1], y, bound + (w * special).abs() * (k + 2) * 2.0 ** -24)
    else:
        want = special * w
        assert torch.equal(got[0].isnan(), want.isnan())
        assert torch.equal(got[0][~want.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("tokens", [1, 8])
def test_quantised_weights(hip, dev, tokens):
    """FP32 weights through the quantiser and the packer to the product, within
    the quantiser's half step of the FP32 product."""
    import numpy as np
    g = torch.Generator().manual_seed(5)
    w = torch.randn((300, 896), generator=g) * 0.02
    x = torch.randn((tokens, 896), generator=g).to(torch.bfloat16)
    for group in (32, 64, 128):
        q, s = hip.quantize_w4a16(w.numpy(), group)
        packed, tiled = hip.pack_w4a16(q, s, group)
        out = torch.empty((tokens, 300), dtype=torch.bfloat16, device=dev)
        hip.gemv_w4a16(torch.from_numpy(packed).to(dev),
                       torch.from_numpy(tiled.view(np.int16)).view(torch.bfloat16).to(dev), group,
                       None, x.to(dev), out, tokens, 300, 896)
        sb = torch.from_numpy(s.view(np.int16)).view(torch.bfloat16)
        y, bound = ref.product(torch.from_numpy(q), sb, group, None, x)
        check(out.cpu(), y, bound)
        # a weight is off by half a step (s / 2) and its scale's rounding (7 s 2^-8)
        step = sb.double().repeat_interleave(group, dim=1) * (0.5 + 7 * 2.0 ** -8) * (1 + 2.0 ** -7)
        far = (y - x.double() @ w.double().t()).abs()
        assert (far <= x.double().abs() @ step.t()).all()


def test_captured(hip, dev):
    q, s, x, b = make(896, 4864, 64, 4, 3, bias=True)
    packed, tiled = (t.to(dev) for t in ref.pack(q, s))
    dx, db = x.to(dev), b.to(dev)
    out = torch.zeros((4, 896), dtype=torch.bfloat16, device=dev)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hip.gemv_w4a16(packed, tiled, 64, db, dx, out, 4, 896, 4864)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        hip.gemv_w4a16(packed, tiled, 64, db, dx, out, 4, 896, 4864)
    for seed in range(3):
        x = torch.randn((4, 4864), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
        dx.copy_(x)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out.cpu(), *ref.product(q, s, 64, b, x))
        eager = torch.empty_like(out)
        hip.gemv_w4a16(packed, tiled, 64, db, dx, eager, 4, 896, 4864)
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))


def test_cpp_face(dev):
    binary = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_w4a16")
    assert os.path.exists(binary), "build() compiles tests/cpp/test_w4a16"
    out = subprocess.run([binary], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "PASSED" in out.stdout, out.stdout + out.stderr
