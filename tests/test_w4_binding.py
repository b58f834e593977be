"""What gemv_w4a16 of the Python binding refuses before the C call: tensors that
are too short for the packed forms, of other types, or not on the current GPU."""
import pytest
import torch

import w4_ref

N, K, GROUP, TOKENS = 37, 160, 32, 3  # rows and columns that do not fill their tiles


def args(dev="cpu", **change):
    packed, tiled = w4_ref.pack(torch.zeros((N, K), dtype=torch.int8),
                                torch.ones((N, K // GROUP), dtype=torch.bfloat16))
    f = dict(weight=packed, scales=tiled, group_size=GROUP,
             bias=torch.zeros(N, dtype=torch.bfloat16), input=torch.zeros((TOKENS, K), dtype=torch.bfloat16),
             output=torch.zeros((TOKENS, N), dtype=torch.bfloat16), tokens=TOKENS, out_features=N,
             in_features=K)
    f.update(change)
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in f.items()}


BAD = [("weight", lambda t: t[:N * K // 2], "bytes"),  # not padded to whole tiles
       ("weight", lambda t: t[:-1], "bytes"), ("scales", lambda t: t[:N * (K // GROUP)], "bytes"),
       ("scales", lambda t: t[:-1], "bytes"), ("bias", lambda t: t[:-1], "bytes"),
       ("input", lambda t: t[:2], "bytes"), ("output", lambda t: t[:2], "bytes"),
       ("scales", lambda t: t.float(), "scales"), ("input", lambda t: t.float(), "input"),
       ("output", lambda t: t.float(), "output"), ("bias", lambda t: t.float(), "bias"),
       ("input", lambda t: t.half(), "input"), ("weight", lambda t: t.float(), "weight")]


@pytest.mark.parametrize("name,change,why", BAD)
def test_sizes_and_types_are_refused(hip, name, change, why):
    good = args()
    # the other tensors as addresses, which are not looked at and never followed
    rest = {k: 4096 if isinstance(v, torch.Tensor) else v for k, v in good.items()}
    with pytest.raises(hip.InferError, match=why):
        hip.gemv_w4a16(**dict(rest, **{name: change(good[name])}))


def test_tensors_off_the_gpu_are_refused(hip):
    with pytest.raises(hip.InferError, match="GPU"):
        hip.gemv_w4a16(**args())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["weight", "scales", "bias", "input", "output"])
def test_one_tensor_off_the_gpu_or_not_contiguous_is_refused(hip, dev, name):
    good = args(dev)
    hip.gemv_w4a16(**good)
    with pytest.raises(hip.InferError, match="GPU"):
        hip.gemv_w4a16(**dict(good, **{name: good[name].cpu()}))
    apart = torch.stack([good[name], good[name]], dim=-1)[..., 0]
    with pytest.raises(hip.InferError, match="contiguous"):
        hip.gemv_w4a16(**dict(good, **{name: apart}))


@pytest.mark.gpu
def test_larger_buffers_words_and_addresses_are_taken(hip, dev):
    """Room to spare, scales and activations as 16-bit integers, plain addresses."""
    g = torch.Generator().manual_seed(1)
    q = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
    s = torch.rand((N, K // GROUP), generator=g).to(torch.bfloat16)
    packed, tiled = (t.to(dev) for t in w4_ref.pack(q, s))
    x = torch.randn((TOKENS, K), generator=g).to(torch.bfloat16).to(dev)
    want = torch.empty((TOKENS, N), dtype=torch.bfloat16, device=dev)
    hip.gemv_w4a16(packed, tiled, GROUP, None, x, want, TOKENS, N, K)
    out = torch.empty((TOKENS + 1, N), dtype=torch.int16, device=dev)
    hip.gemv_w4a16(torch.cat([packed, packed]), tiled.view(torch.int16), GROUP, None,
                   x.view(torch.int16), out, TOKENS, N, K)
    assert torch.equal(out[:TOKENS], want.view(torch.int16))
    hip.gemv_w4a16(packed.data_ptr(), tiled.data_ptr(), GROUP, None, x.data_ptr(), out.data_ptr(),
                   TOKENS, N, K)
    assert torch.equal(out[:TOKENS], want.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(tokens=0), dict(tokens=17), dict(group_size=48),
                                    dict(group_size=0), dict(out_features=0), dict(in_features=0),
                                    dict(in_features=-128)])
def test_shapes_are_refused_by_the_operator(hip, dev, change):
    with pytest.raises(hip.InferError):
        hip.gemv_w4a16(**dict(args(dev), **change))
