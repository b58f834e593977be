"""4-bit weights (infer_hip_gemv_w4a16) from their definition, in torch."""
import torch

COLUMN = (0, 2, 4, 6, 1, 3, 5, 7)  # of each nibble of a dword


def pack(q, scales):
    """Packed weight bytes and tiled scales of int8 q [N, K] and BF16 scales."""
    n, k = q.shape
    rows, cols = -(-n // 16) * 16, -(-k // 128) * 128
    u = torch.full((rows, cols), 8, dtype=torch.uint8)
    u[:n, :k] = (q + 8).to(torch.uint8)
    out = torch.zeros((rows // 16, cols // 128, 4, 16, 4), dtype=torch.int64)
    for nibble, c in enumerate(COLUMN):
        # [tile row, r, tile, i, b] -> [tile row, tile, b, r, i]
        col = u.view(rows // 16, 16, cols // 128, 4, 4, 8)[..., c].permute(0, 2, 4, 1, 3)
        out |= col.to(torch.int64) << (4 * nibble)
    packed = torch.stack([(out >> (8 * i)) & 255 for i in range(4)], dim=-1).to(torch.uint8)
    s = torch.zeros((rows, scales.shape[1]), dtype=torch.bfloat16)
    s[:n] = scales
    return packed.reshape(-1), s.view(rows // 16, 16, -1).transpose(1, 2).contiguous().view(-1)


def unpack(packed, n, k):
    """int8 q [n, k] of packed weight bytes (whole tiles of rows)."""
    words = packed.view(n // 16, -(-k // 128), 4, 16, 4, 4).to(torch.int64)
    dword = sum(words[..., i] << (8 * i) for i in range(4))  # [tile row, tile, b, r, i]
    u = torch.stack([(dword >> (4 * COLUMN.index(c))) & 15 for c in range(8)], dim=-1)
    # -> [tile row, r, tile, i, b, column]
    return (u.permute(0, 3, 1, 4, 2, 5).reshape(n, -1)[:, :k] - 8).to(torch.int8)


def product(q, scales, group, bias, x):
    """(Y in 64 bits, the bound on its FP32 sums): a group's sum is taken of
    products as large as 31 |x| (the elements are held as 16 + u, u = q + 8, and
    24 times the group's sum of x taken off), in 2 `group` roundings of 2^-24,
    and the scaled sums of K / group groups added in as many."""
    n, k = q.shape
    s = scales.double()
    w = q.double() * s.repeat_interleave(group, dim=1)
    y = x.double() @ w.t()
    ax = x.double().abs()
    by_group = ax.view(x.shape[0], k // group, group).sum(dim=2) @ s.abs().t()
    bound = by_group * 31 * 2 * group * 2.0 ** -24
    bound += (ax @ w.abs().t()) * (k // group + 2) * 2.0 ** -24
    if bias is not None:
        y = y + bias.double()
        bound = bound + bias.double().abs() * 2.0 ** -23
    return y, bound
