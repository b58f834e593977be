"""The paged KV cache's operators in 64 bits, from their definitions, on CPU
tensors: what tests/test_gpu_paged.py compares the kernels with."""
import math

import torch

LIMIT = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def rope_table(positions, d, theta=1e6):
    """FP32 (cos, sin) [positions, d / 2, 2]."""
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (
        -2.0 * torch.arange(d // 2, dtype=torch.float64) / d)
    return torch.stack([a.cos(), a.sin()], dim=-1).float()


def rotate(x, cs):
    """(rotated rows, the magnitude their rounding goes by) of [n, heads, d]."""
    x, h = x.double(), x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    big = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1), torch.cat(big, dim=-1)


def fused_free(x, cs):
    """The same rotation in FP32, each operation rounded: what is quantised."""
    x, h = x.float(), x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def held_error(rows, fmt):
    """How far a held element may be from its row's value: half a step of the
    format (BF16 2^-8 and E4M3 2^-4 relative, the latter at least half of its
    smallest step 2^-9; INT8 half of the scale), and a few FP32 roundings of the
    scale and the quotient."""
    if fmt == "bf16":
        return rows.abs() * 2.0 ** -8
    s = rows.abs().amax(dim=-1, keepdim=True) / LIMIT[fmt]
    step = s / 2 if fmt == "int8" else torch.maximum(rows.abs() * 2.0 ** -4, s * 2.0 ** -10)
    return step + rows.abs().amax(dim=-1, keepdim=True) * 2.0 ** -21


def attend(q, k, v):
    """Attention of q [heads, d] over k, v [kv heads, n, d] (float64): the
    output, sum p |v| / sum p, and the largest sum |q k| / sqrt(d) of a head."""
    heads, d = q.shape
    kv, n, _ = k.shape
    if n == 0:
        z = torch.zeros((heads, d), dtype=torch.float64)
        return z, z, 0.0
    q = q.double().view(kv, heads // kv, d)
    s = q @ k.transpose(1, 2) / math.sqrt(d)
    p = torch.softmax(s, dim=-1)
    big = float((q.abs() @ k.abs().transpose(1, 2)).max()) / math.sqrt(d)
    return (p @ v).view(heads, d), (p @ v.abs()).view(heads, d), big


def attend_tolerance(out, mean_abs, big, n, d):
    """Roundings of the operator: the output to BF16 (2^-8 of it); every weight
    times value scale to BF16 (2^-8 of sum p |v|); scores, sums of d products in
    FP32 (d 2^-24 of sum |q k|, in p and in the normaliser), their exponential and
    the sums over n keys (n 2^-24, 2^-20 for the rest)."""
    each = 2.0 ** -8 + 2 * (d * big + n) * 2.0 ** -24 + 2.0 ** -20
    return out.abs() * 2.0 ** -8 + mean_abs * each + 1e-30


class Pool:
    """Random pages and their values in 64 bits."""

    def __init__(self, fmt, pages, page, kv, d, gen, std=1.0):
        self.fmt, self.page = fmt, page
        shape = (pages, kv, page, d)
        self.scales = [None, None]
        self.parts = []
        for i in range(2):
            x = torch.randn(shape, generator=gen) * std
            if fmt == "bf16":
                self.parts.append(x.to(torch.bfloat16))
                continue
            s = x.abs().amax(dim=-1) / LIMIT[fmt]
            q = x / s[..., None]
            self.parts.append(q.round().clamp(-127, 127).to(torch.int8) if fmt == "int8"
                              else q.clamp(-448, 448).to(torch.float8_e4m3fn))
            self.scales[i] = s

    def values(self, i):
        x = self.parts[i].float().double()
        return x if self.scales[i] is None else x * self.scales[i].double()[..., None]

    def rows(self, i, table_row, n):
        """Positions [0, n) of a sequence, [kv heads, n, d]."""
        if n <= 0:
            return self.values(i)[0][:, :0]
        pages = [int(p) for p in table_row[:-(-n // self.page)]]
        picked = self.parts[i].view(torch.uint8)[pages] if self.fmt == "fp8" else self.parts[i][pages]
        x = (picked.view(torch.float8_e4m3fn) if self.fmt == "fp8" else picked).float().double()
        if self.scales[i] is not None:
            x = x * self.scales[i][pages].double()[..., None]
        return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n]

    def to_device(self, paged, dev):
        sc = [None if s is None else s.to(dev) for s in self.scales]
        return paged.KvPages(self.parts[0].to(dev), self.parts[1].to(dev), *sc)


def tables(lengths, page, gen, spare=3, width=None):
    """(block table int32 with -1 behind each sequence's pages, pool size)."""
    counts = [-(-max(n, 0) // page) for n in lengths]
    width = width or max(1, max(counts))
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen).to(torch.int32)
    t, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    for i, c in enumerate(counts):
        t[i, :c] = order[at:at + c]
        at += c
    return t, total
