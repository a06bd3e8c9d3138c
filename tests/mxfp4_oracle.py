"""Microscaled 4-bit floating point in 64 bits on the CPU, from its definition."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantized_values(x):
    """[R, K] -> the fp64 values that 4 bits hold (NaN in a block that is not finite)."""
    R, K = x.shape
    v = x.detach().cpu().double()
    v = torch.cat([v, v.new_zeros(R, -K % 32)], 1).view(R, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    ok = torch.isfinite(top)
    e = torch.floor(torch.log2(torch.where(ok & (top > 0), top, torch.ones_like(top)))) - 2
    e = torch.where(top > 0, e.clamp(min=-127), torch.full_like(e, -127))
    a = torch.where(ok, v.abs(), torch.zeros_like(v)) / 2 ** e
    # the nearest of the eight magnitudes, the even code where two are as near
    d = (a[..., None] - GRID).abs() + torch.tensor([0.0, 1e-13] * 4, dtype=torch.float64)
    q = GRID[d.argmin(-1)] * 2 ** e * torch.where(torch.signbit(v), -1.0, 1.0)
    return torch.where(ok, q, torch.full_like(q, math.nan)).view(R, -1)[:, :K]


def decoded(codes, scales, K):
    """codes [R, 16 nb], scales [R, nb] -> fp64 [R, K]"""
    c = codes.cpu().long()
    q = torch.stack([c % 16, c // 16], 2).flatten(1)
    v = GRID[q % 8] * torch.where(q >= 8, -1.0, 1.0)
    s = 2.0 ** (scales.cpu().double() - 127)
    s = torch.where(scales.cpu() == 255, torch.full_like(s, math.nan), s)
    return (v * s.repeat_interleave(32, 1))[:, :K]


def product_bound(a, b, dtype):
    """How far a @ b in fp32 sums of exact products, rounded once to dtype, may be: one step of 2^-24 for each
    addition, half a step of dtype at the end."""
    k = a.shape[1]
    y = (a @ b).abs()
    return 2.0 ** -24 * (k + 2) * (a.abs() @ b.abs()) + torch.finfo(dtype).eps / 2 * y * (1 + 1e-6) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
