"""Plain float64 forms of the 4-bit cache's operators, and the bounds that the kernels' roundings
give.  Tests only; written from the format's definition (include/dilution_hip.h)."""

from __future__ import annotations

import math

import torch

EPS = 1e-9
LOG2E = 1.4426950408889634
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x: torch.Tensor):
    """(codes, scales) of rows (..., D) of any float type, on the CPU: every element's nearest code
    by distance, the lower code where its mantissa bit is even and both are as near."""
    x = x.detach().cpu().double()
    d = x.shape[-1]
    block = min(32, d)
    x = x.unflatten(-1, (d // block, block))
    top = x.abs().amax(dim=-1)
    bad = ~torch.isfinite(x).all(dim=-1)
    frac, power = torch.frexp(torch.where(bad, 1.0, top))                  # top = frac 2^power, frac in [0.5, 1)
    e = torch.where(frac >= 0.875, power - 2, power - 3).clamp(-125, 125)
    e = torch.where(top == 0, -125, e)
    r = torch.ldexp(torch.where(bad[..., None], 0.0, x).abs(), -e[..., None])
    dist = (r[..., None] - torch.tensor(GRID, dtype=torch.float64)).abs()
    low = dist.argmin(dim=-1)                                               # the lower of two as near
    tie = (dist.gather(-1, (low + 1).clamp(max=7)[..., None])[..., 0] == dist.gather(-1, low[..., None])[..., 0]) & (low < 7)
    code = torch.where(tie & (low % 2 == 1), low + 1, low)
    code = code + 8 * torch.signbit(x)
    code = torch.where(bad[..., None], 0, code).flatten(-2).to(torch.uint8)
    scales = torch.where(bad, 255, e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float64 values (..., D) of codes and scales, on their device."""
    grid = torch.tensor([*GRID, *(-g for g in GRID)], dtype=torch.float64, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()
    factor = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    factor = torch.where(scales == 0, 0.0, torch.where(scales == 255, float("nan"), factor))
    return (grid[c].unflatten(-1, (scales.shape[-1], -1)) * factor[..., None]).flatten(-2)


def step_f64(q, k, v, committed, length: int):
    """(out, committed, spread, p) of one slice in float64: q (D,), k and v (cap, D) values.
    spread: the weights times |v|, what a relative error of the weights is multiplied with."""
    a = (k[:length].double() @ q.double()) / math.sqrt(q.shape[0])
    p = torch.softmax(a, dim=0)
    new = committed.double().clone()
    new[:length] += p
    share = p / (new[:length] + EPS)
    w = share / (share.sum() + EPS)
    vd = v[:length].double()
    return w @ vd, new, w @ vd.abs(), p


def share_error(q, k, length: int) -> float:
    """Bound on the relative error of a bid p, and so of a share (p / (c + p + eps) is less than
    proportional to p).  u = 2^-24, an fp32 rounding.  The affinity: a sum of D exact products of
    a query element and a code, scaled and multiplied by log2(e) / sqrt(D): at most D + 8 roundings of
    partial sums no larger than sum |q||k| (twice for the order within v_dot2), and a - lse one
    more of each; the same error enters lse.  The sum of the bids and its logarithm: length / 64
    additions in one lane at most, 16 across lanes and waves.  exp2, log2 and rcp: 2^-22 each."""
    u = 2.0 ** -24
    d = q.shape[-1]
    big = (k[:length].double().abs() @ q.double().abs()).max().item() * LOG2E / math.sqrt(d)
    affinity = 2 * (d + 8) * u * big
    return math.log(2.0) * 2 * affinity + (length / 64 + 16) * u + 3 * 2.0 ** -22


def out_bound(out, spread, dtype, err: float, length: int):
    """Elementwise bound on an output: rounded once to its type; the shares' errors in the sums
    of share v and of the shares (2 err times the spread); those sums' own additions, length / 64 in
    one lane and 16 across lanes and waves, and the products' and the division's roundings."""
    u = torch.finfo(dtype).eps / 2
    sums = 2 * (length / 64 + 24) * 2.0 ** -24
    return u * out.abs() + (1 + u) * (2 * err + sums) * spread + 1e-30
