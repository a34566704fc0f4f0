"""The bids of the 4-bit decode step against float64, with a bound from the kernels' own arithmetic: how
they split a query, and how many fp32 roundings a score and a bid take.  Tests only.

A row whose demand was zero holds its bids after a step, so each score is seen through
p_j = 2^(a_j - max a) / sum 2^(a - max a): with affinities of tens of log2 units a bid's relative error
is tens of times its score's.
"""

from __future__ import annotations

import math

import torch

import fp4_reference as ref

PARTS = 8
LOG2E = 1.4426950408889634
U = 2.0 ** -24                                              # half a step of fp32, relative


def blocks(d: int):
    """(blocks of a row, elements of a block)."""
    return d // min(32, d), min(32, d)


def split(q: torch.Tensor) -> torch.Tensor:
    """The query (D,) as PARTS rows of float64: part i the nearest whole multiple of 2^(E - 3 - 5 i) to what
    the parts before leave, E the exponent of the largest element of its block."""
    rest = q.detach().double().cpu().unflatten(-1, blocks(q.shape[-1]))
    _, power = torch.frexp(rest.abs().amax(dim=-1, keepdim=True))           # the largest is 1.m 2^(power - 1)
    parts = []
    for i in range(PARTS):
        unit = torch.ldexp(torch.ones_like(rest), power - 4 - 5 * i)
        part = (rest / unit).round() * unit
        parts.append(part.flatten())
        rest = rest - part
    return torch.stack(parts)


def score_error(q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """Bound on the error of the scores q.k of keys (L, D).  What the parts leave of the query; and the fp32
    additions, since the sum of a part over one block is exact: whole numbers up to 16 times codes.  An
    instruction adds the blocks of 128 products (4, or the row's where it has fewer: the others are 0)
    and what was summed before, each addition off by at most a step (2^-23) of a partial sum; parts i and i + 4
    and the halves of a row share one sum.  Joining the four sums takes two additions of half a step in
    a row.  No partial sum passes T, the sum of |part||k|."""
    parts, q, k = split(q), q.detach().double().cpu(), k.double().cpu().abs()
    n = blocks(q.shape[-1])[0]
    adds = 2 * max(1, n // 4) * min(4, n) - 1
    total = k @ parts.abs().sum(0)
    return (adds + 1) * 2 * U * total + k @ (q - parts.sum(0)).abs()


def bids(q: torch.Tensor, k: torch.Tensor):
    """(p, bound on p's relative error) of the step of query q (D,) over the keys k (L, D) in float64.

    An affinity is a score times log2(e) / sqrt(D), which is off by three roundings, and is rounded itself;
    a - max is rounded once more.  2^x is off by a step.  The sum: of a lane's keys (4 in a chunk of
    1024 keys, one for each 1024 where a workgroup takes the slice) two powers, a product and an addition
    each; three joins over the lanes of one power, one product and six additions; one more step
    of the first kind for each 64 chunks.  Then a division and a product."""
    q64, k = q.detach().double().cpu(), k.double().cpu()
    length, d = k.shape
    scale = LOG2E / math.sqrt(d)
    a = k @ q64 * scale
    p = torch.softmax(a * math.log(2.0), dim=0)
    below = a.max() - a
    e = scale * score_error(q, k) + 4 * U * a.abs() + U * below
    lane = max(4, -(-length // 1024)) + -(-length // (64 * 1024))
    roundings = 6 * lane + 3 * 9 + 2 + 2 + 1
    e = math.log(2.0) * (e + (p * e).sum() + 3 * U * (p * below).sum()) + roundings * U
    return p, torch.expm1(e)


def worst(p: torch.Tensor, want: torch.Tensor, rel: torch.Tensor) -> float:
    """The largest error of bids p over its bound (powers below 2^-126 may count as 0)."""
    return ((p.double().cpu() - want).abs() / (rel * want + 2.0 ** -125)).max().item()


# ---------------------------------------------------------------------------
# inputs that show each part of a query


SPREADS = (0, 6, 12, 20)


def inputs(d: int, length: int, spread: int, seed: int, dtype=torch.float32, reach: float = 40.0):
    """(q (D,), codes, scales) on the CPU.  spread > 0: the first element of every block is the block's largest,
    2^spread above the others, and has code 0 in every key, so that the scores come from the query's later parts.
    The keys' signs follow those of one part each (of q, or none): its products add up.  Affinities
    reach up to `reach`."""
    g = torch.Generator().manual_seed(seed)
    n, block = blocks(d)
    q = torch.randn(d, generator=g)
    if spread:
        q = q * 2.0 ** -spread
        q[::block] = 1.37
    q = q.to(dtype)
    parts = split(q)
    sign = torch.randint(0, 2, (length, d), generator=g)
    for i, row in enumerate((*parts, q.double())):
        at = torch.arange(i, length, PARTS + 2)
        sign[at] = torch.where(row == 0, sign[at], (row < 0).long())
    code = torch.randint(1, 8, (length, d), generator=g)
    if spread:
        code[:, ::block] = 0
    code = (code + 8 * sign).to(torch.uint8)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    scales = (127 - torch.randint(0, 3, (length, n), generator=g)).to(torch.uint8)
    total = ref.values(codes, scales).abs() @ parts.abs().sum(0) * LOG2E / math.sqrt(d)
    return q, codes, scales + math.floor(math.log2(reach / total.max().item()))


def small_query(d: int, length: int, top: int, seed: int, dtype=torch.float32, beside: bool = False, reach: float = 40.0):
    """`inputs` with a query of elements near 2^top (top < 0) and keys of powers as large as 2^125, and one key in
    seven of powers down to 2^-125.  beside: the row's first block is of ordinary size, on keys of ordinary size."""
    q, codes, scales = inputs(d, length, 0, seed, reach=reach / 2)
    n, block = blocks(d)
    power = min(-top, 125 + 127 - int(scales.max()))
    small = torch.ldexp(q, torch.tensor(top)).to(dtype)
    shifted = scales + power
    if beside:
        small[:block] = q[:block].to(dtype)
        shifted[:, 0] = scales[:, 0]
    at = torch.arange(0, length, 7)
    shifted[at] = torch.randint(2, 60, (len(at), n), generator=torch.Generator().manual_seed(seed)).to(torch.uint8)
    return small, codes, shifted


def largest_sums(d: int, length: int, value: float, seed: int, reach: float = 40.0):
    """Every product of a block as large as can be and of one sign, but, in two keys of three, one of the smallest
    code: a third of the keys each with none, a positive and a negative one."""
    g = torch.Generator().manual_seed(seed)
    sign = torch.randint(0, 2, (d,), generator=g)
    q = value * (1 - 2 * sign.float())
    code = (7 + 8 * sign).repeat(length, 1)                 # 6 times the query's sign
    at = torch.randint(0, d, (length,), generator=g)
    kind = torch.arange(length) % 3
    small = 1 + 8 * (sign[at] ^ (kind == 2).long())         # 0.5: the product's sign by kind
    rows = torch.arange(length)[kind > 0]
    code[rows, at[rows]] = small[rows]
    code = code.to(torch.uint8)
    power = math.floor(math.log2(reach / (6 * value * LOG2E * math.sqrt(d))))
    return q, code[:, 0::2] | (code[:, 1::2] << 4), torch.full((length, blocks(d)[0]), 127 + power, dtype=torch.uint8)


# ---------------------------------------------------------------------------
# the kernels' scores redone, with mistakes if asked


def computed_bids(q: torch.Tensor, k: torch.Tensor, part=lambda i, x: x) -> torch.Tensor:
    """The bids from scores as the kernels add them, in fp32; `part(i, x)` gives what is taken for part i (D,)."""
    parts = torch.stack([part(i, x) for i, x in enumerate(split(q))])
    k = k.double().cpu()
    d = q.shape[-1]
    n, block = blocks(d)
    sums = torch.zeros(4, k.shape[0])
    for half in range(max(1, n // 4)):
        for i in range(PARTS):
            for b in range(4 * half, min(n, 4 * half + 4)):
                at = slice(b * block, (b + 1) * block)
                sums[i % 4] += (k[:, at] @ parts[i, at]).float()
    x = (sums[0] + sums[1]) + (sums[2] + sums[3])
    a = (torch.tensor(LOG2E) / torch.tensor(float(d)).sqrt()) * x
    return torch.softmax(a.double() * math.log(2.0), dim=0)
