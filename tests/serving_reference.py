"""Plain float64 forms of the operators on drafted tokens and of eviction, for one
(batch, head) slice, and the bounds that the kernels' roundings give.  Tests only;
tests/test_serving_reference.py pins them against the oracle's decode step."""

from __future__ import annotations

import math

import torch

EPS = 1e-9
LOG2E = 1.4426950408889634


def chain_of(parents, i: int):
    """Node i's chain from the context down to i, or None for an absent node."""
    chain = []
    while i != -1:
        if not (0 <= i < len(parents)) or (chain and i >= chain[-1]):
            return None
        chain.append(i)
        i = parents[i]
    return chain[::-1]


def tree_f64(q, k, v, committed, length: int, parents):
    """(out (N, D), lse (N,), spread (N, D)) of one slice: every node by decoding its
    path token by token.  spread: sum of the weights times |v|, what a relative
    error of the weights is multiplied with."""
    n, d = q.shape
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(n, d, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    lse = torch.full((n,), math.inf, dtype=torch.float64, device=q.device)
    for i in range(n):
        chain = chain_of(list(parents), i)
        if chain is None:
            continue
        demand = torch.cat([committed[:length].double(), torch.zeros(len(chain), dtype=torch.float64, device=q.device)])
        rows = torch.tensor(list(range(length)) + [length + c for c in chain], device=q.device)
        for step, node in enumerate(chain):
            see = rows[: length + step + 1]
            a = (k[see] @ q[node]) / math.sqrt(d)
            p = torch.softmax(a, dim=0)
            demand[: length + step + 1] += p
        share = p / (demand + EPS)
        w = share / (share.sum() + EPS)
        out[i], spread[i] = w @ v[rows], w @ v[rows].abs()
        lse[i] = torch.logsumexp(a, dim=0) * LOG2E
    return out, lse, spread


def accept_f64(q, k, committed, length: int, lse, path):
    """(committed over [0, length + A), positions of the accepted rows) of one slice."""
    d = q.shape[1]
    at = torch.tensor(list(path), device=q.device)
    rows = torch.cat([k[:length], k[length + at]]).double()
    p = torch.exp2((q[at].double() @ rows.T) * (LOG2E / math.sqrt(d)) - lse[at].double()[:, None])
    new = torch.cat([committed[:length].double() + p[:, :length].sum(0), p[:, length:].tril().sum(0)])
    return new, length + at


def evict_f64(committed, length: int, keep: int, first: int, recent: int):
    """The kept positions of one slice, by an explicit order: demand down (NaN on
    top), then position up."""
    vals = committed[:length].double().tolist()
    key = lambda j: (0 if math.isnan(vals[j]) else 1, 0.0 if math.isnan(vals[j]) else -vals[j], j)  # noqa: E731
    mid = sorted(range(first, length - recent), key=key)[: keep - first - recent]
    return list(range(first)) + sorted(mid) + list(range(length - recent, length))


def score_error(q, k, d: int) -> float:
    """Bound on an affinity's error in log2 units: an fp32 sum of d exact products
    and one scaling, u = 2^-24 each, of the largest sum of |q||k| (times 2 for the
    order within matrix instructions)."""
    big = (q.double().abs() @ k.double().abs().transpose(-1, -2)).max().item() * LOG2E / math.sqrt(d)
    return 2 * (d + 8) * 2.0 ** -24 * big


def out_bound(out, spread, dtype, delta: float):
    """Elementwise bound on a node's output.  u: half a step of the outputs' type.
    The output is rounded once (u |out|); the shares are rounded to the type of the
    product's operands (u; bf16 and fp16 only), and their relative error from the
    affinities and lse (ln 2 delta each, both in the bid and in the demand), the
    demand's split into two bf16 parts (2^-16, 16-bit types only), exp2, log2 and
    rcp (2^-20 together) multiplies the spread, once for the sum of share v and
    once for the sum of the shares."""
    u = torch.finfo(dtype).eps / 2
    share = (u + 2.0 ** -16 if dtype != torch.float32 else 0.0) + 4 * delta + 2.0 ** -20
    return u * out.abs() + (2 * share) * spread + 1e-9
