"""Serving operators on a dilution decode cache, case by case: attention for a tree of
drafted tokens, the acceptance of one of its paths, and eviction by demand.

    own                  False: run() computes the plain form; True: the framework's kernels
    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call: queries, caches, trees
    run(state)           one pass through an operator, with its outputs
    work(case)           bytes and operations that one pass cannot do without
    exact(case, seed)    the outputs in float64, from the definitions

Kinds of cases (B sequences of H heads of width D over a cache of L keys):

    tree    N drafted tokens of every sequence, each seeing the cache, its ancestors among
            the drafted and itself, with the demand that its ancestors add.  The queries are
            views of a (B, N, H D) projection, as an attention layer calls it.
    accept  A of the N drafted tokens become part of the cache: the demand takes their bids,
            their rows move together.
    evict   the cache shrinks from L to `keep` keys: the first `first`, the last `recent`, and
            those of the rest with the most demand.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-9
LOG2E = 1.4426950408889634
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kernels():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dilution-attention_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dilution import kernels

    return kernels


def _tree(name, b, h, length, n, d=64, prec="bf16", shape="bushy", padded=False):
    return {"name": name, "kind": "tree", "b": b, "h": h, "len": length, "n": n, "d": d, "prec": prec, "shape": shape,
            "padded": padded}


def _accept(name, b, h, length, n, count, d=64, prec="bf16"):
    return {"name": name, "kind": "accept", "b": b, "h": h, "len": length, "n": n, "count": count, "d": d, "prec": prec}


def _evict(name, b, h, length, keep, first, recent, room=0, d=64, prec="bf16", quiet=0.0):
    return {"name": name, "kind": "evict", "b": b, "h": h, "len": length, "keep": keep, "first": first, "recent": recent,
            "room": room, "d": d, "prec": prec, "quiet": quiet}


def listed():
    return [
        # one sequence at a short context checks a handful of drafted tokens: launches and latency count
        _tree("tree_short", 1, 16, 1000, 8),
        # serving 8 sequences at a 16K context, a tree of 32 drafted tokens each
        _tree("tree_16k", 8, 16, 16384, 32),
        # odd head counts, lengths and trees, heads of 128 in fp16; the sequences' trees differ in size
        _tree("tree_ragged", 3, 5, 5003, 13, d=128, prec="fp16", padded=True),
        # fp32 activations and caches
        _tree("tree_fp32", 2, 8, 4096, 16, prec="fp32"),
        # the largest trees over long contexts
        _tree("tree_64k", 8, 16, 65536, 64),
        # a draft without branches at a long context, one sequence
        _tree("tree_chain_128k", 1, 16, 131072, 5, shape="chain"),
        # the short context's step accepts three of its tokens
        _accept("accept_short", 1, 16, 1000, 8, 3),
        # long contexts of 8 sequences accept six tokens
        _accept("accept_64k", 8, 16, 65536, 32, 6),
        # odd counts, narrow heads, fp32
        _accept("accept_fp32", 2, 12, 9001, 24, 5, d=32, prec="fp32"),
        # one sequence halves a short cache
        _evict("evict_short", 1, 16, 4096, 2048, 4, 256),
        # long prompts of 4 sequences shrink to a quarter, with room for new tokens
        _evict("evict_128k", 4, 16, 131072, 32768, 4, 1024, room=1024),
        # odd sizes, wide heads, fp32, many keys that hold no demand at all (ties)
        _evict("evict_ragged", 3, 5, 7001, 2999, 3, 501, room=77, d=128, prec="fp32", quiet=0.7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["tree", "tree", "accept", "evict"])
        b, h, length = _log_int(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), _log_int(rng, 16, 131072)
        d = rng.choice([16, 32, 64, 64, 64, 128, 128, 256])
        prec = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        c = {"kind": kind, "b": b, "h": h, "len": length, "d": d, "prec": prec}
        if kind == "evict":
            keep = max(1, min(length, int(length * rng.uniform(0.1, 0.95))))
            first = rng.randint(0, min(keep, 16))
            recent = int((keep - first) * rng.choice([0.0, 0.1, 0.25, 0.5]))
            c.update(keep=keep, first=first, recent=recent, room=rng.choice([0, 1, 64, 500]), quiet=rng.choice([0.0, 0.0, 0.3, 0.8]))
        else:
            c["n"] = _log_int(rng, 1, 64)
            if kind == "tree":
                c.update(shape=rng.choice(["bushy", "bushy", "chain", "flat"]), padded=rng.choice([False, True]))
            else:
                c["count"] = rng.randint(1, min(c["n"], 12))
        nodes = c.get("n", 1)
        if work(c)["bytes"] <= 2.1e9 and b * h * nodes * length <= 128 * 64 * 65536:
            return c


# ---------------------------------------------------------------------------
# inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _demand(g, b, h, length, capacity, quiet=0.0):
    """A demand vector like the one that `length` rows leave: early keys hold more; zero from
    the first free position on.  quiet: the share of keys whose bids all fell below fp32."""
    pos = torch.arange(length, device=DEV, dtype=torch.float32)
    com = torch.zeros(b, h, capacity, device=DEV)
    noise = torch.randn(b, h, length, generator=g, device=DEV) * 0.5
    com[:, :, :length] = torch.log((length + 1) / (pos + 1.0)) * torch.exp(noise)
    if quiet:
        com[:, :, :length] *= torch.rand(b, h, length, generator=g, device=DEV) >= quiet
    return com


def _parents(case, seed):
    """(B, N) int32 parents: node 0 hangs on the context, the others on an earlier node; -2
    marks the padding of a smaller tree."""
    b, n = case["b"], case["n"]
    g = torch.Generator().manual_seed(seed)
    parents = torch.full((b, n), -1, dtype=torch.int32)
    shape = case.get("shape", "bushy")
    for i in range(1, n):
        if shape == "chain":
            parents[:, i] = i - 1
        elif shape == "flat":
            parents[:, i] = 0
        else:
            parents[:, i] = i - 1 - (torch.rand(b, generator=g) * min(i, 6)).int()
    if case.get("padded"):
        sizes = torch.randint((n + 1) // 2, n + 1, (b,), generator=g)
        parents[torch.arange(n) >= sizes[:, None]] = -2
    return parents.to(DEV)


def _tree_inputs(case, seed):
    g, dt = _gen(seed), _TYPES[case["prec"]]
    b, h, length, n, d = case["b"], case["h"], case["len"], case["n"], case["d"]
    capacity = length + n
    q = _randn(g, (b, n, h * d), dt).view(b, n, h, d).transpose(1, 2)
    k, v = (_randn(g, (b, h, capacity, d), dt) for _ in range(2))
    return q, k, v, _demand(g, b, h, length, capacity), _parents(case, seed)


def _accept_inputs(case, seed):
    """The step before has left the row statistics; the accepted path starts at node 0."""
    q, k, v, com, parents = _tree_inputs(case, seed)
    g = torch.Generator().manual_seed(seed + 1)
    rest = [torch.randperm(case["n"] - 1, generator=g)[: case["count"] - 1].sort().values + 1 for _ in range(case["b"])]
    path = torch.cat([torch.zeros(case["b"], 1, dtype=torch.int64), torch.stack(rest)], dim=1)
    # each accepted token hangs on the one accepted before it
    parents.scatter_(1, path[:, 1:].to(DEV), path[:, :-1].to(DEV, torch.int32))
    seen, _ = _seen(parents)
    lse = _lse64(q, k, case["len"], seen).float()
    return q, k, v, com, lse, path.to(DEV, torch.int32)


def _evict_inputs(case, seed):
    g, dt = _gen(seed), _TYPES[case["prec"]]
    b, h, length, d = case["b"], case["h"], case["len"], case["d"]
    k, v = (_randn(g, (b, h, length, d), dt) for _ in range(2))
    return k, v, _demand(g, b, h, length, length, case["quiet"])


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "tree":
        names, values = ("q", "k", "v", "committed", "parents"), _tree_inputs(case, seed)
    elif case["kind"] == "accept":
        names, values = ("q", "k", "v", "committed", "lse", "path"), _accept_inputs(case, seed)
    else:
        names, values = ("k", "v", "committed"), _evict_inputs(case, seed)
    state.update(zip(names, values))
    return state


# ---------------------------------------------------------------------------
# the plain forms


def _seen(parents):
    """(B, N, N): whether node i sees node a (an ancestor, or i itself); (B, N): whether i's
    chain of parents reaches the context."""
    n = parents.shape[1]
    node = torch.arange(n, device=parents.device)
    step = (parents[:, :, None] == node).float() + torch.eye(n, device=parents.device)
    seen = torch.linalg.matrix_power(step, max(n - 1, 1)) > 0
    absent = (parents < -1) | (parents >= node)
    return seen, ~(seen & absent[:, None, :]).any(dim=2)


def _plain_tree(s):
    length, n, d = s["case"]["len"], s["case"]["n"], s["case"]["d"]
    seen, present = _seen(s["parents"])
    mask = torch.nn.functional.pad(seen, (length, 0), value=True)[:, None]
    a = s["q"].float() @ s["k"][:, :, : length + n].float().transpose(2, 3) * (LOG2E / math.sqrt(d))
    a = a.masked_fill(~mask, float("-inf"))
    m = a.amax(dim=3, keepdim=True)
    e = torch.exp2(a - m)
    total = e.sum(dim=3, keepdim=True)
    p = e / total
    demand = s["committed"][:, :, None, : length + n] + seen.float()[:, None] @ p
    share = (p / (demand + EPS)).masked_fill(~mask, 0.0)
    w = share / (share.sum(dim=3, keepdim=True) + EPS)
    out = w @ s["v"][:, :, : length + n].float()
    gone = ~present[:, None, :, None]
    return {"out": out.masked_fill(gone, 0.0).to(s["q"].dtype),
            "lse": (m + torch.log2(total)).masked_fill(gone, float("inf")).squeeze(3)}


def _plain_accept(s):
    case = s["case"]
    length, count, d = case["len"], case["count"], case["d"]
    k, v, com = s["k"], s["v"], s["committed"]
    at = s["path"].long()[:, None, :, None].expand(-1, case["h"], -1, d)
    q, lse = s["q"].gather(2, at).float() * (LOG2E / math.sqrt(d)), s["lse"].gather(2, at[..., 0])[..., None]
    kd, vd = k.gather(2, length + at), v.gather(2, length + at)
    com[:, :, :length] += torch.exp2(q @ k[:, :, :length].float().transpose(2, 3) - lse).sum(dim=2)
    com[:, :, length : length + count] = torch.exp2(q @ kd.float().transpose(2, 3) - lse).tril().sum(dim=2)
    k[:, :, length : length + count], v[:, :, length : length + count] = kd, vd
    return {"k": k, "v": v, "committed": com}


def _kept(case, committed):
    """(B, H, keep) positions, ascending; among equal demands the lowest position stays."""
    length, first, recent = case["len"], case["first"], case["recent"]
    order = committed[:, :, first : length - recent].sort(dim=2, descending=True, stable=True).indices
    heavy = order[:, :, : case["keep"] - first - recent].sort(dim=2).values + first
    rows = torch.arange(length, device=committed.device).expand(*committed.shape[:2], length)
    return torch.cat([rows[:, :, :first], heavy, rows[:, :, length - recent :]], dim=2)


def _plain_evict(s):
    case = s["case"]
    index = _kept(case, s["committed"])
    rows = index[..., None].expand(-1, -1, -1, case["d"])
    pad = (0, 0, 0, case["room"])
    return {"k": torch.nn.functional.pad(s["k"].gather(2, rows), pad), "v": torch.nn.functional.pad(s["v"].gather(2, rows), pad),
            "committed": torch.nn.functional.pad(s["committed"].gather(2, index), (0, case["room"])),
            "index": index.to(torch.int32)}


# ---------------------------------------------------------------------------
# one pass


def _own(s):
    ops, case = _kernels(), s["case"]
    if case["kind"] == "tree":
        out, aux = ops.dilution_tree_step(s["q"], s["k"], s["v"], s["committed"], case["len"], s["parents"], return_aux=True)
        return {"out": out, "lse": aux["lse"]}
    if case["kind"] == "accept":
        ops.dilution_tree_accept(s["q"], s["k"], s["v"], s["committed"], case["len"], s["lse"], s["path"])
        return {"k": s["k"], "v": s["v"], "committed": s["committed"]}
    k, v, com, index = ops.dilution_evict(s["k"], s["v"], s["committed"], case["len"], case["keep"], first=case["first"],
                                          recent=case["recent"], capacity=case["keep"] + case["room"])
    return {"k": k, "v": v, "committed": com, "index": index}


def run(state):
    with torch.no_grad():
        if own:
            return _own(state)
        return {"tree": _plain_tree, "accept": _plain_accept, "evict": _plain_evict}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    size = 4 if case["prec"] == "fp32" else 2
    slices, length, row = case["b"] * case["h"], case["len"], case["d"] * size
    if case["kind"] == "tree":
        n = case["n"]
        return {"bytes": slices * ((length + n) * (2 * row + 4) + n * (2 * row + 4)), "flops": 4 * slices * n * length * case["d"]}
    if case["kind"] == "accept":
        count = case["count"]
        return {"bytes": slices * (length * (row + 8) + count * (6 * row + 8)), "flops": 2 * slices * count * length * case["d"]}
    keep, capacity = case["keep"], case["keep"] + case["room"]
    return {"bytes": slices * (length * 4 + keep * (2 * row + 4) + capacity * (2 * row + 4)), "flops": slices * length}


# ---------------------------------------------------------------------------
# the same in float64


def _lse64(q, k, length, seen):
    """Base-2 row statistics (B, H, N) of the drafted rows, slice by slice."""
    b, h, n, d = q.shape
    lse = torch.empty(b, h, n, device=DEV, dtype=torch.float64)
    for i in range(b):
        for j in range(h):
            a = (q[i, j].double() @ k[i, j, : length + n].double().T) / math.sqrt(d)
            a[:, length:].masked_fill_(~seen[i], float("-inf"))
            lse[i, j] = torch.logsumexp(a, dim=1) * LOG2E
    return lse


def _tree64(q, k, v, com, parents, length):
    """One slice: node after node, the demand carried down each path."""
    n, d = q.shape
    out = torch.zeros(n, d, device=DEV, dtype=torch.float64)
    lse = torch.full((n,), float("inf"), device=DEV, dtype=torch.float64)
    a = (q.double() @ k[: length + n].double().T) / math.sqrt(d)
    com, vd = com[: length + n].double(), v[: length + n].double()
    demand, visible = [None] * n, [None] * n
    for i, parent in enumerate(parents):
        if parent >= i or parent < -1 or (parent >= 0 and demand[parent] is None):
            continue
        visible[i] = (visible[parent] if parent >= 0 else []) + [length + i]
        columns = torch.cat([torch.arange(length, device=DEV), torch.tensor(visible[i], device=DEV)])
        row = a[i, columns]
        lse[i] = torch.logsumexp(row, dim=0) * LOG2E
        p = torch.zeros(length + n, device=DEV, dtype=torch.float64)
        p[columns] = torch.softmax(row, dim=0)
        demand[i] = (demand[parent] if parent >= 0 else com) + p
        share = p / (demand[i] + EPS)
        out[i] = (share / (share.sum() + EPS)) @ vd
    return out, lse


def _exact_tree(case, seed):
    q, k, v, com, parents = _tree_inputs(case, seed)
    out = torch.empty(q.shape, device=DEV, dtype=torch.float64)
    lse = torch.empty(q.shape[:3], device=DEV, dtype=torch.float64)
    trees = parents.tolist()
    for i in range(case["b"]):
        for j in range(case["h"]):
            out[i, j], lse[i, j] = _tree64(q[i, j], k[i, j], v[i, j], com[i, j], trees[i], case["len"])
    return {"out": out, "lse": lse}


def _exact_accept(case, seed):
    q, k, v, com, lse, path = _accept_inputs(case, seed)
    length, count, d = case["len"], case["count"], case["d"]
    new, paths = com.double(), path.tolist()
    for i in range(case["b"]):
        at = torch.tensor(paths[i], device=DEV)
        for j in range(case["h"]):
            qd = q[i, j, at].double() * (LOG2E / math.sqrt(d))
            rows = torch.cat([k[i, j, :length], k[i, j, length + at]]).double()
            p = torch.exp2(qd @ rows.T - lse[i, j, at].double()[:, None])
            new[i, j, :length] += p[:, :length].sum(dim=0)
            new[i, j, length : length + count] = p[:, length:].tril().sum(dim=0)
        k[i, :, length : length + count] = k[i, :, length + at].clone()
        v[i, :, length : length + count] = v[i, :, length + at].clone()
    return {"k": k.double(), "v": v.double(), "committed": new}


def _exact_evict(case, seed):
    k, v, com = _evict_inputs(case, seed)
    b, h, keep, room = case["b"], case["h"], case["keep"], case["room"]
    first, stop = case["first"], case["len"] - case["recent"]
    ko = torch.zeros(b, h, keep + room, case["d"], device=DEV, dtype=torch.float64)
    vo, co = torch.zeros_like(ko), torch.zeros(b, h, keep + room, device=DEV, dtype=torch.float64)
    index = torch.empty(b, h, keep, device=DEV, dtype=torch.int32)
    for i in range(b):
        for j in range(h):
            flags = torch.ones(case["len"], device=DEV, dtype=torch.bool)
            flags[first:stop] = False
            wanted = keep - first - case["recent"]
            if wanted:
                mid = com[i, j, first:stop]
                least = mid.topk(wanted).values[-1]
                above, ties = mid > least, mid == least
                flags[first:stop] = above | (ties & (ties.cumsum(0) <= wanted - above.sum()))
            rows = flags.nonzero()[:, 0]
            index[i, j] = rows.int()
            ko[i, j, :keep], vo[i, j, :keep], co[i, j, :keep] = k[i, j, rows].double(), v[i, j, rows].double(), com[i, j, rows].double()
    return {"k": ko, "v": vo, "committed": co, "index": index}


def exact(case, seed):
    with torch.no_grad():
        return {"tree": _exact_tree, "accept": _exact_accept, "evict": _exact_evict}[case["kind"]](case, seed)
