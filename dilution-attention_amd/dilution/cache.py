"""Prefill -> decode state hand-off on the HIP kernels.

The reference keeps the decode state of one attention layer in a dict
``{"k", "v", "len", "committed"}``:

* k / v: ``(B, H, capacity, D)`` buffers allocated once and filled by slice
  assignment (src/dilution/model.py:76-83, ``_alloc_cache``);
* len: the number of valid positions;
* committed: the ``(B, H, capacity)`` fp32 demand -- column totals of the
  bids over every row seen so far (model.py:224-228).

``begin_cache`` prefills a prompt (model.py:198-229) and ``step_cache`` runs
one decode token (model.py:231-241, the kernel branch), with the same dict, the
same capacity rule (``max(capacity, prompt length)``, model.py:79) and the same
error past capacity (model.py:88-89).  Unlike the reference, which prefills the
whole prompt in one forward call, ``begin_cache(..., chunk=C)`` prefills it in
chunks of C rows through ``dilution_prefill_chunk``, writing K/V and the
demand straight into the cache buffers; with ``chunk=None`` it runs the
one-call forward as the reference does.  Both give the same outputs and demand.

The ablation variants (``bid`` / ``share_cumsum`` / ``shift`` keywords, the
operators of ``kernels_bid``) prefill in one call and decode through the
variant decode step (model.py:198-241 with ``_bid_kw``).

``tree_step`` and ``accept_tree`` decode several drafted tokens at once (a tree
of them, of which one path is taken), and ``evict_cache`` shrinks a cache to the
keys that carry the demand.  The reference has no counterpart: it decodes one
token at a time and its caches only grow.  Between a tree step and the next
change of the length the dict also holds ``draft``, the number of that step.

A cache may hold its rows in 4 bits: ``k`` and ``v`` are then ``kernels.Fp4Rows``
(``begin_cache(..., bits=4)`` or ``pack_cache``; ``unpack_cache`` is the way back).
``append_kv`` and ``step_cache`` take both kinds; a tree step and an eviction need
ordinary rows.
"""

from __future__ import annotations

import itertools

import torch

from . import kernels
from . import kernels_bid


def _precision(dtype: torch.dtype) -> str:
    # model.py:203: bf16 activations use bf16 operands, anything else tf32
    return "bf16" if dtype == torch.bfloat16 else "tf32"


def alloc_cache(k: torch.Tensor, v: torch.Tensor, capacity: int | None = None) -> dict:
    """Cache buffers holding k, v (B, H, T, D) in positions [0, T) of a
    capacity of ``max(capacity, T)`` (model.py:76-83), with a zero demand."""
    batch, heads, seq, head_dim = k.shape
    capacity = max(capacity if capacity is not None else seq, seq)
    k_buf = k.new_zeros(batch, heads, capacity, head_dim)
    v_buf = v.new_zeros(batch, heads, capacity, head_dim)
    k_buf[:, :, :seq] = k
    v_buf[:, :, :seq] = v
    committed = torch.zeros(batch, heads, capacity, device=k.device, dtype=torch.float32)
    return {"k": k_buf, "v": v_buf, "len": seq, "committed": committed}


_draft_numbers = itertools.count(1)
"""A number for every tree step: a cache holds that of the last one on it, until it moves on."""


def moved_on(cache: dict, length: int) -> None:
    """Set the length after rows were written: what was drafted behind the old one is gone."""
    cache["len"] = length
    cache.pop("draft", None)


def is_packed(cache: dict) -> bool:
    """Whether the cache holds its rows in 4 bits."""
    return isinstance(cache["k"], kernels.Fp4Rows)


def _need_rows(cache: dict, what: str) -> None:
    if is_packed(cache):
        raise ValueError(f"{what} needs a cache of ordinary rows: unpack_cache() makes one of a 4-bit cache")


def pack_cache(cache: dict, capacity: int | None = None) -> dict:
    """A cache in 4 bits of ``max(capacity, length)`` positions (``capacity`` defaults to the
    given one's) with the rows of a cache of ordinary ones, quantised, and its demand.  The
    cache given is not changed."""
    _need_rows(cache, "pack_cache")
    k, v, length = cache["k"], cache["v"], cache["len"]
    batch, heads, old, head_dim = k.shape
    capacity = max(old if capacity is None else capacity, length)
    rows = [kernels.alloc_fp4_rows(batch, heads, capacity, head_dim, k.device) for _ in range(2)]
    kernels.dilution_fp4_write(k[:, :, :length], v[:, :, :length], *rows, 0)
    return {"k": rows[0], "v": rows[1], "len": length, "committed": _demand_in(cache, capacity)}


def unpack_cache(cache: dict, capacity: int | None = None, dtype: torch.dtype = torch.bfloat16) -> dict:
    """A cache of ordinary rows in ``dtype``, with ``max(capacity, length)`` positions, holding what
    a cache in 4 bits stands for, and its demand.  The cache given is not changed."""
    if not is_packed(cache):
        raise ValueError("unpack_cache needs a cache in 4 bits")
    capacity = cache["k"].shape[2] if capacity is None else capacity
    k, v = kernels.dilution_fp4_read(cache["k"], cache["v"], 0, cache["len"], dtype)
    new = alloc_cache(k, v, capacity)
    new["committed"] = _demand_in(cache, new["k"].shape[2])
    return new


def _demand_in(cache: dict, capacity: int) -> torch.Tensor:
    """The demand of the cached positions in a new buffer of `capacity`, zero behind them."""
    new = cache["committed"].new_zeros(*cache["committed"].shape[:2], capacity)
    new[:, :, : cache["len"]] = cache["committed"][:, :, : cache["len"]]
    return new


def append_kv(cache: dict, k1: torch.Tensor, v1: torch.Tensor) -> int:
    """Write one new position (k1, v1: (B, H, 1, D)) and return the new
    length (model.py:86-93)."""
    t = cache["len"]
    if t >= cache["k"].shape[2]:
        raise ValueError("decode step past the cache capacity (context_length)")
    if is_packed(cache):
        if k1.dim() != 4 or k1.shape[2] != 1:
            raise ValueError(f"one new position is appended, k1 and v1 of (B, H, 1, D), got {tuple(k1.shape)}")
        kernels.dilution_fp4_write(k1, v1, cache["k"], cache["v"], t)
    else:
        cache["k"][:, :, t] = k1[:, :, 0]
        cache["v"][:, :, t] = v1[:, :, 0]
    moved_on(cache, t + 1)
    return t + 1


def begin_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, capacity: int | None = None,
                chunk: int | None = None, dot_precision: str | None = None, bits: int | None = None, **bid_kw):
    """Prefill a prompt: returns (y, cache) with y (B, H, T, D) in q.dtype.

    chunk=None runs the one-call forward and copies ``committed_total`` into
    the cache (model.py:202-228); chunk=C prefills C rows at a time with the
    demand carried in the cache's buffer.  ``bid_kw`` (bid, share_cumsum,
    shift) selects an ablation variant, always prefilled in one call.  bits=4
    gives a cache in 4 bits (``pack_cache``): the prompt's own rows are computed from
    its unrounded keys and values, the steps behind it from the quantised ones; production
    operator only.
    """
    if bits is not None:
        if bits != 4:
            raise ValueError(f"bits must be None or 4, got {bits}")
        if bid_kw:
            raise ValueError("a cache in 4 bits needs the production operator")
        y, cache = begin_cache(q, k, v, chunk=chunk, dot_precision=dot_precision)
        return y, pack_cache(cache, capacity)
    prec = dot_precision or _precision(q.dtype)
    seq = q.shape[2]
    cache = alloc_cache(k, v, capacity)
    if bid_kw:
        y, aux = kernels_bid.dilution_attention_forward(q, k, v, dot_precision=prec, return_aux=True,
                                                        **bid_kw)
        cache["committed"][:, :, :seq] = aux["committed_total"]
        return y.to(q.dtype), cache
    if chunk is None:
        y, aux = kernels.dilution_attention_forward(q, k, v, dot_precision=prec, return_aux=True)
        cache["committed"][:, :, :seq] = aux["committed_total"]
        return y.to(q.dtype), cache
    if chunk < 1:
        raise ValueError("chunk must be positive")
    # every chunk writes its rows of y, in q's type where the kernels write it
    # (fp64 queries get the fp32 outputs, converted)
    y = torch.empty(q.shape, device=q.device, dtype=q.dtype if q.dtype in kernels._DTYPES else torch.float32)
    for start in range(0, seq, chunk):
        stop = min(start + chunk, seq)
        kernels.dilution_prefill_chunk(q[:, :, start:stop], cache["k"], cache["v"], cache["committed"], start,
                                       dot_precision=prec, _out=y[:, :, start:stop])
    return y.to(q.dtype), cache


def step_cache(q1: torch.Tensor, k1: torch.Tensor, v1: torch.Tensor, cache: dict, **bid_kw) -> torch.Tensor:
    """One decode token: append (k1, v1) and return the new row's output
    (B, H, 1, D) in q1.dtype, advancing the cache's demand in place
    (model.py:231-241); ``bid_kw`` as in ``begin_cache``."""
    if is_packed(cache):
        if bid_kw:
            raise ValueError("a cache in 4 bits needs the production operator")
        t = cache["len"]
        if t >= cache["k"].shape[2]:
            raise ValueError("decode step past the cache capacity (context_length)")
        y = kernels.dilution_decode_step_fp4(q1, cache["k"], cache["v"], cache["committed"], t + 1, k1, v1)
        moved_on(cache, t + 1)
        return y
    t = append_kv(cache, k1, v1)
    if bid_kw:
        return kernels_bid.dilution_decode_step(q1, cache["k"], cache["v"], cache["committed"], t, **bid_kw)
    return kernels.dilution_decode_step(q1, cache["k"], cache["v"], cache["committed"], t)


def tree_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, parents):
    """Attention for N drafted tokens (q, k, v: (B, H, N, D)) that hang in a tree
    below the cached context (``parents`` as in ``kernels.dilution_tree_step``).
    Writes their k and v behind the cached positions and returns (y, draft): y
    (B, H, N, D) in q.dtype, draft what ``accept_tree`` needs.  The cache's
    length and demand stay.  A later step overwrites rows that were not accepted:
    of several tree steps the last one's draft can be, until the cache moves on."""
    # all that the kernels would refuse, before any row is written
    _need_rows(cache, "a tree step")
    if q.dim() != 4 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k and v must have one shape (B, H, N, D), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    batch, heads, capacity, head_dim = cache["k"].shape
    nodes = q.shape[2]
    if (*q.shape[:2], q.shape[3]) != (batch, heads, head_dim):
        raise ValueError(f"drafted rows {tuple(q.shape)} do not match the cache {tuple(cache['k'].shape)}")
    if not 1 <= nodes <= kernels.MAX_TREE_NODES:
        raise ValueError(f"a tree holds 1 to {kernels.MAX_TREE_NODES} drafted nodes, got {nodes}")
    if q.dtype != cache["k"].dtype or q.device != cache["k"].device:
        raise ValueError("q must have the caches' dtype and device")
    t, stop = cache["len"], cache["len"] + nodes
    if stop > capacity:
        raise ValueError("drafted tokens past the cache capacity (context_length)")
    parents = kernels._parents_on(q.device, parents)
    if parents.shape not in ((nodes,), (batch, nodes)):
        raise ValueError(f"parents {tuple(parents.shape)} do not match the drafted rows {tuple(q.shape)}")
    cache["draft"] = number = next(_draft_numbers)
    cache["k"][:, :, t:stop] = k
    cache["v"][:, :, t:stop] = v
    y, aux = kernels.dilution_tree_step(q, cache["k"], cache["v"], cache["committed"], t, parents, return_aux=True)
    return y, {"q": q, "lse": aux["lse"], "len": t, "number": number}


def check_draft(cache: dict, draft: dict) -> None:
    """ValueError unless ``draft`` is what the last ``tree_step`` on this cache returned, and the
    cache is where it was."""
    if draft["len"] != cache["len"] or "draft" not in cache or draft.get("number") != cache["draft"]:
        raise ValueError("the cache has moved on since this tree step")


def accept_tree(cache: dict, draft: dict, path) -> int:
    """Take a path of the tree of the last ``tree_step`` on this cache into it
    (``path`` as in ``kernels.dilution_tree_accept``); returns the new length."""
    check_draft(cache, draft)
    length = kernels.dilution_tree_accept(draft["q"], cache["k"], cache["v"], cache["committed"], cache["len"],
                                          draft["lse"], path)
    if length != cache["len"]:
        moved_on(cache, length)
    return length


def evict_cache(cache: dict, keep: int, first: int = 0, recent: int = 0, capacity: int | None = None) -> dict:
    """A cache of the ``keep`` positions that carry the demand (the first
    ``first`` and the last ``recent`` stay whatever they carry: the newest keys
    have had the fewest rows to gather demand from), in new buffers of
    ``max(capacity, keep)`` positions.  The keys hold no position, so decoding
    goes on over the kept ones.  A cache of at most ``keep`` positions is returned as it is."""
    _need_rows(cache, "an eviction")
    if cache["len"] <= keep:
        return cache
    k, v, committed, _ = kernels.dilution_evict(cache["k"], cache["v"], cache["committed"], cache["len"], keep,
                                                first=first, recent=recent, capacity=capacity)
    return {"k": k, "v": v, "len": keep, "committed": committed}
