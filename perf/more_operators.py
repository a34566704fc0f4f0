"""A dilution decode cache in 4 bits, case by case: rows quantised as they are written, read
back, and the decode step over them.

    own                  False: run() computes the plain form; True: the framework's kernels
    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call: rows, queries, caches
    run(state)           one pass through an operator, with its outputs
    work(case)           bytes and operations that one pass cannot do without
    exact(case, seed)    the outputs in float64, from the definitions

Kinds of cases (B sequences of H heads of width D):

    write   `rows` new rows of K and V go into the caches from position `start` on, and come
            back as the values that they now stand for.  "packed": the rows are views of a
            (B, T, 3 H D) projection, as an attention layer has them.
    read    `rows` cached rows from `start` on as ordinary rows of type `prec`.
    step    one query row of every sequence against `len` cached keys, the demand advanced.

The format: a row in blocks of min(32, D) elements, an element one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
with a sign (4 bits, the even element of a pair in the low half of a byte) times its block's power of
two, 2^(s - 127) with s a byte: the smallest power for which no element rounds beyond 6, but from
2^-125 to 2^125 (elements beyond 6 times that count as 6); s = 255 marks a block that held a NaN or an infinity.
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
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _kernels():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dilution-attention_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dilution import kernels

    return kernels


def _write(name, b, h, rows, start, room, d=64, prec="bf16", packed=True):
    return {"name": name, "kind": "write", "b": b, "h": h, "rows": rows, "start": start, "cap": start + rows + room, "d": d,
            "prec": prec, "packed": packed}


def _read(name, b, h, rows, start, room, d=64, prec="bf16"):
    return {"name": name, "kind": "read", "b": b, "h": h, "rows": rows, "start": start, "cap": start + rows + room, "d": d,
            "prec": prec}


def _step(name, b, h, length, room, d=64, prec="bf16"):
    return {"name": name, "kind": "step", "b": b, "h": h, "len": length, "cap": length + room, "d": d, "prec": prec}


def listed():
    return [
        # a decoded token of 8 sequences goes into a layer's cache: launches and latency count
        _write("write_token", 8, 16, 1, 1000, 24),
        # a layer's prompts of 8 sequences, from the fused projection
        _write("write_prompt", 8, 16, 16384, 0, 128),
        # odd sizes, wide heads, fp32 rows of their own
        _write("write_ragged", 3, 5, 1001, 77, 5, d=128, prec="fp32", packed=False),
        # a short cache becomes an ordinary one, for an operator that takes those
        _read("read_short", 1, 16, 1000, 0, 24),
        # long contexts read back whole
        _read("read_128k", 4, 16, 131072, 0, 0),
        # a range from the middle of a cache, the widest heads, fp16
        _read("read_ragged", 3, 7, 2001, 33, 9, d=256, prec="fp16"),
        # one sequence at a short context: launches and latency count
        _step("step_short", 1, 16, 1000, 24),
        # serving 8 sequences at a 16K context
        _step("step_16k", 8, 16, 16384, 128),
        # odd head counts, lengths and widths, fp16 activations
        _step("step_ragged", 3, 5, 5003, 30, d=128, prec="fp16"),
        # fp32 activations
        _step("step_fp32", 2, 8, 4096, 0, prec="fp32"),
        # the longest contexts: one sequence, and a full batch
        _step("step_one_128k", 1, 16, 131072, 0),
        _step("step_128k", 16, 16, 131072, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["write", "read", "step", "step", "step"])
        b, h = _log_int(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        d = rng.choice([16, 32, 64, 64, 64, 128, 128, 256])
        prec = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        c = {"kind": kind, "b": b, "h": h, "d": d, "prec": prec}
        if kind == "step":
            length = _log_int(rng, 1, 131072)
            c.update(len=length, cap=length + rng.choice([0, 1, 24, 128]))
            if b * h * length * d <= 256 * 131072 * 64:
                return c
            continue
        rows, start = _log_int(rng, 1, 65536), rng.choice([0, 0, 1, 31, 500])
        c.update(rows=rows, start=start, cap=start + rows + rng.choice([0, 1, 24, 128]))
        if kind == "write":
            c["packed"] = rng.choice([True, True, False])
        if b * h * rows * d <= 128 * 16384 * 64:
            return c


# ---------------------------------------------------------------------------
# inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _blocks(d):
    """(blocks of a row, elements of a block)."""
    return d // min(32, d), min(32, d)


def _write_inputs(case, seed):
    """New rows whose channels have scales of their own, as projections have."""
    g, dt = _gen(seed), _TYPES[case["prec"]]
    b, h, t, d = case["b"], case["h"], case["rows"], case["d"]
    scale = torch.exp(torch.randn(h * d, generator=g, device=DEV) * 0.7)
    if case["packed"]:
        qkv = torch.randn(b, t, 3 * h * d, generator=g, device=DEV, dtype=dt)
        qkv[:, :, h * d : 2 * h * d] *= scale.to(dt)
        _, k, v = (x.view(b, t, h, d).transpose(1, 2) for x in qkv.split(h * d, dim=2))
    else:
        k, v = (torch.randn(b, h, t, d, generator=g, device=DEV, dtype=dt) for _ in range(2))
        k *= scale.view(h, 1, d).to(dt)
    return k, v


def _cache_inputs(case, seed):
    """Caches of normal rows, made a sequence at a time: (codes, scales) of K and of V."""
    g = _gen(seed)
    b, h, cap, d = case["b"], case["h"], case["cap"], case["d"]
    caches = []
    for _ in range(2):
        codes = torch.empty(b, h, cap, d // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(b, h, cap, _blocks(d)[0], dtype=torch.uint8, device=DEV)
        for i in range(b):
            codes[i], scales[i] = _quantise(torch.randn(h, cap, d, generator=g, device=DEV))
        caches.append((codes, scales))
    return caches


def _step_inputs(case, seed):
    """A query, the caches, and a demand like the one that `len` - 1 rows leave: early keys hold
    more, the newest one none."""
    caches = _cache_inputs(case, seed)
    g = _gen(seed + 1)
    b, h, length, d = case["b"], case["h"], case["len"], case["d"]
    q = _randn(g, (b, 1, h * d), _TYPES[case["prec"]]).view(b, 1, h, d).transpose(1, 2)
    pos = torch.arange(length, device=DEV, dtype=torch.float32)
    com = torch.zeros(b, h, case["cap"], device=DEV)
    com[:, :, :length] = torch.log(length / (pos + 1.0)) * torch.exp(torch.randn(b, h, length, generator=g, device=DEV) * 0.5)
    return q, caches, com


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "write":
        state["k"], state["v"] = _write_inputs(case, seed)
        # earlier rows are there
        caches = _cache_inputs(case, seed + 1)
    elif case["kind"] == "read":
        caches = _cache_inputs(case, seed)
    else:
        state["q"], caches, state["committed"] = _step_inputs(case, seed)
    (state["k_codes"], state["k_scales"]), (state["v_codes"], state["v_scales"]) = caches
    return state


# ---------------------------------------------------------------------------
# the plain forms


def _quantise(x):
    """(..., D) rows as (codes (..., D / 2), scales (..., blocks)), both uint8."""
    x = x.float().unflatten(-1, _blocks(x.shape[-1]))
    top = x.abs().amax(dim=-1, keepdim=True)
    # the exponent of the largest element, one higher from 1.75 * 2^n on, two lower for the scale
    s = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)
    bad = ~torch.isfinite(top)
    y = x * ((254 - s) << 23).view(torch.float32)
    mag = y.abs()
    code = (mag > 0.25).to(torch.uint8)
    for above in (mag >= 0.75, mag > 1.25, mag >= 1.75, mag > 2.5, mag >= 3.5, mag > 5.0):
        code += above
    code += torch.signbit(y).to(torch.uint8) << 3
    code = code.masked_fill(bad, 0).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), s.masked_fill(bad, 255).squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    """The fp32 values (..., D) that codes and scales stand for."""
    grid = torch.tensor(_GRID, device=DEV)
    grid = torch.cat([grid, -grid])
    pairs = torch.stack([grid.repeat(16), grid.repeat_interleave(16)], dim=1)      # by byte
    x = pairs[codes.int()].flatten(-2)
    factor = (scales.int() << 23).view(torch.float32).masked_fill(scales == 255, float("nan"))
    return (x.unflatten(-1, (scales.shape[-1], -1)) * factor[..., None]).flatten(-2)


def _plain_write(s):
    case = s["case"]
    at = slice(case["start"], case["start"] + case["rows"])
    out = {}
    for name in ("k", "v"):
        codes, scales = _quantise(s[name])
        s[name + "_codes"][:, :, at], s[name + "_scales"][:, :, at] = codes, scales
        out[name] = _values(s[name + "_codes"][:, :, at], s[name + "_scales"][:, :, at]).to(s[name].dtype)
    return out


def _plain_read(s):
    case = s["case"]
    at = slice(case["start"], case["start"] + case["rows"])
    return {name: _values(s[name + "_codes"][:, :, at], s[name + "_scales"][:, :, at]).to(_TYPES[case["prec"]])
            for name in ("k", "v")}


def _plain_step(s):
    length, d = s["case"]["len"], s["case"]["d"]
    com = s["committed"][:, :, :length]
    k = _values(s["k_codes"][:, :, :length], s["k_scales"][:, :, :length])
    a = (s["q"].float() @ k.transpose(2, 3)).squeeze(2) * (LOG2E / math.sqrt(d))
    del k
    m = a.amax(dim=2, keepdim=True)
    e = torch.exp2(a - m)
    p = e / e.sum(dim=2, keepdim=True)
    com += p
    share = p / (com + EPS)
    w = share / (share.sum(dim=2, keepdim=True) + EPS)
    v = _values(s["v_codes"][:, :, :length], s["v_scales"][:, :, :length])
    return {"out": (w[:, :, None] @ v).to(s["q"].dtype), "committed": s["committed"]}


# ---------------------------------------------------------------------------
# one pass


def _own(s):
    ops, case = _kernels(), s["case"]
    k_cache = ops.Fp4Rows(s["k_codes"], s["k_scales"])
    v_cache = ops.Fp4Rows(s["v_codes"], s["v_scales"])
    if case["kind"] == "step":
        out = ops.dilution_decode_step_fp4(s["q"], k_cache, v_cache, s["committed"], case["len"])
        return {"out": out, "committed": s["committed"]}
    if case["kind"] == "write":
        ops.dilution_fp4_write(s["k"], s["v"], k_cache, v_cache, case["start"])
    k, v = ops.dilution_fp4_read(k_cache, v_cache, case["start"], case["rows"], dtype=_TYPES[case["prec"]])
    return {"k": k, "v": v}


def run(state):
    with torch.no_grad():
        if own:
            return _own(state)
        return {"write": _plain_write, "read": _plain_read, "step": _plain_step}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    size, d = 4 if case["prec"] == "fp32" else 2, case["d"]
    slices, held = case["b"] * case["h"], 2 * (d // 2 + _blocks(d)[0])         # bytes of a key and its value
    if case["kind"] == "step":
        return {"bytes": slices * (case["len"] * (held + 8) + 2 * d * size), "flops": 4 * slices * case["len"] * d}
    rows = slices * case["rows"]
    if case["kind"] == "write":
        return {"bytes": rows * (4 * d * size + held), "flops": 8 * rows * d}
    return {"bytes": rows * (2 * d * size + held), "flops": 2 * rows * d}


# ---------------------------------------------------------------------------
# the same in float64


def _exact_values(x):
    """The nearest values of the format, a row tensor's blocks each on its own grid."""
    x = x.double().unflatten(-1, _blocks(x.shape[-1]))
    frac, power = torch.frexp(x.abs().amax(dim=-1, keepdim=True))             # frac in [0.5, 1)
    e = (power - 3 + (frac >= 0.875)).clamp(-125, 125)
    r = torch.ldexp(x.abs(), -e)
    step = torch.where(r < 2.0, 0.5, torch.where(r < 4.0, 1.0, 2.0)).double()
    return torch.copysign(torch.ldexp(((r / step).round() * step).clamp(max=6.0), e), x).flatten(-2)


def _held_values(codes, scales):
    """What a cache stands for, by sign, exponent and mantissa bits of its codes."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()
    exponent, mantissa = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(exponent == 0, 0.5 * mantissa, torch.ldexp(1.0 + 0.5 * mantissa, exponent - 1))
    mag = torch.where(c >= 8, -mag, mag).unflatten(-1, (scales.shape[-1], -1))
    return torch.ldexp(mag, scales.int()[..., None] - 127).flatten(-2)


def _exact_step(case, seed):
    q, ((kc, ks), (vc, vs)), com = _step_inputs(case, seed)
    length, d = case["len"], case["d"]
    out, new = torch.empty(q.shape, dtype=torch.float64, device=DEV), com.double()
    for i in range(case["b"]):
        for j in range(case["h"]):
            a = _held_values(kc[i, j, :length], ks[i, j, :length]) @ q[i, j, 0].double() / math.sqrt(d)
            p = torch.softmax(a, dim=0)
            new[i, j, :length] += p
            share = p / (new[i, j, :length] + EPS)
            out[i, j, 0] = (share / (share.sum() + EPS)) @ _held_values(vc[i, j, :length], vs[i, j, :length])
    return {"out": out, "committed": new}


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "step":
            return _exact_step(case, seed)
        if case["kind"] == "write":
            k, v = _write_inputs(case, seed)
            return {"k": _exact_values(k), "v": _exact_values(v)}
        at = slice(case["start"], case["start"] + case["rows"])
        (kc, ks), (vc, vs) = _cache_inputs(case, seed)
        return {"k": _held_values(kc[:, :, at], ks[:, :, at]), "v": _held_values(vc[:, :, at], vs[:, :, at])}
