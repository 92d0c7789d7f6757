"""Operators over a key/value cache that is held in eight bits, as cases that can be timed and checked one by one.

A cache entry holds a row - one token's keys (or values) of one head, D numbers - as D codes and one exponent e: the row
stands for code * 2^e.  "e4m3": codes are e4m3 numbers, e the smallest with max|x| <= 448 * 2^e; "int8": codes are whole
numbers, e the smallest with max|x| <= 127 * 2^e.  e stays within -50..50 (codes saturate), is 0 for a row of zeros and is
stored as the byte e + 127; a row with an infinity or NaN is stored as byte 255 and reads back as NaN.

Kinds of case:
  write   a step's projections are given their bias, their norms per head and their rotation, keys and values are appended to the pages,
          and what the step's requests then have cached is read back in the compute type, 64 keys a block
  attend  causal attention of a step's queries over the pages: single tokens (decoding), portions of prompts, or both
Codes are returned as the values they stand for.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64                     # keys of a block of read-back rows
THETA = 1000000.0
EPS = 1e-6
TOP = {"e4m3": 448.0, "int8": 127.0}
# (query heads, key/value heads, head size): the layers of the repository's configurations and benchmark
HEADS = {"0.5B": (14, 2, 64), "3B": (16, 2, 128), "7B": (28, 4, 128), "wide": (32, 8, 128)}


def _case(name, kind, heads, store, requests, cached, rows, page=16, **more):
    """`requests` requests share `rows` new tokens unevenly (`singles` of them bring one each) and have up to `cached` tokens behind them."""
    case = dict(kind=kind, heads=heads, store=store, requests=requests, cached=cached, rows=rows, page=page, singles=0, window=0, keep=0,
                sink=False, norm=False, rot=HEADS[heads][2], ragged=True)
    case.update(more)
    return dict(case, name=name) if name else case


def listed():
    return [
        # The first decoded token behind a short prompt: latency alone.
        _case("write_one", "write", "0.5B", "e4m3", 1, 11, 1),
        # A whole prompt, as chunked prefill brings it.
        _case("write_prompt", "write", "7B", "e4m3", 1, 0, 2048, ragged=False),
        # Several prompts of odd lengths in one step, queries and keys normalised per head, half of every head rotated.
        _case("write_norms", "write", "wide", "int8", 5, 700, 1511, page=32, norm=True, rot=64),
        # Decoding: one request behind a short context.
        _case("decode_one_short", "attend", "0.5B", "e4m3", 1, 517, 1),
        # The engine's headline: eight requests behind 4,096 tokens.
        _case("decode_eight", "attend", "0.5B", "e4m3", 8, 4096, 8, ragged=False),
        # A full batch of uneven lengths, which is what a cache of half the size makes room for.
        _case("decode_batch", "attend", "7B", "e4m3", 64, 8192, 64),
        # One request behind a long document.
        _case("decode_long", "attend", "7B", "int8", 1, 131072, 1, page=64, ragged=False),
        # Window attention with a learned sink and kept first tokens.
        _case("decode_window", "attend", "3B", "int8", 48, 6000, 48, window=1024, keep=4, sink=True),
        # A short question behind a cached document.
        _case("portion_short", "attend", "0.5B", "int8", 1, 5000, 37, ragged=False),
        # A portion behind a long history.
        _case("portion_history", "attend", "7B", "e4m3", 1, 8192, 509, page=32, ragged=False),
        # The largest portion of a long prompt.
        _case("portion_long", "attend", "3B", "int8", 1, 16384, 2048, ragged=False),
        # Continuous batching: decoded tokens beside portions of prompts.
        _case("mixed_step", "attend", "3B", "e4m3", 24, 3000, 421, singles=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice(sorted(HEADS))
    store = rng.choice(["e4m3", "int8"])
    page = rng.choice([8, 16, 16, 32, 64])
    kind = rng.choice(["write", "decode", "decode", "portion", "mixed"])
    window = rng.choice([0, 0, 0, _log(rng, 40, 4000)])
    seen = dict(window=window, keep=rng.choice([0, rng.randint(1, 9)]) if window else 0, sink=rng.random() < 0.25)
    if kind == "write":
        requests = _log(rng, 1, 16)
        rot = HEADS[heads][2] // rng.choice([1, 1, 2])
        return _case(None, "write", heads, store, requests, rng.choice([0, _log(rng, 1, 2000)]), max(requests, _log(rng, 1, 4096)), page,
                     norm=rng.random() < 0.5, rot=rot)
    if kind == "decode":
        _, kv_heads, dim = HEADS[heads]
        cached = _log(rng, 1, 131072)
        requests = _log(rng, 1, max(1, min(128, int(2.8e8 / (cached * 2 * kv_heads * (dim + 1))))))
        return _case(None, "attend", heads, store, requests, cached, requests, page, **seen)
    if kind == "portion":
        requests = _log(rng, 1, 4)
        rows = max(2 * requests, _log(rng, 2, 2048))
        return _case(None, "attend", heads, store, requests, rng.choice([0, _log(rng, 1, 8192)]), rows, page, **seen)
    singles, others = _log(rng, 1, 32), _log(rng, 1, 3)
    return _case(None, "attend", heads, store, singles + others, _log(rng, 1, 4000), singles + max(2 * others, _log(rng, 2, 700)), page,
                 singles=singles, **seen)


def _lengths(case):
    """(tokens cached before the step, tokens the step brings) of every request; sizes alone decide, so that a case always does the same work."""
    g = torch.Generator().manual_seed(case["requests"] * 7919 + case["rows"] * 31 + case["cached"])
    n, singles = case["requests"], case["singles"]
    spread = torch.rand(n, generator=g).tolist()
    starts = [int(case["cached"] * (0.2 + 0.8 * spread[i])) if case["ragged"] and i else case["cached"] for i in range(n)]
    counts = [1] * n
    if case["rows"] > n:
        least = 1 if case["kind"] == "write" else 2
        others = n - singles
        left = case["rows"] - singles - least * others
        shares = [0.1 + x for x in torch.rand(others, generator=g).tolist()]
        extra = [int(left * s / sum(shares)) for s in shares]
        extra[0] += left - sum(extra)
        counts = [1] * singles + [least + x for x in extra]
    return starts, counts


def _first_seen(start, case):
    return max(0, start - case["window"] + 1) if case["window"] else 0


def _blocks(case):
    """(request, block of 64 keys) of every block that a read-back brings, in order."""
    starts, counts = _lengths(case)
    return [(i, b) for i, (s, c) in enumerate(zip(starts, counts)) for b in range((s + c + BLOCK - 1) // BLOCK)]


def work(case):
    Hq, Hkv, D = HEADS[case["heads"]]
    starts, counts = _lengths(case)
    T = sum(counts)
    rows = 2 * Hkv * (D + 1)                                 # a token's codes and scales
    if case["kind"] == "write":
        tokens = sum(s + c for s, c in zip(starts, counts))
        return {"bytes": T * (Hq + 2 * Hkv) * D * 2 + T * Hq * D * 2 + T * case["rot"] * 4 + T * rows + tokens * rows + len(_blocks(case)) * BLOCK * Hkv * D * 4,
                "flops": 8 * T * (Hq + 2 * Hkv) * D}
    bytes_, flops = T * Hq * D * 4, 0
    for s, c in zip(starts, counts):
        lo = _first_seen(s, case)
        bytes_ += (s + c - lo + min(case["keep"], lo)) * rows
        if case["window"]:
            pairs = sum(p + 1 - _first_seen(p, case) + min(case["keep"], _first_seen(p, case)) for p in range(s, s + c))
        else:
            pairs = c * s + c * (c + 1) // 2
        flops += 4 * pairs * Hq * D
    return {"bytes": bytes_, "flops": flops}


# ---- rows in eight bits ------------------------------------------------------------------------------------------------------
def _quantise(x, store):
    """(codes, scale bytes) of float32 rows."""
    amax = x.abs().amax(-1)
    frac, exp = torch.frexp(amax)                            # amax = frac * 2^exp, frac in [0.5, 1)
    e = exp - (9 if store == "e4m3" else 7) + (frac > (0.875 if store == "e4m3" else 0.9921875))
    e = torch.where(amax > 0, e.clamp(-50, 50), torch.zeros_like(e))
    fine = torch.isfinite(amax)
    e = torch.where(fine, e, torch.zeros_like(e))
    y = torch.where(fine[..., None], x, torch.zeros_like(x)) * torch.exp2(-e.float())[..., None]
    y = y.clamp(-TOP[store], TOP[store])
    codes = y.to(torch.float8_e4m3fn) if store == "e4m3" else y.round().to(torch.int8)
    return codes, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _values(codes, scales):
    factor = torch.where(scales == 255, torch.full_like(scales, float("nan"), dtype=torch.float32), torch.exp2(scales.float() - 127.0))
    return codes.float() * factor[..., None]


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    Hq, Hkv, D = HEADS[case["heads"]]
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    starts, counts = _lengths(case)
    n, T, page, store = len(starts), sum(counts), case["page"], case["store"]
    per = [(s + c + page - 1) // page for s, c in zip(starts, counts)]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=gc).to(torch.int32)
    table = torch.full((n, max(per)), -1, dtype=torch.int32)
    used = 0
    for i, p in enumerate(per):
        table[i, :p] = order[used:used + p]
        used += p
    randn = lambda *shape, scale=1.0: torch.randn(*shape, generator=g, device=dev) * scale
    # Channels of keys differ in size as a model's do; a few tokens are much larger than the others.
    channel = torch.exp(0.7 * randn(D))
    loud = lambda *shape: torch.where(torch.rand(*shape, generator=g, device=dev) < 0.02, 6.0, 1.0)
    shape = (pages, Hkv, page)
    kc, ks = _quantise(randn(*shape, D) * channel * loud(*shape)[..., None], store)
    vc, vs = _quantise(randn(*shape, D) * torch.exp(0.5 * randn(*shape))[..., None], store)
    row_segment = torch.repeat_interleave(torch.arange(n), torch.tensor(counts))
    q_start = torch.cumsum(torch.tensor([0] + counts), 0)[:-1]
    positions = torch.arange(T) - q_start[row_segment] + torch.tensor(starts)[row_segment]
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).to(dev)
    state = dict(case=case, starts=starts, counts=counts, scale=D ** -0.5, table=table.to(dev), k_pages=kc, v_pages=vc, k_scales=ks, v_scales=vs,
                 positions=i32(positions), row_segment=i32(row_segment), seg_q_start=i32(q_start), seg_q_len=i32(counts),
                 seg_kv_len=i32([s + c for s, c in zip(starts, counts)]), blocks=torch.tensor(_blocks(case), dtype=torch.int64).reshape(-1, 2).to(dev))
    if case["kind"] == "write":
        state["qkv"] = randn(T, (Hq + 2 * Hkv) * D).to(torch.bfloat16)
        state["bias"] = randn((Hq + 2 * Hkv) * D, scale=0.5)
        angle = torch.arange(max(s + c for s, c in zip(starts, counts)), dtype=torch.float64)[:, None] \
            * THETA ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        state["cos"], state["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        state["q_norm"], state["k_norm"] = ((1 + randn(D, scale=0.2)), (1 + randn(D, scale=0.2))) if case["norm"] else (None, None)
        state["q"] = torch.empty(T, Hq * D, dtype=torch.bfloat16, device=dev)
    else:
        # Queries that lean towards some key of theirs, as trained heads do: scores spread over several units.
        state["q"] = (randn(T, Hq * D) / channel.repeat(Hq) * 1.5).to(torch.bfloat16)
        state["sink"] = randn(Hq, scale=2.0) if case["sink"] else None
        state["out"] = torch.empty(T, Hq * D, dtype=torch.bfloat16, device=dev)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------------
_kernels = None


def _handles(state):
    """The kernel set, and what a step function makes once a step for all layers: the step's batch with its work lists, the view of
    the cache entry, and the workspace."""
    global _kernels
    if "handles" not in state:
        from kvcache_b200.engine.workspace import Workspace
        from kvcache_b200.kernels.api import CudaKernels
        from kvcache_b200.parts.base import PagedKVSpec, PagedKVView, StepBatch, StepPlan
        if _kernels is None:
            _kernels = CudaKernels("cuda:0")
        case = state["case"]
        Hq, Hkv, D = HEADS[case["heads"]]
        spec = PagedKVSpec(Hkv, D, case["window"] or None, None, case["keep"], store=case["store"])
        kv = PagedKVView(spec, state["k_pages"], state["v_pages"], state["table"], case["page"], True, state["k_scales"], state["v_scales"])
        plans = {}

        def plan(planner):
            arrays, numbers = planner.plan(state["starts"], state["counts"])
            plans[planner.name] = StepPlan({key: torch.as_tensor(a).to("cuda:0") for key, a in arrays.items()}, numbers)

        plan(_kernels.paged_attention_planner())
        plan(_kernels.cache_expand_planner(spec.reach, spec.keep_first))
        T, n = sum(state["counts"]), len(state["counts"])
        none = state["positions"][:0]
        batch = StepBatch(T, n, 0, none, state["positions"], state["row_segment"], state["seg_q_start"], state["seg_q_len"], state["seg_kv_len"],
                          none, none, plans=plans, max_q_len=max(state["counts"]),
                          max_kv_len=max(s + c for s, c in zip(state["starts"], state["counts"])))
        state["handles"] = (_kernels, batch, kv, Workspace("cuda:0"))
    return state["handles"]


def run(state):
    case = state["case"]
    Hq, Hkv, D = HEADS[case["heads"]]
    if own:
        kernels, batch, kv, workspace = _handles(state)
        if case["kind"] == "write":
            kernels.qkv_rope_append(state["qkv"], state["bias"], state["cos"], state["sin"], batch, kv, state["q"], Hq,
                                    q_norm=state["q_norm"], k_norm=state["k_norm"], norm_eps=EPS if case["norm"] else 0.0)
            view = kernels.expand_cache(batch, kv, torch.bfloat16, workspace)
            return {"q": state["q"], "k": view.k_pages, "v": view.v_pages}
        kernels.paged_attention(state["q"], batch, kv, state["out"], Hq, state["scale"], workspace, sink=state["sink"])
        return state["out"]
    return _plain_write(state, Hq, Hkv, D) if case["kind"] == "write" else _plain_attend(state, Hq, Hkv, D)


def _plain_write(state, Hq, Hkv, D):
    case, store, page = state["case"], state["case"]["store"], state["case"]["page"]
    T = state["qkv"].shape[0]
    x = (state["qkv"].float() + state["bias"]).view(T, Hq + 2 * Hkv, D)
    turned, v = x[:, :Hq + Hkv], x[:, Hq + Hkv:]
    if case["norm"]:
        weight = torch.cat([state["q_norm"].expand(Hq, D), state["k_norm"].expand(Hkv, D)])
        turned = turned * torch.rsqrt(turned.square().mean(-1, keepdim=True) + EPS) * weight
    half = case["rot"] // 2
    at = state["positions"].long()
    cos, sin = state["cos"][at][:, None], state["sin"][at][:, None]
    a, b, rest = turned[..., :half], turned[..., half:2 * half], turned[..., 2 * half:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
    phys, slot = state["table"].long()[state["row_segment"].long(), at // page], at % page

    def store_rows(rows, codes, scales):
        c, s = _quantise(rows, store)
        codes.view(torch.uint8)[phys, :, slot] = c.view(torch.uint8)
        scales[phys, :, slot] = s

    store_rows(turned[:, Hq:], state["k_pages"], state["k_scales"])
    store_rows(v, state["v_pages"], state["v_scales"])
    seg, first = state["blocks"][:, 0], state["blocks"][:, 1] * BLOCK
    key = first[:, None] + torch.arange(BLOCK, device=first.device)
    there = key < state["seg_kv_len"].long()[seg][:, None]
    key = torch.where(there, key, torch.zeros_like(key))
    from_page, from_slot = state["table"].long()[seg[:, None], key // page], key % page

    def read_rows(codes, scales):
        values = _values(codes.view(torch.uint8)[from_page, :, from_slot].view(codes.dtype), scales[from_page, :, from_slot])
        return torch.where(there[..., None, None], values, 0.0).transpose(1, 2).to(torch.bfloat16)

    state["q"].copy_(turned[:, :Hq].reshape(T, Hq * D))
    return {"q": state["q"], "k": read_rows(state["k_pages"], state["k_scales"]), "v": read_rows(state["v_pages"], state["v_scales"])}


def _plain_attend(state, Hq, Hkv, D):
    """All requests at once, padded to the most new tokens and to the longest context."""
    case, page = state["case"], state["case"]["page"]
    n, most, G = len(state["counts"]), max(state["counts"]), Hq // Hkv
    longest = max(s + c for s, c in zip(state["starts"], state["counts"]))
    table = state["table"].long().clamp(min=0)
    rows = lambda codes, scales: _values(codes.view(torch.uint8)[table].view(codes.dtype), scales[table]).transpose(1, 2).reshape(n, Hkv, -1, D)[:, :, :longest]
    k, v = rows(state["k_pages"], state["k_scales"]), rows(state["v_pages"], state["v_scales"])
    seg, at = state["row_segment"].long(), state["positions"].long()
    place = at - (state["seg_kv_len"] - state["seg_q_len"]).long()[seg]
    q = torch.zeros(n, most, Hq * D, device=k.device)
    q[seg, place] = state["q"].float()
    pos = torch.full((n, most), 0, dtype=torch.long, device=k.device)
    pos[seg, place] = at
    q = q.view(n, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, G * most, D)
    s = ((q @ k.transpose(-1, -2)) * state["scale"]).view(n, Hkv, G, most, longest)
    j = torch.arange(longest, device=k.device)
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= (j > pos[..., None] - case["window"]) | (j < case["keep"])
    s = torch.where(seen[:, None, None], s, torch.tensor(float("-inf"), device=k.device))
    if state["sink"] is not None:
        s = torch.cat([s, state["sink"].view(1, Hkv, G, 1, 1).expand(n, Hkv, G, most, 1)], dim=-1)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True))[..., :longest]
    o = (p.reshape(n, Hkv, G * most, longest) @ v).view(n, Hkv, G, most, D).permute(0, 3, 1, 2, 4).reshape(n, most, Hq * D)
    state["out"].copy_(o[seg, place])
    return state["out"]


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------
def _exact_rows(x, store):
    """What rows x (float64) stand for once stored: the rounding written out."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / TOP[store]))
    e = torch.where(amax > TOP[store] * 2.0 ** e, e + 1, e)
    e = torch.where(amax <= TOP[store] * 2.0 ** (e - 1), e - 1, e)
    e = torch.where(amax > 0, e.clamp(-50, 50), torch.zeros_like(e))
    y = (x / 2.0 ** e).clamp(-TOP[store], TOP[store])
    if store == "int8":
        return y.round() * 2.0 ** e
    binade = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = 2.0 ** (binade - 3)
    return (y / step).round() * step * 2.0 ** e


def _exact_cache(codes, scales, table, page, length):
    """[length, Hkv, D] float64: one request's rows."""
    at = torch.arange(length, device=codes.device)
    phys = table[at // page].long()
    c = codes.view(torch.uint8)[phys, :, at % page].view(codes.dtype).double()
    return c * 2.0 ** (scales[phys, :, at % page].double()[..., None] - 127)


def exact(case, seed):
    Hq, Hkv, D = HEADS[case["heads"]]
    s = prepare(case, seed)
    G, T = Hq // Hkv, sum(s["counts"])
    if case["kind"] == "write":
        x = (s["qkv"].double() + s["bias"].double()).view(T, -1, D)
        heads = []
        for h in range(Hq + Hkv):
            y = x[:, h]
            if case["norm"]:
                y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * (s["q_norm"] if h < Hq else s["k_norm"]).double()
            half, at = case["rot"] // 2, s["positions"].long()
            c, sn = s["cos"].double()[at], s["sin"].double()[at]
            y = torch.cat([y[:, :half] * c - y[:, half:2 * half] * sn, y[:, half:2 * half] * c + y[:, :half] * sn, y[:, 2 * half:]], -1)
            heads.append(y)
        q = torch.cat(heads[:Hq], -1)
        new = {"k": _exact_rows(torch.stack(heads[Hq:], 1), case["store"]), "v": _exact_rows(x[:, Hq + Hkv:], case["store"])}
        out = {"q": q}
        for name in ("k", "v"):
            parts, row = [], 0
            for i, (start, count) in enumerate(zip(s["starts"], s["counts"])):
                rows = torch.zeros((start + count + BLOCK - 1) // BLOCK * BLOCK, Hkv, D, dtype=torch.float64, device=q.device)
                rows[:start] = _exact_cache(s[name + "_pages"], s[name + "_scales"], s["table"][i], case["page"], start)
                rows[start:start + count] = new[name][row:row + count]
                parts.append(rows.view(-1, BLOCK, Hkv, D).transpose(1, 2))
                row += count
            out[name] = torch.cat(parts)
        return out
    if work(case)["flops"] > 1.5e12:
        return None
    out, row = torch.empty(T, Hq, D, dtype=torch.float64, device=s["q"].device), 0
    for i, (start, count) in enumerate(zip(s["starts"], s["counts"])):
        length = start + count
        k = _exact_cache(s["k_pages"], s["k_scales"], s["table"][i], case["page"], length)
        v = _exact_cache(s["v_pages"], s["v_scales"], s["table"][i], case["page"], length)
        pos = torch.arange(start, length, device=k.device)[:, None]
        j = torch.arange(length, device=k.device)[None]
        hidden = j > pos
        if case["window"]:
            hidden = hidden | ((j <= pos - case["window"]) & (j >= case["keep"]))
        for h in range(Hq):
            y = s["q"][row:row + count].double().view(count, Hq, D)[:, h] @ k[:, h // G].T * s["scale"]
            y = y.masked_fill(hidden, float("-inf"))
            top = y.amax(-1, keepdim=True)
            if s["sink"] is not None:
                top = top.clamp(min=float(s["sink"][h]))
            p = (y - top).exp()
            total = p.sum(-1, keepdim=True)
            if s["sink"] is not None:
                total = total + (s["sink"][h].double() - top).exp()
            out[row:row + count, h] = p @ v[:, h // G] / total
        row += count
    return out.view(T, Hq * D)
