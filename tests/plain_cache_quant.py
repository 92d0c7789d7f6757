"""Cache entries in eight bits, stated plainly in float64: the rounding of a row, paged pools made of such rows, append and attention."""
import dataclasses

import torch

from kvcache_b200.parts.base import STORE_DTYPES, PagedKVSpec, PagedKVView, StepBatch, StepPlan

TOP = {"e4m3": 448.0, "int8": 127.0}
STORES = ("e4m3", "int8")


def quantise(x, store):
    """(what the codes stand for before the scale, scale bytes) of float64 rows [..., D]."""
    amax = x.abs().amax(-1)
    fine = torch.isfinite(amax)
    x = torch.where(fine[..., None], x, torch.zeros_like(x))
    amax = torch.where(fine, amax, torch.ones_like(amax))
    e = torch.full_like(amax, -50.0)
    for exponent in range(-50, 50):                          # the smallest e with amax <= TOP 2^e
        e = torch.where(amax > TOP[store] * 2.0 ** exponent, torch.full_like(e, exponent + 1), e)
    e = torch.where((amax == 0) | ~fine, torch.zeros_like(e), e)
    y = (x / 2.0 ** e[..., None]).clamp(-TOP[store], TOP[store])
    return round_code(y, store), torch.where(fine, e + 127, torch.full_like(e, 255.0)).to(torch.uint8)


def step_at(y, store):
    """The distance of neighbouring codes around y."""
    if store == "int8":
        return torch.ones_like(y)
    return 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


def round_code(y, store):
    step = step_at(y, store)
    return (y / step).round() * step


def to_pool(codes, store):
    return codes.float().to(STORE_DTYPES[store])             # exact: the numbers are codes already


def values(codes, scales):
    """float64 numbers that codes and scale bytes stand for."""
    factor = torch.where(scales == 255, torch.tensor(float("nan"), dtype=torch.float64), 2.0 ** (scales.double() - 127))
    return codes.to(torch.float32).double() * factor[..., None]


def make_step(segments, Hkv, D, page, store, seed=0, window=None, keep=0, chunk=None, planners=(), spread=0.7, spare=2, writes=True):
    """A step of `segments` (cached, new) over a pool with pages in random order; every slot of the pool holds some row."""
    g = torch.Generator().manual_seed(seed)
    n = len(segments)
    per = [-(-(s + c) // page) for s, c in segments]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((n, max(per) + 1), -1, dtype=torch.int32)
    used = 0
    for i, p in enumerate(per):
        table[i, :p] = order[used:used + p]
        used += p
    def pool(strength):
        rows = torch.randn(pages, Hkv, page, D, generator=g, dtype=torch.float64) * torch.exp(spread * torch.randn(pages, Hkv, page, 1, generator=g, dtype=torch.float64))
        codes, scales = quantise(rows * strength, store)
        return to_pool(codes, store), scales
    k, ks = pool(1.0)
    v, vs = pool(1.0)
    counts = torch.tensor([c for _, c in segments])
    starts = torch.tensor([s for s, _ in segments])
    seg = torch.repeat_interleave(torch.arange(n), counts)
    q_start = torch.cumsum(counts, 0) - counts
    pos = torch.arange(int(counts.sum())) - q_start[seg] + starts[seg]
    i32 = lambda t: t.to(torch.int32)
    plans = {}
    for planner in planners:
        arrays, numbers = planner.plan(starts.numpy(), counts.numpy())
        plans[planner.name] = StepPlan({name: torch.tensor(a) for name, a in arrays.items()}, numbers)
    empty = torch.zeros(0, dtype=torch.int32)
    batch = StepBatch(len(pos), n, 0, i32(torch.arange(len(pos))), i32(pos), i32(seg), i32(q_start), i32(counts), i32(starts + counts), i32(torch.arange(n)),
                      empty, plans=plans, max_q_len=int(counts.max()), max_kv_len=int((starts + counts).max()))
    spec = PagedKVSpec(Hkv, D, window, None, keep, chunk, store=store)
    return batch, PagedKVView(spec, k, v, table, page, writes, ks, vs)


def kv_to(kv, device):
    move = lambda t: None if t is None else t.to(device).clone()
    return dataclasses.replace(kv, k_pages=move(kv.k_pages), v_pages=move(kv.v_pages), block_table=move(kv.block_table), k_scales=move(kv.k_scales),
                               v_scales=move(kv.v_scales))


def rows_of(kv, seg, length):
    """(keys, values) [length, Hkv, D] float64 of a segment."""
    j = torch.arange(length)
    page = kv.block_table[seg, j // kv.page_size].long().clamp(min=0)
    def take(codes, scales):
        c = codes.view(torch.uint8)[page, :, j % kv.page_size].contiguous().view(codes.dtype)
        return values(c, scales[page, :, j % kv.page_size])
    return take(kv.k_pages, kv.k_scales), take(kv.v_pages, kv.v_scales)


def attention(q, batch, kv, Hq, scale, sink=None, score_cap=None, slopes=None, reach=None):
    """(results, sum of |weight value|, largest |scale q| . |k| of a row) [T, Hq, D] and [T, Hq], float64."""
    Hkv, D, G = kv.spec.num_kv_heads, kv.spec.head_dim, Hq // kv.spec.num_kv_heads
    reach = kv.spec.reach if reach is None else reach
    T = batch.num_tokens
    q = q.double().view(T, Hq, D)
    out, size = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    strength = torch.zeros(T, Hq, dtype=torch.float64)
    for i in range(batch.num_segments):
        row, count, length = int(batch.seg_q_start[i]), int(batch.seg_q_len[i]), int(batch.seg_kv_len[i])
        if count == 0:
            continue
        k, v = rows_of(kv, i, length)
        pos, j = torch.arange(length - count, length)[:, None], torch.arange(length)[None]
        seen = j <= pos
        if reach > 0:
            seen &= (j > pos - reach) | (j < kv.spec.keep_first)
        if reach < 0:
            seen &= j >= pos - pos % -reach
        for h in range(Hq):
            kh, vh, qh = k[:, h // G], v[:, h // G], q[row:row + count, h]
            s = qh @ kh.T * scale
            strength[row:row + count, h] = torch.where(seen, qh.abs() @ kh.abs().T * abs(scale), 0.0).amax(-1)
            if score_cap:
                s = score_cap * torch.tanh(s / score_cap)
            if slopes is not None:
                s = s - slopes[h].double() * (pos - j)
            s = torch.where(seen, s, torch.tensor(float("-inf"), dtype=torch.float64))
            if sink is not None:
                s = torch.cat([s, sink[h].double().expand(count, 1)], 1)
            p = torch.softmax(s, -1)[:, :length]
            out[row:row + count, h], size[row:row + count, h] = _weigh(p, vh, seen), _weigh(p, vh.abs(), seen)
    return out, size, strength


def _weigh(p, v, seen):
    """p @ v where a value that a row does not see adds nothing, whatever it is."""
    if torch.isfinite(v).all():
        return p @ v
    return torch.stack([p[r, seen[r]] @ v[seen[r]] for r in range(p.shape[0])])


# ---- a stand-in kernel set and a whole model over such entries ----------------------------------------------------------------
from torch_kernels import TorchKernels  # noqa: E402


class QuantKernels(TorchKernels):
    """The plain kernel set of the engine's host tests, with cache entries in eight bits."""

    def qkv_rope_append(self, qkv, bias, cos, sin, batch, kv, q_out, num_heads, **more):
        if kv.spec.store is None:
            return super().qkv_rope_append(qkv, bias, cos, sin, batch, kv, q_out, num_heads, **more)
        wide = lambda pages: torch.zeros(pages.shape, dtype=torch.float64, device=pages.device)
        plain = dataclasses.replace(kv, spec=dataclasses.replace(kv.spec, store=None), k_pages=wide(kv.k_pages), v_pages=wide(kv.v_pages))
        super().qkv_rope_append(qkv, bias, cos, sin, batch, plain, q_out, num_heads, **more)
        if not kv.writes:
            return
        pos = batch.positions.long()
        page, slot = kv.block_table[batch.row_segment.long(), pos // kv.page_size].long(), pos % kv.page_size
        for rows, codes, scales in ((plain.k_pages, kv.k_pages, kv.k_scales), (plain.v_pages, kv.v_pages, kv.v_scales)):
            c, s = quantise(rows[page, :, slot], kv.spec.store)
            codes.view(torch.uint8)[page, :, slot] = to_pool(c, kv.spec.store).view(torch.uint8)
            scales[page, :, slot] = s

    def paged_attention(self, q, batch, kv, out, num_heads, scale, workspace=None, **more):
        if kv.spec.store is not None:
            kv = dataclasses.replace(kv, spec=dataclasses.replace(kv.spec, store=None), k_pages=values(kv.k_pages, kv.k_scales),
                                     v_pages=values(kv.v_pages, kv.v_scales))
        super().paged_attention(q, batch, kv, out, num_heads, scale, workspace, **more)


def logits_of(config, weights, tokens, store):
    """Logits of one whole sequence whose layers attend to quantised keys and values."""
    import plain_qwen2 as plain
    x = plain.embed(weights["model.embed_tokens.weight"], tokens)
    positions = torch.arange(len(tokens))
    for layer in range(config["num_hidden_layers"]):
        made = []
        plain.block(x, weights, config, layer, positions, kv_out=made)
        held = [values(to_pool(c, store), s).to(x.dtype) for c, s in (quantise(rows.double(), store) for rows in made[0])]
        x = plain.block(x, weights, config, layer, positions, shared_kv=tuple(held))
    x = plain.rms_norm(x, weights["model.norm.weight"], config["rms_norm_eps"])
    head = weights["model.embed_tokens.weight"] if config.get("tie_word_embeddings") else weights["lm_head.weight"]
    return plain.linear(x, head)
