"""Cache entries in eight bits on the GPU: paths of the kernels that need certain sizes or orders of work, each shown to be the one that ran.

Tolerances are those of test_cache_quant_gpu.py where nothing else is said."""
import dataclasses

import pytest
import torch

import plain_cache_quant as plain
import test_cache_quant_gpu as quant
from helpers import batch_to
from plain_cache_quant import kv_to, make_step
from test_cache_quant_gpu import DEV, kernels, workspace  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# ---- what is read back and then attended to -----------------------------------------------------------------------------------
@pytest.mark.parametrize("steps, Hq, Hkv, D, page, singles, forms", [
    (([(3000, 600)], [(2500, 700)]), 16, 2, 128, 2, False, {"attention_pairs"}),
    (([(3000, 600), (900, 1)], [(2500, 700), (1200, 1)]), 16, 2, 128, 1, True, {"attention_pairs", "flash_decode_tma"}),
    (([(700, 300), (900, 500)], [(100, 200), (0, 700)]), 8, 2, 64, 2, False, {"attention_units"}),
    (([(700, 1), (90, 1), (1200, 1)], [(40, 1), (2000, 1), (333, 1)]), 8, 2, 64, 1, True, {"flash_decode_tma"}),
    (([(700, 1), (90, 1), (1200, 1)], [(40, 1), (2000, 1), (333, 1)]), 8, 2, 80, 16, True, {"flash_decode_cluster"})])
def test_steps_in_turn_whose_pages_are_made(kernels, workspace, steps, Hq, Hkv, D, page, singles, forms):  # noqa: F811
    """Forms whose codes no kernel reads in place: the read-back is right in front of kernels that elsewhere look pages up early."""
    before = kernels.launch_forms + kernels.launch_counts
    planners = quant.planners
    try:
        quant.planners = lambda k, kv_like: planners(k, kv_like, singles)
        quant.test_steps_in_turn_read_back_what_is_theirs(kernels, workspace, steps, Hq, Hkv, D, page)
    finally:
        quant.planners = planners
    ran = kernels.launch_forms + kernels.launch_counts - before
    assert {"cache_expand", *forms} <= set(ran) and not ran["attention_quant"] and not ran["attention_quant_any"]


# ---- queries of any size ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("power", [99, 101, 110, 120, 127, 128])
@pytest.mark.parametrize("segments, D, dtype", [([(40, 1), (700, 1)], 64, torch.bfloat16), ([(300, 9)], 64, torch.bfloat16), ([(40, 1), (300, 9)], 20, torch.bfloat16),
                                                ([(40, 1), (300, 1)], 64, torch.float32)])
def test_queries_up_to_the_largest_bfloat16(kernels, workspace, segments, D, dtype, power, store):  # noqa: F811
    """Keys 2^-30 times as large as usual bring the scores back into float32, where they differ by far more than a softmax needs: every row is
    the value of its best key, and nothing else."""
    Hq, Hkv = 8, 2
    batch, kv = make_step(segments, Hkv, D, 16, store, seed=12)
    kv.k_scales.sub_(30)
    g = torch.Generator().manual_seed(2)
    q = (2 * torch.rand(batch.num_tokens, Hq * D, generator=g) - 1) * 0.99
    q.view(-1, D)[:, 0] = 0.99                                 # every head's largest lies below 2^power, half of it above 2^(power - 1)
    q = (q.double() * 2.0 ** power).float().to(torch.bfloat16).to(dtype)
    assert torch.isfinite(q).all()
    want = torch.zeros(batch.num_tokens, Hq, D, dtype=torch.float64)
    for i, (start, count) in enumerate(segments):
        k, v = plain.rows_of(kv, i, start + count)
        for r in range(count):
            row = int(batch.seg_q_start[i]) + r
            for h in range(Hq):
                query = q[row].double().view(Hq, D)[h]
                s = (k[:start + r + 1, h // 4] @ query)
                best, second = torch.topk(s, 2).values
                # Fixed point of 2^-15 of a row's largest number: a score is off by 2^-15 of the largest times the sum of |k|.
                off = 2.0 ** -14 * query.abs().max() * k[:start + r + 1, h // 4].abs().sum(-1).max()
                if best - second > 2 * off:
                    want[row, h] = v[int(s.argmax()), h // 4]
                else:
                    want[row, h] = float("nan")
    assert torch.isnan(want[..., 0]).double().mean() < 0.1
    out = torch.full_like(q, float("nan")).to(DEV)
    kernels.paged_attention(q.to(DEV), batch_to(batch, DEV), kv_to(kv, DEV), out, Hq, 1.0, workspace)
    kernels.check_errors()
    got = out.cpu().double().view(want.shape)
    assert torch.isfinite(got).all() and ((got == want) | torch.isnan(want)).all()


# ---- every key reaches the rows that see it, once -------------------------------------------------------------------------------
UNIT, PIECE_COST, GROUP, MOST = 32, 12, 16, 32             # as in csrc/attention_quant.cu


def seen_from(start, reach, keep):
    """(first units kept, first unit of the rest, first key) that a row at `start` sees."""
    lo = quant.plain_first(start, reach)
    first = lo // UNIT
    return min(-(-keep // UNIT), first) if reach > 0 else 0, first, lo


def how_it_is_cut(kernels, segments, Hq, Hkv, D, reach=0, keep=0):
    """("whole" or "line", most pieces of one row tile, keys of a piece) of a step whose codes are read in place: the kernel's own rule, restated."""
    group, longest = Hq // Hkv, max(c for _, c in segments)
    rows = 8 if longest * group <= 8 else 16
    blocks = kernels.sm_count * ((4 if D <= 64 else 3) if rows == 8 else (3 if D <= 64 else 2))
    tiles = []
    for start, count in segments:
        kept, first, _ = seen_from(start, reach, keep)
        tiles += [kept + (start + count - 1) // UNIT + 1 - first] * (-(-count * group // rows) * Hkv)
    units, items, least = sum(tiles), len(tiles), kernels.quant_min_units
    line = -(-(units + items * PIECE_COST) // blocks)
    if items < blocks:
        share = -(-units // (blocks - items))
        if 4 * share <= 5 * max(2 * least, line):
            sizes = [max(share, n if n <= 2 * least else least if n <= 12 * least else 2 * least) for n in tiles]
            return "whole", max(-(-n // s) for n, s in zip(tiles, sizes)), UNIT * max(sizes)
    share = max(2 * least, line)
    return "line", max(n // share + 2 if n > share else 1 for n in tiles), UNIT * share


# (segments, Hq, Hkv, D, page, window, kept, chunk, how it is cut, least pieces of a row tile)
CUTS = [
    ([(19999, 1)], 7, 1, 64, 16, None, 0, None, "whole", MOST + 1),
    ([(149999, 1)], 7, 1, 64, 16, None, 0, None, "whole", GROUP * MOST + 1),       # groups of groups of pieces
    ([(40000, 2), (3000, 1)], 14, 2, 64, 32, None, 0, None, "whole", MOST + 1),
    ([(24000, 1)], 8, 1, 128, 16, None, 0, None, "whole", MOST + 1),
    ([(9000, 1)], 9, 1, 32, 4, None, 0, None, "whole", MOST + 1),
    ([(9000, 1)], 4, 1, 96, 16, None, 0, None, "whole", MOST + 1),
    ([(37 * i % 2000, 1) for i in range(120)], 28, 4, 64, 16, None, 0, None, "line", 2),
    ([(53 * i % 1100, 1) for i in range(50)], 16, 8, 128, 16, None, 0, None, "line", 2),
    ([(600, 100), (31, 64), (1500, 90)], 28, 4, 64, 16, None, 0, None, "line", 1),
    ([(5000, 3), (64, 1)], 14, 2, 64, 16, None, 0, None, "whole", 2),
    ([(3000, 1), (1030, 1), (50, 1)], 16, 2, 128, 16, 1000, 70, None, "whole", 2),
    ([(3000, 20), (200, 1)], 16, 2, 64, 16, 500, 33, None, "whole", 2),
    ([(3490, 40)], 16, 2, 64, 8, None, 0, 700, "whole", 2),
]
cuts = pytest.mark.parametrize("cut", CUTS, ids=lambda c: f"{len(c[0])}x{max(s for s, _ in c[0])}.{c[3]}")


def cut_step(kernels, cut, store, seed):
    segments, Hq, Hkv, D, page, window, keep, chunk, mode, pieces = cut
    reach = window or -(chunk or 0)
    got = how_it_is_cut(kernels, segments, Hq, Hkv, D, reach, keep)
    assert got[0] == mode and got[1] >= pieces, got
    per = [-(-(s + c) // page) for s, c in segments]
    g = torch.Generator().manual_seed(seed)
    n, pages = len(segments), sum(per) + 2
    order, table, used = torch.randperm(pages, generator=g).to(torch.int32), torch.full((n, max(per) + 1), -1, dtype=torch.int32), 0
    for i, p in enumerate(per):
        table[i, :p] = order[used:used + p]
        used += p
    counts, starts = torch.tensor([c for _, c in segments]), torch.tensor([s for s, _ in segments])
    seg = torch.repeat_interleave(torch.arange(n), counts)
    q_start = torch.cumsum(counts, 0) - counts
    pos = torch.arange(int(counts.sum())) - q_start[seg] + starts[seg]
    i32 = lambda t: t.to(torch.int32)
    from kvcache_b200.parts.base import STORE_DTYPES, PagedKVSpec, PagedKVView, StepBatch
    batch = StepBatch(len(pos), n, 0, i32(torch.arange(len(pos))), i32(pos), i32(seg), i32(q_start), i32(counts), i32(starts + counts), i32(torch.arange(n)),
                      torch.zeros(0, dtype=torch.int32), max_q_len=int(counts.max()), max_kv_len=int((starts + counts).max()))
    zeros = lambda: torch.zeros(pages, Hkv, page, D, dtype=torch.uint8).view(STORE_DTYPES[store])
    kv = PagedKVView(PagedKVSpec(Hkv, D, window, None, keep, chunk, store=store), zeros(), zeros(), table, page, True,
                     torch.full((pages, Hkv, page), 127, dtype=torch.uint8), torch.full((pages, Hkv, page), 127, dtype=torch.uint8))
    return batch, kv, reach, keep


def code_bytes(x, store):
    """Bytes of numbers that are codes."""
    return plain.to_pool(x, store).view(torch.uint8)


def sees(key, pos, reach, keep):
    return key <= pos and (key >= quant.plain_first(pos, reach) or (reach > 0 and key < keep))


@cuts
@pytest.mark.parametrize("store", plain.STORES)
def test_every_key_counts_once(kernels, workspace, cut, store):  # noqa: F811
    """Queries of zeros weigh all keys alike; a value is 1 in the column of its unit of 32 keys (modulo the head's size), so that a column's result
    is the share of its keys among those that the row sees.  Weights, sums and their quotient are exact but for the quotient's roundings, and a
    unit that is lost or met twice is at least 1 % of its column."""
    segments, Hq, Hkv, D, page = cut[:5]
    batch, kv, reach, keep = cut_step(kernels, cut, store, 5)
    table, values = kv.block_table.long(), kv.v_pages.view(torch.uint8)
    want = torch.zeros(batch.num_tokens, D, dtype=torch.float64)
    for i, (start, count) in enumerate(segments):
        key = torch.arange(start + count)
        column = key // UNIT % D
        values[table[i, key // page], :, key % page] = code_bytes(torch.nn.functional.one_hot(column, D).double(), store)[:, None]
        for r in range(count):
            pos = start + r
            seen = (key <= pos) & ((key >= quant.plain_first(pos, reach)) | ((key < keep) if reach > 0 else torch.zeros_like(key, dtype=torch.bool)))
            share = torch.bincount(column[seen], minlength=D).double()
            want[int(batch.seg_q_start[i]) + r] = share / share.sum()
    q = torch.zeros(batch.num_tokens, Hq * D, dtype=torch.bfloat16, device=DEV)
    dev, placed, first, before = kv_to(kv, DEV), batch_to(batch, DEV), None, kernels.launch_counts["attention_quant"]
    for _ in range(3):
        out = torch.full_like(q, float("nan"))
        kernels.paged_attention(q, placed, dev, out, Hq, 1.0, workspace)
        got = out.cpu().double().view(-1, Hq, D)
        assert ((got - want[:, None]).abs() <= want[:, None] * (quant.BF16 + 2.0 ** -22)).all()
        assert first is None or torch.equal(first, out)         # and the tickets are zero again
        first = out
    kernels.check_errors()
    assert kernels.launch_counts["attention_quant"] == before + 3


@cuts
@pytest.mark.parametrize("store", plain.STORES)
def test_single_keys_are_found(kernels, workspace, cut, store):  # noqa: F811
    """One key a column outweighs all others by e^64 for a query along that column: the row is that key's value, bit for bit, but that a zero may be off by
    the others' share (150,000 keys with values of up to 448: 150,000 * 448 e^-64 < 2^-60).  The keys lie at the borders of units, of pieces, of windows
    and of the request, and where a row does not see one its result is something else."""
    segments, Hq, Hkv, D, page = cut[:5]
    batch, kv, reach, keep = cut_step(kernels, cut, store, 6)
    g = torch.Generator().manual_seed(7)
    table, top = kv.block_table.long(), plain.TOP[store]
    piece = how_it_is_cut(kernels, segments, Hq, Hkv, D, reach, keep)[2]
    chosen = {}
    for i, (start, count) in enumerate(segments):
        length = start + count
        rows = torch.arange(length)
        rand = torch.randn(length, Hkv, D, generator=g, dtype=torch.float64)
        kv.v_pages.view(torch.uint8)[table[i, rows // page], :, rows % page] = code_bytes(plain.round_code((rand * top / 8).clamp(-top, top), store), store)
        kv.v_scales[table[i, rows // page], :, rows % page] = (120 + torch.randint(0, 8, (length, Hkv), generator=g)).to(torch.uint8)
        kept, first, lo = seen_from(start, reach, keep)
        edges = {0, length - 1, start, lo, max(lo - 1, 0), keep, max(keep - 1, 0)}
        edges |= {first * UNIT + piece * x + y for x in range(1, 1 + (length - first * UNIT) // piece) for y in (-1, 0)}
        edges |= {UNIT * int(x) + y for x in torch.randint(0, length // UNIT + 1, (2 * D,), generator=g) for y in (-1, 0)}
        edges = [e for e in sorted(edges) if 0 <= e < length]
        order = torch.randperm(len(edges), generator=g).tolist()
        picked = [edges[x] for x in order[:D]]
        picked += [picked[0]] * (D - len(picked))
        chosen[i] = picked
        for d in reversed(range(D)):                         # (a key that stands for several columns has its largest number in the first)
            row = torch.zeros(D, dtype=torch.float64)
            row[d] = 64.0
            if picked.index(picked[d]) == d:
                kv.k_pages.view(torch.uint8)[table[i, picked[d] // page], :, picked[d] % page] = code_bytes(row, store)
    dev, placed = kv_to(kv, DEV), batch_to(batch, DEV)
    group = Hq // Hkv
    for turn in range(-(-D // group)):
        q = torch.zeros(batch.num_tokens, Hq, D, dtype=torch.bfloat16)
        for h in range(Hq):
            q[:, h, (turn * group + h % group) % D] = 1.0
        out = torch.full((batch.num_tokens, Hq * D), float("nan"), dtype=torch.bfloat16, device=DEV)
        kernels.paged_attention(q.view(batch.num_tokens, Hq * D).to(DEV), placed, dev, out, Hq, 1.0, workspace)
        got = out.cpu().view(-1, Hq, D)
        for i, (start, count) in enumerate(segments):
            for h in range(Hq):
                d = (turn * group + h % group) % D
                key = chosen[i][d]
                if chosen[i].index(key) != d:
                    continue
                place = table[i, key // page], h // group, key % page
                value = plain.values(kv.v_pages[place], kv.v_scales[place]).to(torch.bfloat16)
                for r in range(count):
                    row = got[int(batch.seg_q_start[i]) + r, h]
                    same = torch.equal(torch.where((value == 0) & (row.abs() < 2.0 ** -60), value, row), value)
                    assert same == sees(key, start + r, reach, keep), (i, h, key, r)
    kernels.check_errors()


# ---- how far results are off ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("step", [s for s in quant.STEPS if s[3] in (32, 64, 96, 128) and s[4] >= 4 and max(c for _, c in s[0]) < 128] +
                         [([(53 * i % 1100, 1) for i in range(50)], 16, 8, 128, 16, {}), ([(19999, 1)], 7, 1, 64, 16, {})])
def test_codes_read_in_place_are_held_to_half_precision(kernels, workspace, step, store):  # noqa: F811
    """A weight is rounded to 2^-11 of itself (below 2^-14 of the reference: by 2^-25 of it, and a value is at most twice the largest of all), the result to
    2^-8; a score is off by float32's roundings, a few 2^-24 of scale |q| |k|, of its cap and of its distance term, 2^-20 of which is allowed, and for int8 by the queries' fixed point, 2^-15 of
    a row's largest number beside every key number.  Numerator and denominator err so, hence twice."""
    segments, Hq, Hkv, D, page, options = step
    reach, keep = options.get("window") or -(options.get("chunk") or 0), options.get("keep", 0)
    batch, kv = make_step(segments, Hkv, D, page, store, seed=31, window=options.get("window"), keep=keep, chunk=options.get("chunk"))
    g = torch.Generator().manual_seed(32)
    q = torch.randn(batch.num_tokens, Hq * D, generator=g).to(torch.bfloat16)
    sink = 3.0 * torch.randn(Hq, generator=g) if options.get("sink") else None
    slopes = 0.02 * torch.rand(Hq, generator=g) if options.get("slopes") else None
    ref, size, strength = plain.attention(q, batch, kv, Hq, D ** -0.5, sink, options.get("cap"), slopes)
    off = 2.0 ** -20 * (strength + (options.get("cap") or 0.0) + (0.02 * max(s + c for s, c in segments) if slopes is not None else 0.0))
    if store == "int8":
        for i, (start, count) in enumerate(segments):
            k = plain.rows_of(kv, i, start + count)[0].abs().sum(-1).amax(0).repeat_interleave(Hq // Hkv)        # [Hq]
            rows = slice(int(batch.seg_q_start[i]), int(batch.seg_q_start[i]) + count)
            off[rows] += 2.0 ** -15 * q[rows].double().view(count, Hq, D).abs().amax(-1) * k * D ** -0.5
    place = lambda t: None if t is None else t.to(DEV)
    out = torch.full((batch.num_tokens, Hq * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    before = kernels.launch_counts["attention_quant"]
    kernels.paged_attention(q.to(DEV), batch_to(batch, DEV), kv_to(kv, DEV), out, Hq, D ** -0.5, workspace, sink=place(sink), score_cap=options.get("cap"), slopes=place(slopes))
    kernels.check_errors()
    assert kernels.launch_counts["attention_quant"] == before + 1
    largest, keys = plain.values(kv.v_pages, kv.v_scales).abs().max(), max(s + c for s, c in segments)
    slack = ref.abs() * quant.BF16 + size * (2 * quant.HALF + 2 * off[..., None]) + 2 * keys * 2.0 ** -25 * largest
    error = (out.cpu().double().view(ref.shape) - ref).abs()
    assert (error <= slack).all(), (error / slack).max()
    # Taken together: the result's rounding, evenly spread, is off by 2^-8 / sqrt(3) of it at most; half precision's weights by no more than the sum of
    # all of theirs.
    rms = lambda x: x.square().mean().sqrt()
    assert rms(error) <= rms(ref) * quant.BF16 / 3 ** 0.5 + rms(size * (quant.HALF + off[..., None]))


# ---- streams and graphs ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D, page", [(64, 16), (128, 16), (48, 16)])
def test_two_streams_at_once(kernels, D, page):  # noqa: F811
    """Steps on two streams, each with a workspace of its own and nothing between them: the bits that each gets by itself."""
    from kvcache_b200.engine.workspace import Workspace
    Hq, Hkv = 16, 2
    steps = [[(3000, 1), (700, 1)], [(2000, 200), (9, 1)], [(1500, 1), (100, 1), (64, 1)], [(40, 30)]]
    made = []
    for side in range(2):
        one = []
        for i, segments in enumerate(steps):
            batch, kv = make_step(segments, Hkv, D, page, "e4m3", seed=50 + 10 * side + i, planners=quant.planners(kernels, (0, 0)))
            q = torch.randn(batch.num_tokens, Hq * D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
            one.append((q.to(DEV), batch_to(batch, DEV), kv_to(kv, DEV)))
        made.append(one)
    def run(side, workspace):
        out = []
        for q, batch, kv in made[side]:
            out.append(torch.full_like(q, float("nan")))
            kernels.paged_attention(q, batch, kv, out[-1], Hq, D ** -0.5, workspace)
        return out
    spaces, streams = [Workspace(DEV), Workspace(DEV)], [torch.cuda.Stream(), torch.cuda.Stream()]
    want = []
    for side in range(2):
        with torch.cuda.stream(streams[side]):
            want.append(run(side, spaces[side]))
        torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for side in range(2):
            with torch.cuda.stream(streams[side]):
                got.append((side, run(side, spaces[side])))
    torch.cuda.synchronize()
    kernels.check_errors()
    for side, outs in got:
        assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(outs, want[side]))


@pytest.mark.parametrize("store", plain.STORES)
def test_graphs_that_share_a_workspace_and_lengths_that_grow(kernels, workspace, store):  # noqa: F811
    """Two recorded steps of single tokens in one workspace, replayed in turn, the requests longer every time: what a step gets that is launched."""
    Hq, Hkv, D, page, graphs = 14, 2, 64, 16, []
    for n, at in ((3, 0), (40, 1)):
        final = [(900 + 40 * i, 1) for i in range(n)]
        batch, kv = make_step(final, Hkv, D, page, store, seed=60 + at)
        q = torch.randn(n, Hq * D, generator=torch.Generator().manual_seed(at)).to(torch.bfloat16).to(DEV)
        placed, dev, out = batch_to(batch, DEV), kv_to(kv, DEV), torch.zeros(n, Hq * D, dtype=torch.bfloat16, device=DEV)
        step = lambda q=q, placed=placed, dev=dev, out=out: kernels.paged_attention(q, placed, dev, out, Hq, D ** -0.5, workspace)
        step()
        graphs.append((placed, out, step, q))
    torch.cuda.synchronize()
    recorded = []
    for placed, out, step, _ in graphs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        recorded.append(graph)
    for less in (880, 500, 31, 0):
        for (placed, out, step, _), graph in zip(graphs, recorded):
            full = 901 + 40 * torch.arange(len(out), device=DEV, dtype=torch.int32)
            placed.seg_kv_len.copy_(full - less)
            placed.positions.copy_(full - less - 1)
            torch.cuda.synchronize()
            out.fill_(float("nan"))
            step()
            torch.cuda.synchronize()
            want = out.clone()
            for _ in range(2):
                out.fill_(float("nan"))
                graph.replay()
                torch.cuda.synchronize()
                assert torch.isfinite(out).all() and torch.equal(out, want)
    kernels.check_errors()
