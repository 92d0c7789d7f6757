"""Cache entries in eight bits on the GPU: append, read-back and attention against float64.

Tolerances count roundings.  A bfloat16 result is off by 2^-8 of itself at most (half a step).  Attention weights are rounded to 2^-11 of
themselves where the codes are read in place (half precision) and to 2^-8 where they are read back first (bfloat16); both sums of a
quotient err so, hence twice that times sum p|v| in the worst case.  Weights below 2^-14 of a row's largest are off by 2^-25 of it.  A
score s = scale q.k of D products carries an error of a few 2^-24 of scale |q|.|k|, and moves a weight by that share: 2^-18 of it is allowed."""
import dataclasses

import pytest
import torch

import plain_cache_quant as plain
from helpers import batch_to
from plain_cache_quant import kv_to, make_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF, BF16 = 2.0 ** -11, 2.0 ** -8


@pytest.fixture(scope="module")
def kernels():
    from kvcache_b200.kernels.api import CudaKernels
    return CudaKernels(DEV)


@pytest.fixture()
def workspace():
    from kvcache_b200.engine.workspace import Workspace
    return Workspace(DEV)


def planners(kernels, kv_like, singles=True):
    reach, keep = kv_like
    return (kernels.paged_attention_planner(), kernels.cache_expand_planner(reach, keep, singles))


def pool_bytes(kv):
    return [t.view(torch.uint8).cpu().clone() for t in (kv.k_pages, kv.v_pages, kv.k_scales, kv.v_scales)]


# ---- append ------------------------------------------------------------------------------------------------------------------
def projections(T, Hq, Hkv, D, dtype, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D + extra, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    return qkv.to(dtype), torch.randn((Hq + 2 * Hkv) * D, generator=g), 1 + 0.3 * torch.randn(2, D, generator=g)


def turned(qkv, bias, weights, eps, cos, sin, batch, Hq, Hkv, D):
    """[T, Hq + 2 Hkv, D] float64: what is rounded to queries or quantised."""
    x = qkv[:, :(Hq + 2 * Hkv) * D].double()
    x = (x if bias is None else x + bias.double()).view(-1, Hq + 2 * Hkv, D)
    qk = x[:, :Hq + Hkv]
    if eps:
        qk = qk / (qk.square().mean(-1, keepdim=True) + eps).sqrt()
        if weights is not None:
            qk = qk * torch.cat([weights[0].expand(Hq, D), weights[1].expand(Hkv, D)]).double()
    if cos is not None:
        half = cos.shape[1]
        c, s = cos[batch.positions.long()].double()[:, None], sin[batch.positions.long()].double()[:, None]
        a, b = qk[..., :half], qk[..., half:2 * half]
        qk = torch.cat([a * c - b * s, b * c + a * s, qk[..., 2 * half:]], -1)
    return torch.cat([qk, x[:, Hq + Hkv:]], 1)


def angles(length, half):
    a = torch.arange(length, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    return a.cos().float(), a.sin().float()


def check_rows(pages, scales, want, store):
    """Stored rows of float64 rows `want`: within half a step of them, and 2^-20 of a row's largest for float32's roundings before it."""
    got, byte = plain.quantise(want, store)
    e = 2.0 ** (scales.double() - 127)
    amax = want.abs().amax(-1)
    fine = torch.isfinite(amax)
    assert (scales[~fine] == 255).all() and (pages.view(torch.uint8)[~fine] == 0).all()
    border = (amax / (plain.TOP[store] * 2.0 ** (byte.double() - 127))).sub(1).abs() < 2.0 ** -18
    border |= (amax / (plain.TOP[store] * 2.0 ** (byte.double() - 128))).sub(1).abs() < 2.0 ** -18
    assert ((scales == byte) | border)[fine].all()
    back = plain.values(pages, scales)
    inside = amax <= plain.TOP[store] * 2.0 ** 50
    y = want / e[..., None]
    slack = 0.5 * plain.step_at(y.abs() * (1 + 2.0 ** -20), store) * e[..., None] + 2.0 ** -20 * amax[..., None]
    ok = ((back - want).abs() <= slack) | ~(fine & inside)[..., None]
    assert ok.all(), (back - want).abs()[~ok].max()


# (segments, Hq, Hkv, D, page, type, bias, norm eps, weights, rotated halves, columns behind)
APPENDS = [
    ([(0, 1)], 14, 2, 64, 16, torch.bfloat16, True, 0.0, False, 32, 0),
    ([(11, 1), (0, 1), (64, 1)], 28, 4, 128, 16, torch.bfloat16, True, 0.0, False, 64, 0),
    ([(0, 300), (5, 33)], 16, 2, 128, 32, torch.bfloat16, False, 1e-6, True, 64, 0),
    ([(7, 129), (40, 1)], 32, 8, 128, 8, torch.bfloat16, True, 1e-5, True, 32, 8),
    ([(3, 70)], 4, 1, 64, 64, torch.bfloat16, True, 1e-6, False, 0, 16),
    ([(3, 41)], 4, 2, 256, 16, torch.bfloat16, False, 0.0, False, 16, 0),
    ([(3, 41)], 8, 2, 32, 4, torch.bfloat16, True, 1e-6, True, 16, 0),
    ([(3, 41)], 3, 3, 96, 2, torch.bfloat16, True, 1e-6, True, 48, 0),
    ([(3, 19)], 5, 1, 20, 1, torch.bfloat16, True, 1e-6, True, 5, 3),
    ([(3, 41)], 6, 2, 64, 16, torch.float32, True, 1e-6, True, 32, 0),
    ([(3, 41), (0, 2)], 5, 5, 33, 8, torch.float32, False, 0.0, False, 11, 1),
]


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("case", APPENDS)
def test_append(kernels, case, store):
    segments, Hq, Hkv, D, page, dtype, with_bias, eps, weighted, half, extra = case
    batch, kv = make_step(segments, Hkv, D, page, store, seed=3)
    qkv, bias, weights = projections(batch.num_tokens, Hq, Hkv, D, dtype, 4, extra)
    # Rows of zeros, of infinities and NaN, of very large and very small numbers, among the values.
    if batch.num_tokens > 20 and not with_bias:
        v = qkv[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D]
        v[1], v[2, 0], v[3, 1], v[4], v[5] = 0.0, float("inf"), float("nan"), v[4] * 1e30, v[5] * 1e-30
    bias, weights = bias if with_bias else None, weights if weighted else None
    cos, sin = angles(max(s + c for s, c in segments), half) if half else (None, None)
    want = turned(qkv, bias, weights, eps, cos, sin, batch, Hq, Hkv, D)
    dev, place = kv_to(kv, DEV), lambda t: None if t is None else t.to(DEV)
    before = pool_bytes(dev)
    q = torch.empty(batch.num_tokens, Hq * D, dtype=dtype, device=DEV)
    kernels.qkv_rope_append(qkv.to(DEV), place(bias), place(cos), place(sin), batch_to(batch, DEV), dev, q, Hq,
                            q_norm=None if weights is None else weights[0].to(DEV), k_norm=None if weights is None else weights[1].to(DEV), norm_eps=eps)
    kernels.check_errors()
    want_q = want[:, :Hq].reshape(batch.num_tokens, -1)
    slack = want_q.abs() * (BF16 if dtype == torch.bfloat16 else 2.0 ** -24) + want[:, :Hq].abs().amax(-1, keepdim=True).expand(-1, -1, D).reshape(want_q.shape) * 2.0 ** -20
    assert ((q.cpu().double() - want_q).abs() <= slack).all()
    pos, seg = batch.positions.long(), batch.row_segment.long()
    pages, slots = kv.block_table[seg, pos // page].long(), pos % page
    for codes, scales, rows in ((dev.k_pages, dev.k_scales, want[:, Hq:Hq + Hkv]), (dev.v_pages, dev.v_scales, want[:, Hq + Hkv:])):
        check_rows(codes.cpu().view(torch.uint8)[pages, :, slots].contiguous().view(codes.dtype), scales.cpu()[pages, :, slots], rows, store)
    written = torch.zeros(kv.k_scales.shape[0], page, dtype=torch.bool)
    written[pages, slots] = True
    for old, new in zip(before, pool_bytes(dev)):              # every other slot as it was
        keep = ~written[:, None].expand(old.shape[:3])
        assert torch.equal(old[keep], new[keep])


def test_append_of_queries_alone_and_of_a_reader(kernels):
    batch, kv = make_step([(3, 30)], 2, 64, 16, "e4m3", seed=3)
    qkv, bias, weights = projections(30, 6, 2, 64, torch.bfloat16, 5)
    cos, sin = angles(33, 32)
    args = (bias.to(DEV), cos.to(DEV), sin.to(DEV), batch_to(batch, DEV))
    out = []
    for columns, writes, alone in ((640, True, False), (640, False, False), (384, False, True)):
        dev = dataclasses.replace(kv_to(kv, DEV), writes=writes)
        before, q = pool_bytes(dev), torch.empty(30, 384, dtype=torch.bfloat16, device=DEV)
        kernels.qkv_rope_append(qkv[:, :columns].contiguous().to(DEV), *args, dev, q, 6, queries_only=alone)
        out.append(q)
        assert all(torch.equal(a, b) for a, b in zip(before, pool_bytes(dev))) == (not writes)
    kernels.check_errors()
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 20)])
def test_append_reports_pages_and_positions(kernels, dtype, D):
    from kvcache_b200.kernels.api import KernelError
    batch, kv = make_step([(3, 30)], 2, D, 16, "int8", seed=3)
    qkv, bias, _ = projections(30, 4, 2, D, dtype, 5)
    q = torch.empty(30, 4 * D, dtype=dtype, device=DEV)
    for table, length, words in ((-1, 64, "page"), (10 ** 6, 64, "page"), (None, 20, "position")):
        dev = kv_to(kv, DEV)
        if table is not None:
            dev.block_table[0, 1] = table
        cos, sin = angles(length, D // 4)
        kernels.qkv_rope_append(qkv.to(DEV), bias.to(DEV), cos.to(DEV), sin.to(DEV), batch_to(batch, DEV), dev, q, 4)
        with pytest.raises(KernelError, match=words):
            kernels.check_errors()


# ---- read-back ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("case", [
    ([(0, 1)], 2, 64, 16, None, 0, None), ([(0, 64), (100, 1), (63, 1), (500, 77)], 4, 128, 16, None, 0, None),
    ([(900, 30), (10, 5)], 2, 96, 8, 200, 0, None), ([(900, 30), (70, 1)], 1, 32, 64, 100, 70, None),
    ([(333, 100), (48, 48)], 2, 64, 32, None, 0, 48), ([(30, 41)], 3, 20, 1, None, 0, None)])
def test_read_back(kernels, workspace, case, store, dtype):
    segments, Hkv, D, page, window, keep, chunk = case
    reach = window or -(chunk or 0)
    batch, kv = make_step(segments, Hkv, D, page, store, seed=6, window=window, keep=keep, chunk=chunk, planners=planners(kernels, (reach, keep)))
    kv.v_scales[kv.block_table[0, 0].long(), 0, 0] = 255
    for i, (start, _) in enumerate(segments):                 # pages that the window has passed are given back
        lo = plain_first(start, reach)
        kv.block_table[i, -(-keep // page):lo // page] = -1
    view = kernels.expand_cache(batch_to(batch, DEV), kv_to(kv, DEV), dtype, workspace)
    kernels.check_errors()
    at = 0
    ranges = batch.plans[kernels.cache_expand_planner(reach, keep).name].arrays["ranges"].view(-1, 3)
    for i, (start, count) in enumerate(segments):
        k, v = plain.rows_of(kv, i, start + count)
        lo = plain_first(start, reach)
        for b in range(int(ranges[i + 1, 0] - ranges[i, 0])):
            block = b if b < ranges[i, 1] else int(ranges[i, 2]) + b - int(ranges[i, 1])
            assert int(view.block_table[i, block]) == at
            key = torch.arange(64 * block, 64 * block + 64)
            seen = (key < start + count) & ((key >= lo) | (key < (keep if reach > 0 else 0)))
            for got, rows in ((view.k_pages[at], k), (view.v_pages[at], v)):
                want = torch.zeros(64, Hkv, D, dtype=torch.float64)
                want[seen] = rows[key[seen]]
                assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=12345.0), torch.nan_to_num(want.transpose(0, 1), nan=12345.0))
            at += 1
    assert at == view.k_pages.shape[0]


def plain_first(start, reach):
    from kvcache_b200.parts.base import first_seen
    return first_seen(start, reach)


# ---- attention ---------------------------------------------------------------------------------------------------------------
def check_attention(out, ref, size, strength, longest_value, keys, weight_step):
    got = out.cpu().double().view(ref.shape)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    result = BF16 if out.dtype == torch.bfloat16 else 2.0 ** -24
    slack = ref.abs() * result + size * (2 * weight_step + 2 * 2.0 ** -18 * strength[..., None] + 2.0 ** -16) + keys * 2.0 ** -25 * longest_value
    ok = ((got - ref).abs() <= slack) | nan
    assert ok.all(), ((got - ref).abs() / slack)[~ok].max()


def run_attention(kernels, workspace, segments, Hq, Hkv, D, page, store, dtype=torch.bfloat16, window=None, keep=0, chunk=None, sink=False, cap=None, slopes=False,
                  seed=8, spread=0.7, strength=1.0, plan=True, change=None, weight_step=BF16, calls=2):
    reach = window or -(chunk or 0)
    batch, kv = make_step(segments, Hkv, D, page, store, seed=seed, window=window, keep=keep, chunk=chunk, spread=spread,
                          planners=planners(kernels, (reach, keep)) if plan else ())
    if change is not None:
        change(kv)
    g = torch.Generator().manual_seed(seed + 1)
    q = (strength * torch.randn(batch.num_tokens, Hq * D, generator=g)).to(dtype)
    sinks = 3.0 * torch.randn(Hq, generator=g) if sink else None
    slope = 0.02 * torch.rand(Hq, generator=g) if slopes else None
    ref, size, most = plain.attention(q, batch, kv, Hq, D ** -0.5, sinks, cap, slope)
    for i, (start, _) in enumerate(segments):
        kv.block_table[i, -(-keep // page):plain_first(start, reach) // page] = -1
    v = plain.values(kv.v_pages, kv.v_scales)
    place = lambda t: None if t is None else t.to(DEV)
    dev, first = kv_to(kv, DEV), None
    for _ in range(calls):
        out = torch.full((batch.num_tokens, Hq * D), float("nan"), dtype=dtype, device=DEV)
        kernels.paged_attention(q.to(DEV), batch_to(batch, DEV), dev, out, Hq, D ** -0.5, workspace, sink=place(sinks), score_cap=cap, slopes=place(slope))
        kernels.check_errors()
        check_attention(out, ref, size, most, v[torch.isfinite(v)].abs().max(), max(s + c for s, c in segments),
                        weight_step if dtype == torch.bfloat16 else 2.0 ** -20)
        assert first is None or torch.equal(torch.nan_to_num(first), torch.nan_to_num(out))       # the same bits
        first = out
    return out, ref


# (segments, Hq, Hkv, D, page, options)
STEPS = [
    ([(0, 1)], 14, 2, 64, 16, {}),
    ([(1, 1), (15, 1), (16, 1), (127, 1), (128, 1), (300, 1), (31, 1)], 14, 2, 64, 16, {}),
    ([(4000, 1), (0, 1), (900, 1)], 28, 4, 128, 16, {}),
    ([(5000, 1)], 16, 2, 128, 64, {}),
    ([(700, 1), (90, 1)], 32, 8, 128, 8, dict(sink=True)),
    ([(700, 1), (90, 1)], 12, 1, 96, 4, dict(sink=True, cap=15.0, slopes=True)),
    ([(700, 1), (90, 1)], 20, 1, 32, 32, {}),
    ([(700, 1)], 40, 1, 64, 16, {}),
    ([(2000, 1), (50, 1), (300, 1)], 16, 2, 128, 16, dict(window=256, keep=5, sink=True)),
    ([(2000, 1), (50, 1), (300, 1)], 14, 2, 64, 16, dict(window=1)),
    ([(2000, 1), (50, 1), (300, 1)], 4, 4, 64, 16, dict(window=300, keep=400)),
    ([(2000, 1), (95, 1), (96, 1)], 4, 2, 64, 16, dict(chunk=96)),
    ([(600, 2), (30, 5), (0, 3)], 14, 2, 64, 16, {}),
    ([(600, 37)], 16, 2, 128, 16, dict(sink=True)),
    ([(600, 37), (60, 21)], 8, 2, 64, 8, dict(window=50, keep=3)),
    ([(600, 37), (60, 21)], 8, 2, 64, 8, dict(chunk=64, cap=10.0)),
    ([(0, 130), (1000, 1), (77, 64), (5, 1)], 12, 2, 128, 32, {}),
    ([(1000, 500), (3, 1)], 4, 2, 64, 16, dict(slopes=True)),
    ([(0, 450)], 4, 1, 128, 16, dict(window=100)),
    ([(300, 9), (0, 40), (7, 1)], 4, 2, 48, 16, {}),
    ([(300, 9), (0, 40), (7, 1)], 4, 2, 64, 2, {}),
    ([(300, 9), (0, 40), (7, 1)], 3, 1, 20, 1, dict(sink=True)),
]


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("step", STEPS)
def test_attention(kernels, workspace, step, store):
    run_attention(kernels, workspace, *step[:5], store, **step[5])


@pytest.mark.parametrize("step", [STEPS[1], STEPS[5], STEPS[8], STEPS[14], STEPS[16], STEPS[21]])
def test_attention_without_lists_or_workspace(kernels, step):
    run_attention(kernels, None, *step[:5], "e4m3", plan=False, **step[5])


def test_a_batch_that_does_not_say_how_long_its_portions_are(kernels, workspace):
    """`max_q_len` left at its default: every row has its result all the same, and rows behind the last request's stay as they are."""
    batch, kv = make_step([(40, 9), (3, 1)], 2, 64, 16, "int8")
    batch = batch_to(dataclasses.replace(batch, max_q_len=1), DEV)
    q = torch.randn(12, 8 * 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = torch.full_like(q, 7.0).to(DEV)
    kernels.paged_attention(q.to(DEV), batch, kv_to(kv, DEV), out, 8, 0.125, workspace)
    kernels.check_errors()
    ref, size, most = plain.attention(q[:10], make_step([(40, 9), (3, 1)], 2, 64, 16, "int8")[0], kv, 8, 0.125)
    check_attention(out[:10], ref, size, most, plain.values(kv.v_pages, kv.v_scales).abs().max(), 49, BF16)
    assert (out[10:] == 7.0).all()


@pytest.mark.parametrize("segments", [[(40, 1), (100, 1)], [(40, 30), (100, 1)]])
def test_pages_of_an_odd_number_of_tokens(kernels, workspace, segments):
    run_attention(kernels, workspace, segments, 8, 2, 64, 12, "e4m3")


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("step", [STEPS[1], STEPS[5], STEPS[8], STEPS[13], STEPS[17], STEPS[19]])
def test_attention_in_float32(kernels, workspace, step, store):
    run_attention(kernels, workspace, *step[:5], store, dtype=torch.float32, **step[5])


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("segments", [[(900, 1), (40, 1)], [(500, 20)], [(100, 400)]])
def test_rows_of_very_different_sizes(kernels, workspace, segments, store):
    """Value rows whose scales differ by 2^40, and keys whose scores spread over hundreds."""
    run_attention(kernels, workspace, segments, 14, 2, 64, 16, store, spread=4.0, strength=2.0)


@pytest.mark.parametrize("segments", [[(600, 1), (40, 1)], [(600, 20), (40, 3)]])
def test_rows_that_are_not_finite_reach_those_that_see_them(kernels, workspace, segments):
    """A key or value row that held an infinity makes the results of the heads that see it NaN, and no other."""
    def change(kv):
        page, slot = int(kv.block_table[0, 100 // 16]), 100 % 16
        kv.k_scales[page, 0, slot], kv.k_pages.view(torch.uint8)[page, 0, slot] = 255, 0
        page = int(kv.block_table[1, 41 // 16]) if segments[1][1] > 1 else int(kv.block_table[1, 0])
        slot = 41 % 16 if segments[1][1] > 1 else 3
        kv.v_scales[page, 1, slot], kv.v_pages.view(torch.uint8)[page, 1, slot] = 255, 0
    out, ref = run_attention(kernels, workspace, segments, 8, 2, 64, 16, "e4m3", change=change)
    nan = torch.isnan(ref).any(-1)
    rows = segments[0][1]
    assert nan[:rows, :4].all() and not nan[:rows, 4:].any()
    seen = torch.arange(segments[1][1]) >= 1 if segments[1][1] > 1 else torch.ones(1, dtype=torch.bool)
    assert torch.equal(nan[rows:, 4:], seen[:, None].expand(-1, 4)) and not nan[rows:, :4].any()


@pytest.mark.parametrize("segments", [[(600, 1), (40, 1)], [(600, 20), (40, 3)], [(100, 390)]])
@pytest.mark.parametrize("window", [None, 64])
def test_what_lies_in_unseen_slots_does_not_matter(kernels, workspace, segments, window):
    """Slots behind a request's last key, pages nobody holds and pages that a window has passed: any bytes."""
    def change(kv):
        owned = torch.zeros(kv.k_scales.shape[0], 16, dtype=torch.bool)
        for i, (start, count) in enumerate(segments):
            for key in range(plain_first(start, window or 0), start + count):
                owned[int(kv.block_table[i, key // 16]), key % 16] = True
        for codes, scales in ((kv.k_pages, kv.k_scales), (kv.v_pages, kv.v_scales)):
            codes.view(torch.uint8)[(~owned)[:, None].expand(-1, 2, -1)] = 0x7f
            scales[(~owned)[:, None].expand(-1, 2, -1)] = 255
    run_attention(kernels, workspace, segments, 8, 2, 64, 16, "e4m3", window=window, change=change)


@pytest.mark.parametrize("segments, D, page", [([(600, 1), (40, 1)], 64, 16), ([(600, 1)], 128, 4), ([(600, 20)], 64, 16), ([(100, 400)], 64, 16), ([(40, 3)], 20, 16)])
def test_attention_reports_pages(kernels, workspace, segments, D, page):
    from kvcache_b200.kernels.api import KernelError
    for bad in (-1, 10 ** 6):
        batch, kv = make_step(segments, 2, D, page, "int8", planners=planners(kernels, (0, 0)))
        kv.block_table[0, 1] = bad
        q = torch.zeros(batch.num_tokens, 8 * D, dtype=torch.bfloat16, device=DEV)
        kernels.paged_attention(q, batch_to(batch, DEV), kv_to(kv, DEV), torch.empty_like(q), 8, 1.0, workspace)
        with pytest.raises(KernelError, match="page"):
            kernels.check_errors()


def test_more_requests_than_one_launch_counts(kernels, workspace):
    run_attention(kernels, workspace, [(i % 40, 1) for i in range(4100)], 2, 1, 32, 16, "e4m3", calls=1)


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("segments", [[(300, 1), (40, 1)], [(300, 20), (40, 1)], [(100, 200)]])
def test_pools_that_start_at_odd_addresses(kernels, workspace, segments, store):
    Hq, Hkv, D, page = 8, 2, 64, 16
    batch, kv = make_step(segments, Hkv, D, page, store, planners=planners(kernels, (0, 0)))
    def off_by_one(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        out = flat[1:].view(t.shape)
        out.view(torch.uint8).copy_(t.view(torch.uint8))
        return out
    pool = kv_to(kv, DEV)
    odd = dataclasses.replace(pool, **{name: off_by_one(getattr(kv, name)) for name in ("k_pages", "v_pages", "k_scales", "v_scales")})
    q = torch.randn(batch.num_tokens, Hq * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    b, out = batch_to(batch, DEV), torch.empty(batch.num_tokens, Hq * D, dtype=torch.bfloat16, device=DEV)
    kernels.paged_attention(q.to(DEV), b, odd, out, Hq, D ** -0.5, workspace)
    ref, size, most = plain.attention(q, batch, kv, Hq, D ** -0.5)
    check_attention(out, ref, size, most, plain.values(kv.v_pages, kv.v_scales).abs().max(), max(s + c for s, c in segments), BF16)
    qkv, bias, _ = projections(batch.num_tokens, Hq, Hkv, D, torch.bfloat16, 3)
    for entry in (pool, odd):                # the same codes, wherever the pool lies
        kernels.qkv_rope_append(qkv.to(DEV), bias.to(DEV), None, None, b, entry, torch.empty_like(out), Hq)
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(pool, name).view(torch.uint8), getattr(odd, name).view(torch.uint8))
    view = kernels.expand_cache(b, odd, torch.bfloat16, workspace)
    got = view.k_pages.clone(), view.v_pages.clone()
    view = kernels.expand_cache(b, pool, torch.bfloat16, workspace)
    assert torch.equal(got[0], view.k_pages) and torch.equal(got[1], view.v_pages)
    kernels.check_errors()


# Attention kernels look pages up, and may fetch keys that earlier steps have written, before the kernel in front of them has ended.
@pytest.mark.parametrize("steps, Hq, Hkv, D, page", [
    (([(700, 1), (90, 1), (1200, 1)], [(40, 1), (2000, 1), (333, 1)]), 8, 2, 48, 16),
    (([(700, 1), (90, 1), (1200, 1)], [(40, 1), (2000, 1), (333, 1)]), 8, 2, 64, 24),
    (([(700, 1), (90, 1), (1200, 1)], [(40, 1), (2000, 1), (333, 1)]), 8, 2, 128, 24),
    (([(700, 300), (900, 500)], [(100, 200), (0, 700)]), 8, 2, 64, 16),
    (([(700, 300), (900, 500)], [(100, 200), (0, 700)]), 16, 2, 128, 16)])
def test_steps_in_turn_read_back_what_is_theirs(kernels, workspace, steps, Hq, Hkv, D, page):
    """Two steps of other lengths take turns, nothing between them, in one workspace: each gets the bits that it gets alone."""
    made = []
    for i, segments in enumerate(steps):
        batch, kv = make_step(segments, Hkv, D, page, "e4m3", seed=20 + i, planners=planners(kernels, (0, 0)))
        q = torch.randn(batch.num_tokens, Hq * D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
        made.append((q.to(DEV), batch_to(batch, DEV), kv_to(kv, DEV), plain.attention(q, batch, kv, Hq, D ** -0.5), kv, segments))
    def attend(q, batch, kv):
        out = torch.full_like(q, float("nan"))
        kernels.paged_attention(q, batch, kv, out, Hq, D ** -0.5, workspace)
        return out
    got = []
    for _ in range(12):
        for q, batch, kv, *_ in made:
            got.append(attend(q, batch, kv))
    kernels.check_errors()
    for i, out in enumerate(got):
        assert torch.equal(out, got[i % 2])
    for out, (_, _, _, (ref, size, most), kv, segments) in zip(got, made):
        check_attention(out, ref, size, most, plain.values(kv.v_pages, kv.v_scales).abs().max(), max(s + c for s, c in segments), BF16)


# ---- together ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("store", plain.STORES)
def test_a_prompt_in_portions_then_tokens(kernels, workspace, store):
    """Append and attention of one request as an engine runs it - portions, then single tokens, the last of them replayed from a graph on a
    stream of its own - against attention over what the pages then hold."""
    Hq, Hkv, D, page = 14, 2, 64, 16
    sizes = [70, 3, 400, 1, 1, 1]
    total = sum(sizes)
    qkv, bias, _ = projections(total, Hq, Hkv, D, torch.bfloat16, 9)
    cos, sin = angles(total, 32)
    steps, start = [], 0
    for n in sizes:
        steps.append(make_step([(start, n)], Hkv, D, page, store, seed=10, planners=planners(kernels, (0, 0), singles=False)))
        start += n
    table = torch.arange(-(-total // page), dtype=torch.int32)[None]
    pool = kv_to(dataclasses.replace(steps[-1][1], block_table=table), DEV)
    side = torch.cuda.Stream()
    row = 0
    for i, (batch, _) in enumerate(steps):
        n, b = batch.num_tokens, batch_to(batch, DEV)
        x = qkv[row:row + n].to(DEV)
        q, out = torch.empty(n, Hq * D, dtype=torch.bfloat16, device=DEV), torch.empty(n, Hq * D, dtype=torch.bfloat16, device=DEV)
        args = (bias.to(DEV), cos.to(DEV), sin.to(DEV))
        def step():
            kernels.qkv_rope_append(x, *args, b, pool, q, Hq)
            kernels.paged_attention(q, b, pool, out, Hq, D ** -0.5, workspace)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            if i == len(steps) - 1:
                first = out.clone()
                out.zero_()
                side.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
                graph.replay()
                graph.replay()
        side.synchronize()
        if i == len(steps) - 1:
            assert torch.equal(out, first)
        kernels.check_errors()
        host = dataclasses.replace(pool, k_pages=pool.k_pages.cpu(), v_pages=pool.v_pages.cpu(), block_table=table, k_scales=pool.k_scales.cpu(), v_scales=pool.v_scales.cpu())
        ref, size, most = plain.attention(q.cpu(), batch, host, Hq, D ** -0.5)
        v = plain.values(host.v_pages, host.v_scales)
        check_attention(out, ref, size, most, v.abs().max(), total, BF16)
        want = turned(qkv[row:row + n], bias, None, 0.0, cos, sin, batch, Hq, Hkv, D)
        pos = batch.positions.long()
        check_rows(host.k_pages.view(torch.uint8)[table[0][pos // page].long(), :, pos % page].contiguous().view(host.k_pages.dtype),
                   host.k_scales[table[0][pos // page].long(), :, pos % page], want[:, Hq:Hq + Hkv], store)
        row += n
