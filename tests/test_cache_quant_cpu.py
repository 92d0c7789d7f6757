"""Cache entries in eight bits, without a GPU: the plain statement's own properties, the lists of blocks, refusals."""
import dataclasses

import numpy as np
import pytest
import torch

import plain_cache_quant as plain
from kvcache_b200.kernels.api import CudaKernels, KernelError
from kvcache_b200.kernels.cache_plan import EXPAND_BLOCK, CacheExpandPlanner
from kvcache_b200.parts.base import PagedKVSpec, first_seen


@pytest.mark.parametrize("store", plain.STORES)
def test_a_row_is_off_by_half_a_step(store):
    x = torch.randn(400, 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 10.0 ** torch.linspace(-12, 12, 400)[:, None].double()
    codes, scales = plain.quantise(x, store)
    assert torch.equal(plain.to_pool(codes, store).float().double(), codes)              # they are codes
    back = plain.values(plain.to_pool(codes, store), scales)
    e = 2.0 ** (scales.double() - 127)[:, None]
    assert ((back - x).abs() <= 0.5 * plain.step_at(x / e, store) * e * (1 + 1e-12)).all()
    top = x.abs().amax(-1)
    assert (top <= plain.TOP[store] * e[:, 0]).all() and (top > plain.TOP[store] * e[:, 0] / 2).all()
    assert torch.equal(back.to(torch.bfloat16).double(), back)                           # exact in the compute type


@pytest.mark.parametrize("store", plain.STORES)
def test_rows_at_the_borders(store):
    x = torch.zeros(6, 32, dtype=torch.float64)
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3, 0] = plain.TOP[store] * 2.0 ** 3
    x[4, 0] = 1e30
    x[5, 0] = -1e-30
    codes, scales = plain.quantise(x, store)
    assert scales.tolist() == [127, 255, 255, 130, 177, 77]
    back = plain.values(plain.to_pool(codes, store), scales)
    assert (back[0] == 0).all() and torch.isnan(back[1]).all() and torch.isnan(back[2]).all()
    assert back[3, 0] == x[3, 0] and back[4, 0] == plain.TOP[store] * 2.0 ** 50 and back[5].abs().max() == 0


@pytest.mark.parametrize("reach, keep", [(0, 0), (1, 0), (64, 0), (100, 3), (70, 130), (-96, 0)])
@pytest.mark.parametrize("singles", [True, False])
def test_lists_of_blocks(reach, keep, singles):
    planner = CacheExpandPlanner(reach, keep if reach > 0 else 0, singles)
    starts, counts = [0, 0, 63, 64, 500, 1000, 17], [1, 64, 1, 2, 130, 1, 300]
    arrays, numbers = planner.plan(np.asarray(starts), np.asarray(counts))
    assert set(arrays) == ({"ranges", "portions"} if singles else {"portions"})
    assert all(len(a) <= planner.sections(sum(counts), len(counts))[name] for name, a in arrays.items())
    for name, total in (("ranges", "blocks"), ("portions", "portion_blocks")) if singles else (("portions", "portion_blocks"),):
        check_ranges(arrays[name].reshape(-1, 3), numbers[total], starts, counts, reach, keep, name == "ranges")


def check_ranges(ranges, total, starts, counts, reach, keep, singles):
    at = 0
    for i, (start, count) in enumerate(zip(starts, counts)):
        assert ranges[i, 0] == at
        end = ranges[i + 1, 0] - at
        blocks = [j if j < ranges[i, 1] else ranges[i, 2] + j - ranges[i, 1] for j in range(end)]
        assert blocks == sorted(set(blocks))
        if singles or count > 1:
            lo = first_seen(start, reach)
            want = {k // EXPAND_BLOCK for k in range(start + count) if k >= lo or (reach > 0 and k < keep)}
            assert set(blocks) == want
        else:
            assert not blocks
        at += end
    assert total == at == ranges[-1, 0]


def test_steps_of_single_tokens_have_one_plan():
    planner = CacheExpandPlanner(0, 0, False)
    assert planner.plan([5, 900], [1, 1])[1] == planner.plan([70, 3], [1, 1])[1] == {"portion_blocks": 0}


def _bare():
    return CudaKernels.__new__(CudaKernels)                  # the checks come before anything of a device


def _entry(store="e4m3", **changes):
    batch, kv = plain.make_step([(5, 2)], 2, 32, 8, "int8" if store == "int8" else "e4m3")
    return batch, dataclasses.replace(kv, **changes)


@pytest.mark.parametrize("changes, words", [
    (dict(spec=PagedKVSpec(2, 32, store="fp4")), "held as one of"),
    (dict(spec=PagedKVSpec(2, 32, value_dim=16, store="e4m3")), "as wide as keys"),
    (dict(spec=PagedKVSpec(2, 32, store="int8")), "torch.int8"),
    (dict(spec=PagedKVSpec(1, 32, store="e4m3")), "pages of a cache"),
    (dict(page_size=16), "pages of a cache"),
    (dict(k_scales=None), "scale bytes"),
    (dict(v_scales=torch.zeros(3, 2, 8)), "scale bytes"),
])
def test_views_that_are_refused(changes, words):
    batch, kv = _entry(**changes)
    with pytest.raises(KernelError, match=words):
        _bare()._quantised_entry(kv, "test")


@pytest.mark.parametrize("more, words", [
    (dict(norm_scope="all"), "norm_scope"), (dict(norm_after_rotation=True), "norm_after_rotation"), (dict(value_mix=(None, None)), "value_mix"),
    (dict(q_temperature=(0.1, 4)), "q_temperature"), (dict(key_dim=16), "key_dim"), (dict(value_dim=16), "value_dim"),
    (dict(queries_only=True), "queries alone"), (dict(q_norm=torch.ones(32), norm_eps=1e-6), "or for neither"),
    (dict(q_norm=torch.ones(32), k_norm=torch.ones(32)), "above zero"),
    (dict(q_norm=torch.ones(31), k_norm=torch.ones(32), norm_eps=1e-6), "as many as"),
    (dict(q_norm=torch.ones(32), k_norm=torch.ones(32, dtype=torch.bfloat16), norm_eps=1e-6), "k_norm is float32"),
])
def test_appends_that_are_refused(more, words):
    batch, kv = _entry()
    qkv, q = torch.zeros(2, 8 * 32), torch.zeros(2, 4 * 32)
    with pytest.raises(KernelError, match=words):
        _bare().qkv_rope_append(qkv, None, None, None, batch, kv, q, 4, **more)


def test_tables_that_are_refused():
    batch, kv = _entry()
    qkv, q = torch.zeros(2, 8 * 32), torch.zeros(2, 4 * 32)
    table = torch.zeros(8, 16)
    for bias, cos, sin, words in ((torch.zeros(255), None, None, "do not fit"), (torch.zeros(256, dtype=torch.float64), None, None, "bias is float32"),
                                  (None, table, None, "sines"), (None, table, torch.zeros(8, 8), "sines")):
        with pytest.raises(KernelError, match=words):
            _bare().qkv_rope_append(qkv, bias, cos, sin, batch, kv, q, 4)


@pytest.mark.parametrize("more, words", [
    (dict(sink=torch.zeros(3)), "sink is one"), (dict(sink=torch.zeros(4, dtype=torch.float64)), "sink is one"), (dict(slopes=torch.zeros(5)), "slopes is one")])
def test_attention_that_is_refused(more, words):
    batch, kv = _entry()
    q = torch.zeros(2, 4 * 32)
    with pytest.raises(KernelError, match=words):
        _bare().paged_attention(q, batch, kv, torch.zeros_like(q), 4, 1.0, **more)
    with pytest.raises(KernelError, match="block table"):
        _bare().paged_attention(q, batch, dataclasses.replace(kv, block_table=kv.block_table[:0]), torch.zeros_like(q), 4, 1.0)


def test_sizes_that_are_refused():
    batch, kv = _entry()
    with pytest.raises(KernelError, match="do not fit"):
        _bare().qkv_rope_append(torch.zeros(2, 7 * 32), None, None, None, batch, kv, torch.zeros(2, 4 * 32), 4)
    with pytest.raises(KernelError, match="do not fit"):
        _bare().paged_attention(torch.zeros(2, 3 * 32), batch, kv, torch.zeros(2, 3 * 32), 3, 1.0)
    with pytest.raises(KernelError, match="compute type only"):
        _bare().norm_qkv_rope_append(torch.zeros(2, 64), torch.zeros(1, 64), None, torch.ones(64), 1e-6, None, None, batch, kv, torch.zeros(2, 64), 2)
    with pytest.raises(KernelError, match="list of blocks"):
        _bare().expand_cache(batch, kv, torch.bfloat16, None)


def test_room_for_what_grows():
    from kvcache_b200.engine.workspace import Workspace
    ws = Workspace("cpu")
    sizes, moved = (1, 2, 3, 5, 8, 9, 16, 4), []
    for n in sizes:
        view = ws.roomy("x", (n, 3), torch.float32)
        assert view.shape == (n, 3)
        moved.append(ws.moved)
    assert moved == [0, 1, 2, 3, 3, 4, 4, 4] and ws._buffers["x"].numel() == 48
    assert ws.roomy("x", (5, 3), torch.float32).data_ptr() == ws._buffers["x"].data_ptr()


def test_the_read_back_lets_no_successor_start_early():
    """Attention looks pages up before it waits for the kernel in front of it, and so does what fetches keys of earlier steps.  That is sound only
    where no kernel right before it makes them: the read-back's successor may therefore start only when the read-back has ended, unless the caller knows
    that it waits first - as the attention of portions does, which is told."""
    import os
    import re
    import kvcache_b200
    with open(os.path.join(os.path.dirname(kvcache_b200.__file__), "csrc", "cache_quant.cu")) as fh:
        text = re.sub(r"//[^\n]*", "", fh.read())
    kernels = {m.group(1): m.end() for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\(", text)}
    assert {"expand_any_kernel", "expand_vec_kernel"} <= set(kernels)
    for name in ("expand_any_kernel", "expand_vec_kernel"):
        body = text[kernels[name]:]
        body = body[:body.index("\n}\n")]
        assert "pdl_wait()" in body and body.count("pdl_launch_dependents") == body.count("if (p.early) pdl_launch_dependents();") == 1
    with open(os.path.join(os.path.dirname(kvcache_b200.__file__), "csrc", "attention_pairs.cu")) as fh:
        pairs = re.sub(r"//[^\n]*", "", fh.read())
    copies = pairs[pairs.index("const int* table = p.block_table"):]
    assert copies.index("p.made_table) { waited = true; pdl_wait();") < copies.index("lookup(0)")
