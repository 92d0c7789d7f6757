"""Attention over pages that a kernel of the same step has read back, without a GPU: what the launchers are told, and the kernels' source."""
import os
import re
from collections import Counter

import pytest
import torch

import kvcache_b200
import plain_cache_quant as plain
from kvcache_b200.engine.workspace import Workspace
from kvcache_b200.kernels import api
from kvcache_b200.kernels.attention_plan import PagedAttentionPlanner
from kvcache_b200.kernels.cache_plan import CacheExpandPlanner


class Launchers:
    """In place of a library: every launch is noted, and succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def launch(*args):
            self.calls.append((name, args))
            return 1 << 16 if "scratch" in name or "tickets" in name or "max_clusters" in name else 0
        return launch

    def of(self, name):
        """The last launch's parameters by their names in the C declaration."""
        args = next(args for n, args in reversed(self.calls) if n == name)
        for file in sorted(os.listdir(CSRC)):
            found = re.search(r"KVB_API int %s\(([^)]*)\)" % name, source(file)) if file.endswith(".cu") else None
            if found:
                names = [re.search(r"(\w+)$", part.strip()).group(1) for part in found.group(1).split(",")]
                assert len(names) == len(args) == len(api._SIGNATURES[file[:-3]][name])
                return dict(zip(names, args))
        raise AssertionError(name)

    def names(self):
        return [n for n, _ in self.calls if "scratch" not in n and "tickets" not in n and "max_clusters" not in n]


CSRC = os.path.join(os.path.dirname(kvcache_b200.__file__), "csrc")


def source(file):
    with open(os.path.join(CSRC, file)) as fh:
        return re.sub(r"//[^\n]*", "", fh.read())


@pytest.fixture()
def kernels(monkeypatch):
    """A kernel set whose libraries note what they are told."""
    monkeypatch.setattr(api, "_ptr", lambda t: 0 if t is None else t.data_ptr())
    k = api.CudaKernels.__new__(api.CudaKernels)
    k.launches, k.launch_counts, k.launch_forms, k.libraries = 0, Counter(), Counter(), Launchers()
    k.device, k.sm_count, k.error_word = torch.device("cpu"), 148, torch.zeros(1, dtype=torch.int32)
    k._cache_quant = k._attn_generic = k.libraries
    k._attn_tc = k._attn_pairs = k._flash = {d: k.libraries for d in (32, 48, 64, 96, 128)}
    k._attn_quant = {d: (k.libraries, 1 << 16, 1 << 12) for d in (32, 64, 96, 128)}
    k._zero_slopes, k._tma_cluster_capacity = {}, {}
    k.tc_attention_min_rows, k.tc_history_min_rows, k.tc_history_min_units = 384, 128, 3
    k.tc_pairs_min_units, k.tc_pairs_units_a_tile, k.tc_pairs_min_tiles = 8, {64: 2, 128: 1}, 2
    k.tc_unit_min_tiles, k.prefill_unit_min_tiles = 16, 4
    k.flash_attention, k.decode_merge, k.decode_cluster_max, k.decode_pow2_splits = True, "tma", 8, True
    k.decode_ctas_wanted, k.decode_min_tiles, k.decode_superclusters, k.decode_super_min_tiles = 296, 4, 16, 8
    k._pinned_stream, k._attention_planner, k._expand_cache_planners = 0, None, {}
    return k


def step(kernels, segments, Hq, Hkv, D, page, dtype=torch.bfloat16, singles=True):
    batch, kv = plain.make_step(segments, Hkv, D, page, "e4m3", planners=(PagedAttentionPlanner(), CacheExpandPlanner(0, 0, singles)))
    return batch, kv, torch.zeros(batch.num_tokens, Hq * D, dtype=dtype)


@pytest.mark.parametrize("early", [False, True])
def test_what_is_read_back_says_that_it_is_made(kernels, early):
    batch, kv, _ = step(kernels, [(40, 3), (9, 1)], 4, 2, 64, 16)
    view = kernels.expand_cache(batch, kv, torch.bfloat16, Workspace("cpu"), early=early)
    assert view.made and kernels.libraries.of("kvb_cache_expand")["early"] == early


# (segments, query heads, key heads, head size, page, with lists for single tokens, the launches that read what is read back)
@pytest.mark.parametrize("segments, Hq, Hkv, D, page, singles, readers", [
    ([(9000, 700)], 28, 4, 128, 2, False, {"kvb_attention_pairs": "made_table"}),
    ([(9000, 700)], 28, 4, 64, 1, False, {"kvb_attention_pairs": "made_table"}),
    ([(9000, 700)], 28, 4, 128, 16, False, {"kvb_attention_pairs": "made_table"}),
    ([(900, 1), (70, 1)], 8, 2, 64, 24, True, {"kvb_flash_decode_tma": "made"}),
    ([(900, 1), (70, 1)], 8, 2, 128, 2, True, {"kvb_flash_decode_tma": "made"}),
    ([(900, 1), (70, 1)], 8, 2, 48, 16, True, {"kvb_flash_decode_cluster": "made"}),
    ([(9000, 700), (70, 1)], 28, 4, 128, 2, True, {"kvb_attention_pairs": "made_table", "kvb_flash_decode_tma": "made"}),
])
def test_attention_over_what_is_read_back_is_told_so(kernels, segments, Hq, Hkv, D, page, singles, readers):
    batch, kv, q = step(kernels, segments, Hq, Hkv, D, page, singles=singles)
    kernels.paged_attention(q, batch, kv, torch.empty_like(q), Hq, 0.1, Workspace("cpu"))
    assert kernels.libraries.names() == ["kvb_cache_expand", *readers]
    for name, parameter in readers.items():
        assert kernels.libraries.of(name)[parameter] == 1
    # And of pages in the compute type, which earlier steps have written: not.
    kernels.libraries.calls.clear()
    wide = plain.dataclasses.replace(kv, spec=kv.spec.unstored, k_pages=kv.k_pages.to(torch.bfloat16), v_pages=kv.v_pages.to(torch.bfloat16))
    kernels.paged_attention(q, batch, wide, torch.empty_like(q), Hq, 0.1, Workspace("cpu"))
    for name, parameter in readers.items():
        if name in kernels.libraries.names():
            assert kernels.libraries.of(name)[parameter] == 0


def body_of(text, kernel):
    body = text[re.search(r"__global__[^;{]*?\b%s\(" % kernel, text).end():]
    return body[:body.index("\n}\n")]


def test_attention_waits_before_it_looks_at_made_pages():
    """Only a wait makes another kernel's writes visible, so every kernel that `paged_attention` launches waits before its first look at a table or at
    pages - always, or where the launch says that they are made in this step."""
    flash, generic = source("attention_flash.cu"), source("attention_generic.cu")
    for text, kernel in ((flash, "flash_decode_kernel"), (flash, "flash_prefill_kernel"), (generic, "paged_attention_generic_kernel"),
                         (generic, "attention_rows_kernel")):
        body = body_of(text, kernel)
        looks = [m.start() for m in re.finditer(r"block_table|\btable\[|k_pages|load_tile\(", body) if m.start() > body.index("{")]
        assert body.index("pdl_wait()") < min(looks), kernel
    units = body_of(source("attention_tc.cu"), "attention_tc_kernel")
    assert units.index("{ pdl_wait(); pdl_launch_dependents(); }") < units.index("p.block_table")
    cluster = body_of(flash, "flash_decode_cluster_kernel")
    assert "const bool early = !p.made && " in cluster
    assert re.search(r"if \(early\) \{[^}]*load_stage\(s\)", cluster).start() < cluster.index("pdl_wait()")      # the only look ahead of the wait
    assert cluster[cluster.index("const bool early"):cluster.index("pdl_wait()")].count("load_stage(") == 1
    tma = body_of(flash, "flash_decode_tma_kernel")
    assert tma.index("if (p.made) pdl_wait();") < tma.index("= lookup(") and tma.index("if (p.made) pdl_wait();") < tma.index("load_stage(i, ")


def test_rows_whose_keys_are_not_read_back_meet_no_kernel_that_reads_them(kernels):
    """Without the kernels that go by lists (`flash_attention` off) attention goes through every row of the step, so portions beside single tokens keep
    to their codes as well."""
    batch, kv, q = step(kernels, [(900, 300), (70, 1)], 8, 2, 64, 16, singles=False)
    for on, launches in ((True, ["kvb_cache_expand", "kvb_attention_tc", "kvb_attention_quant"]), (False, ["kvb_attention_quant"])):
        kernels.flash_attention = on
        kernels.libraries.calls.clear()
        kernels.paged_attention(q, batch, kv, torch.empty_like(q), 8, 0.1, Workspace("cpu"))
        assert kernels.libraries.names() == launches
    assert kernels.libraries.of("kvb_attention_quant")["max_q"] == 300


def test_a_read_back_keeps_no_more_than_its_limit(kernels):
    """The buffers grow by powers of two, but not past the limit that decides whether keys and values are read back."""
    block = 2 * 2 * 2 * 64 * 64                              # bytes of keys and values, two heads of 64 in bfloat16
    kernels.CACHE_EXPAND_MAX_BYTES = 100 * block + 17
    for capacity in (0, 48):
        workspace, held = Workspace("cpu", row_capacity=capacity), []
        for keys in (64 * 3, 64 * 5, 64 * 70, 64 * 100):
            batch, kv, q = step(kernels, [(keys - 130, 130)], 4, 2, 64, 16, singles=False)
            kernels.libraries.calls.clear()
            kernels.paged_attention(q, batch, kv, torch.empty_like(q), 4, 0.1, workspace)
            assert kernels.libraries.names()[0] == "kvb_cache_expand"
            held.append(sum(workspace._buffers[f"cache.expand_{x}_bf16"].numel() for x in "kv") * 2 // block)
        assert held == [4, 8, 100, 100]
    batch, kv, q = step(kernels, [(64 * 101 - 130, 130)], 4, 2, 64, 16, singles=False)
    kernels.libraries.calls.clear()
    kernels.paged_attention(q, batch, kv, torch.empty_like(q), 4, 0.1, workspace)
    assert kernels.libraries.names() == ["kvb_attention_quant"]


def test_a_buffer_that_grows_is_given_back_first(monkeypatch):
    workspace, alive = Workspace("cpu"), []
    workspace.buffer("x", (4,), torch.float32)
    real = torch.empty

    def empty(*args, **more):
        alive.append("x" in workspace._buffers or any(k[0] == "x" for k in workspace._views))
        raise MemoryError
    monkeypatch.setattr(torch, "empty", empty)
    with pytest.raises(MemoryError):
        workspace.buffer("x", (5,), torch.float32)
    assert alive == [False] and workspace.moved == 1          # whoever holds the old address is told even if there is no new one
    monkeypatch.setattr(torch, "empty", real)
    assert workspace.buffer("x", (3,), torch.float32).shape == (3,)


def test_a_model_that_refuses_leaves_every_layer_as_it_was():
    from types import SimpleNamespace
    from kvcache_b200.parts.attention import GQAAttention
    from kvcache_b200.parts.model import DecoderModel
    from kvcache_b200.parts.recurrent import GatedLinearAttention, ParallelMixer
    make = lambda **more: GQAAttention(64, 4, 2, 32, **{**dict(qkv_bias=False, out_bias=False, position=None, window=None, prefix="p.", dtype="float32"), **more})
    taken, refused = make(), make(q_temperature=(0.1, 8))
    for mixers in ([taken, refused], [refused, taken]):
        model = SimpleNamespace(blocks=[SimpleNamespace(mixer=m) for m in mixers])
        with pytest.raises(ValueError, match=f"layer {mixers.index(refused)}: a query temperature"):
            DecoderModel.store_cache(model, "int8")
        assert taken.cache_store is None and taken.cache_spec().store is None and refused.cache_store is None
    both = ParallelMixer.__new__(ParallelMixer)
    for left, right in ((taken, refused), (refused, taken)):
        both.left, both.right = left, right
        with pytest.raises(ValueError, match="temperature"):
            both.store_cache("int8")
        assert taken.cache_store is None
    both.right, both.left = GatedLinearAttention.__new__(GatedLinearAttention), taken
    both.store_cache("int8")
    assert taken.cache_store == "int8" and both.left.cache_spec().store == "int8"


def test_bytes_that_a_timed_attention_has_to_move():
    """Queries and results in their own type, codes and scale bytes as they are held."""
    from kvcache_b200.kernels.timing import KernelTiming
    batch, kv = plain.make_step([(40, 3), (9, 1)], 2, 64, 16, "int8")
    batch.host.update(starts=[40, 9], counts=[3, 1])
    q = torch.zeros(4, 8 * 64, dtype=torch.bfloat16)
    rows = 2 * q.numel() * 2
    assert KernelTiming._describe("paged_attention", (q, batch, kv, q, 8, 1.0), {}) == ("paged_attention", rows + 2 * 53 * 2 * (64 + 1))
    wide = plain.dataclasses.replace(kv, spec=kv.spec.unstored, k_pages=kv.k_pages.to(torch.bfloat16), v_pages=kv.v_pages.to(torch.bfloat16), k_scales=None, v_scales=None)
    assert KernelTiming._describe("paged_attention", (q, batch, wide, q, 8, 1.0), {}) == ("paged_attention", rows + 2 * 53 * 2 * 64 * 2)


def test_a_set_without_a_device_number_asks_for_the_current_device_at_every_call(monkeypatch):
    from types import SimpleNamespace
    now = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=100 + (now[0] if torch.device(device).index is None else torch.device(device).index)))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index)
    k = api.CudaKernels.__new__(api.CudaKernels)
    k._pinned_stream = None
    for name, streams in (("cuda", [100, 103]), ("cuda:2", [102, 102])):
        k.device, got = torch.device(name), []
        for now[0] in (0, 3):
            with k.on_current_stream():
                got.append(k._stream())
            assert k._stream() == got[-1]
        assert got == streams


@pytest.mark.parametrize("D, line", [(32, 128), (64, 128), (96, 192), (128, 128)])
def test_from_how_many_rows_on_portions_are_read_back(kernels, D, line):
    for rows in (line - 1, line):
        batch, kv, q = step(kernels, [(2000, rows)], 28, 4, D, 16, singles=False)
        kernels.libraries.calls.clear()
        kernels.paged_attention(q, batch, kv, torch.empty_like(q), 28, 0.1, Workspace("cpu"))
        assert (kernels.libraries.names()[0] == "kvb_cache_expand") == (rows == line)


def test_calls_whose_tables_are_shorter_than_the_step_are_refused(kernels):
    batch, kv, q = step(kernels, [(40, 3), (9, 1)], 4, 2, 64, 16)
    short = plain.dataclasses.replace(kv, block_table=kv.block_table[:1])
    with pytest.raises(api.KernelError, match="block table"):
        kernels.expand_cache(batch, short, torch.bfloat16, Workspace("cpu"))
    with pytest.raises(api.KernelError, match="block table"):
        kernels.qkv_rope_append(torch.zeros(4, 8 * 64, dtype=torch.bfloat16), None, None, None, batch, short, q, 4)
    other, _, _ = step(kernels, [(40, 3)], 4, 2, 64, 16)
    with pytest.raises(api.KernelError, match="list of blocks"):
        kernels.expand_cache(plain.dataclasses.replace(batch, plans=other.plans), kv, torch.bfloat16, Workspace("cpu"))
    with pytest.raises(api.KernelError, match="workspace"):
        kernels.expand_cache(batch, kv, torch.bfloat16, None)
    assert not kernels.libraries.calls
