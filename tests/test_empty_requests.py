"""Steps in which some requests bring no token, as many requests as tokens among them."""
import numpy as np
import pytest
import torch

import plain_cache_quant as plain
from helpers import batch_to
from kvcache_b200.kernels.attention_plan import PagedAttentionPlanner
from plain_cache_quant import kv_to, make_step

DEV = "cuda:0"
COUNTS = [[3, 0, 0], [0, 2], [1, 0, 2], [0, 1, 1, 2], [200] + 199 * [0], [1, 1, 1], [0]]


@pytest.mark.parametrize("counts", COUNTS)
def test_every_row_is_on_the_lists(counts):
    starts = np.arange(len(counts)) * 7
    arrays, numbers = PagedAttentionPlanner().plan(starts, counts)
    assert arrays["decode_items"].tolist() == [i for i, c in enumerate(counts) if c == 1] and numbers["decode_items"] == counts.count(1)
    longer = {(i, r) for i, c in enumerate(counts) if c > 1 for r in range(c)}
    for name, rows, width in (("prefill_units", 64, 8), ("tc_units", 128, 8), ("tc_pairs", 256, 2)):
        if not longer and name not in arrays:
            continue
        on = {(int(u[0]), int(u[1]) + r) for u in arrays[name].reshape(-1, width) for r in range(rows) if int(u[1]) + r < counts[int(u[0])]}
        assert on == longer, name


@pytest.mark.gpu
@pytest.mark.parametrize("store", [None, "e4m3"])
@pytest.mark.parametrize("counts", COUNTS[:-1])
def test_attention(counts, store):
    from kvcache_b200.engine.workspace import Workspace
    from kvcache_b200.kernels.api import CudaKernels
    from test_cache_quant_gpu import BF16, check_attention
    kernels, Hq, Hkv, D = CudaKernels(DEV), 14, 2, 64
    segments = [(40 + 9 * i, c) for i, c in enumerate(counts)]
    batch, kv = make_step(segments, Hkv, D, 16, "e4m3", planners=(kernels.paged_attention_planner(), kernels.cache_expand_planner(0, 0)))
    q = torch.randn(batch.num_tokens, Hq * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    ref, size, most = plain.attention(q, batch, kv, Hq, D ** -0.5)
    v = plain.values(kv.v_pages, kv.v_scales)
    if store is None:                        # the same numbers, which bfloat16 holds
        wide = [plain.values(p, s).to(torch.bfloat16) for p, s in ((kv.k_pages, kv.k_scales), (kv.v_pages, kv.v_scales))]
        kv = plain.dataclasses.replace(kv, spec=kv.spec.unstored, k_pages=wide[0], v_pages=wide[1], k_scales=None, v_scales=None)
    out = torch.full_like(q, float("nan")).to(DEV)
    kernels.paged_attention(q.to(DEV), batch_to(batch, DEV), kv_to(kv, DEV), out, Hq, D ** -0.5, Workspace(DEV))
    kernels.check_errors()
    check_attention(out, ref, size, most, v.abs().max(), max(s + c for s, c in segments), BF16)
