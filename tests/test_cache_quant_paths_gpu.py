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
