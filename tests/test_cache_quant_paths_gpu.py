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
