"""Which blocks of a cache entry in eight bits a step reads back (csrc/cache_quant.cu, `CudaKernels.expand_cache`).

The reference's cache has one type and is read in place (src/qwen_kernels.cu:146-185).
"""
from __future__ import annotations

from typing import Dict, Tuple

import numpy as np

from ..parts.base import StepPlanner, first_seen

EXPAND_BLOCK = 64                # keys of a block that is read back, and tokens of the pages they become


class CacheExpandPlanner(StepPlanner):
    """`ranges`: [segments + 1, 3] - how many blocks the segments before this one bring, and which its own are: blocks 0 .. kept - 1 (the
    first keys that a window keeps), then those from `first` up to its last key's.  The last row holds the total alone.

    `singles` False: segments of one token bring none, so that a step of decoded tokens has the same counts whatever its lengths."""

    def __init__(self, reach: int = 0, keep_first: int = 0, singles: bool = True):
        self.reach, self.keep_first, self.singles = reach, keep_first, singles
        self.name = self.plan_name(reach, keep_first, singles)

    @staticmethod
    def plan_name(reach: int, keep_first: int, singles: bool) -> str:
        return f"cache_expand.r{reach}.k{keep_first}" + ("" if singles else ".portions")

    def sections(self, num_tokens: int, num_segments: int) -> Dict[str, int]:
        return {"ranges": 3 * (num_segments + 1)}

    def plan(self, starts, counts) -> Tuple[Dict[str, np.ndarray], Dict[str, int]]:
        ranges = np.zeros((len(counts) + 1, 3), dtype=np.int32)
        total = 0
        for i, (start, count) in enumerate(zip(starts, counts)):
            ranges[i, 0] = total
            if count < 1 or (count == 1 and not self.singles):
                continue
            first = first_seen(int(start), self.reach) // EXPAND_BLOCK
            kept = min(-(-self.keep_first // EXPAND_BLOCK), first) if self.reach > 0 else 0
            ranges[i, 1:] = kept, first
            total += kept + -(-(int(start) + int(count)) // EXPAND_BLOCK) - first
        ranges[-1, 0] = total
        return {"ranges": ranges.reshape(-1)}, {"blocks": total}
