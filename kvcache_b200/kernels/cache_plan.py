"""Which blocks of a cache entry in eight bits a step reads back (csrc/cache_quant.cu, `CudaKernels.expand_cache`).

The reference's cache has one type and is read in place (src/qwen_kernels.cu:146-185).
"""
from __future__ import annotations

from typing import Dict, Tuple

import numpy as np

from ..parts.base import StepPlanner

EXPAND_BLOCK = 64                # keys of a block that is read back, and tokens of the pages they become


class CacheExpandPlanner(StepPlanner):
    """`ranges`: [segments + 1, 3] - how many blocks the segments before this one bring, and which its own are: blocks 0 .. kept - 1 (the
    first keys that a window keeps), then those from `first` up to its last key's.  The last row holds the total alone.
    `portions`: the same where segments of one token bring none (their attention reads the codes); without `singles` the only list, so that a
    step of decoded tokens has the same counts whatever its lengths."""

    def __init__(self, reach: int = 0, keep_first: int = 0, singles: bool = True):
        self.reach, self.keep_first, self.singles = reach, keep_first, singles
        self.name = self.plan_name(reach, keep_first, singles)

    @staticmethod
    def plan_name(reach: int, keep_first: int, singles: bool) -> str:
        return f"cache_expand.r{reach}.k{keep_first}" + ("" if singles else ".portions")

    def sections(self, num_tokens: int, num_segments: int) -> Dict[str, int]:
        words = 3 * (num_segments + 1)
        return {"ranges": words, "portions": words} if self.singles else {"portions": words}

    def _ranges(self, starts, counts, least: int) -> np.ndarray:
        starts, counts = np.asarray(starts, dtype=np.int64), np.asarray(counts, dtype=np.int64)
        if self.reach > 0:
            lo = np.maximum(0, starts - self.reach + 1)
        elif self.reach < 0:
            lo = starts - starts % -self.reach
        else:
            lo = np.zeros_like(starts)
        first = lo // EXPAND_BLOCK
        kept = np.minimum(-(-self.keep_first // EXPAND_BLOCK), first) if self.reach > 0 else np.zeros_like(first)
        blocks = np.where(counts >= least, kept + -(-(starts + counts) // EXPAND_BLOCK) - first, 0)
        ranges = np.zeros((len(counts) + 1, 3), dtype=np.int32)
        np.cumsum(blocks, out=ranges[1:, 0])
        ranges[:-1, 1], ranges[:-1, 2] = kept, first
        return ranges

    def plan(self, starts, counts) -> Tuple[Dict[str, np.ndarray], Dict[str, int]]:
        portions = self._ranges(starts, counts, 2)
        arrays, numbers = {"portions": portions.reshape(-1)}, {"portion_blocks": int(portions[-1, 0])}
        if self.singles:
            ranges = self._ranges(starts, counts, 1)
            arrays["ranges"], numbers["blocks"] = ranges.reshape(-1), int(ranges[-1, 0])
        return arrays, numbers
