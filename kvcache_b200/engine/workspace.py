"""Named scratch buffers that outlive a step: activations keep their addresses from step
to step (which CUDA graphs need) and nothing is allocated once the sizes have been seen.
The reference allocates its activation buffers once, sized for the longest prompt
(apps/qwen_serve.cu:69-83)."""
from __future__ import annotations

from typing import Dict, Tuple

import torch


class Workspace:
    def __init__(self, device: torch.device | str, row_capacity: int = 0):
        """`row_capacity`: buffers whose first dimension is at most this many rows are made
        for that many rows at once, so they never move afterwards."""
        self.device = torch.device(device)
        self.row_capacity = row_capacity
        self._buffers: Dict[str, torch.Tensor] = {}
        self._views: Dict[tuple, torch.Tensor] = {}      # (name, shape, dtype) -> the view handed out last time
        self.moved = 0        # how many times an existing buffer was replaced by a larger one
        self.frozen = False   # set while a CUDA graph is captured or replayed: growing is an error

    def buffer(self, name: str, shape: Tuple[int, ...], dtype: torch.dtype, room: int = 0) -> torch.Tensor:
        """`room`: a new buffer is made for this first dimension (0: for `row_capacity` rows where they are enough)."""
        key = (name, tuple(shape), dtype)
        view = self._views.get(key)
        if view is not None:
            return view                                  # the same request as before: nothing to compute or to slice
        count = 1
        for s in shape:
            count *= int(s)
        buf = self._buffers.get(name)
        if buf is None or buf.dtype != dtype or buf.numel() < count:
            if self.frozen:
                raise RuntimeError(f"workspace buffer '{name}' would have to grow to {count} elements "
                                   f"while its addresses are pinned by a CUDA graph")
            capacity = max(count, 1)
            if shape and (room or 0 < int(shape[0]) <= self.row_capacity):
                capacity = max(capacity, count // max(int(shape[0]), 1) * (room or self.row_capacity))
            if buf is not None:
                if buf.dtype == dtype:
                    capacity = max(capacity, buf.numel())
                self.moved += 1                          # before anything can fail: the old addresses are gone from here on
                for old in [k for k in self._views if k[0] == name]:
                    del self._views[old]                 # views of the buffer that is replaced
                view = buf = None                        # its memory is given back before the larger one is asked for
                del self._buffers[name]
            buf = torch.empty(capacity, dtype=dtype, device=self.device)
            self._buffers[name] = buf
        view = buf[:count].view(shape)
        self._views[key] = view
        return view

    def roomy(self, name: str, shape: Tuple[int, ...], dtype: torch.dtype, most: int = 1 << 62) -> torch.Tensor:
        """Like `buffer`, with room for the next power of two of the first dimension, or for `most` of it where that is less: what grows from step to
        step moves a few times only."""
        n = int(shape[0])
        return self.buffer(name, shape, dtype, room=max(n, min(1 << max(n - 1, 0).bit_length(), most)))

    def zeros(self, name: str, shape: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        """Like `buffer`, but zero when first made (or remade); its users leave it zero."""
        count = 1
        for s in shape:
            count *= int(s)
        before = self._buffers.get(name)
        view = self.buffer(name, shape, dtype)
        if self._buffers[name] is not before:
            self._buffers[name].zero_()
        return view

    def bytes(self) -> int:
        return sum(b.numel() * b.element_size() for b in self._buffers.values())
