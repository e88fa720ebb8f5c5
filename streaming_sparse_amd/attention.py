"""Workspace buffer cache, as local_experiments/video_runtime_v1/attention.py:7-13.

Buffers are keyed by (name, shape, device, dtype) and reused across calls, so a
returned output tensor is overwritten by the next call with the same key.
"""
from __future__ import annotations

import torch


class Workspace:
    def __init__(self):
        self.entries = {}
        self.views = {}

    def tensor(self, name, shape, device, dtype):
        # torch.Size is a tuple: equal shapes are equal keys in either form
        key = (name, shape if isinstance(shape, tuple) else tuple(shape),
               device if isinstance(device, torch.device) else torch.device(device), dtype)
        buf = self.entries.get(key)
        if buf is None:
            buf = self.entries[key] = torch.empty(shape, device=device, dtype=dtype)
        return buf

    def rows(self, name, shape, device, dtype):
        """(tensor, its pointer, the pointer behind its room): the first shape[0] rows
        of a buffer that has a power of two of them, so that calls of many row
        counts share a few buffers.  A call overwrites what one of another count
        left in the same."""
        key = (name, shape, device, dtype)
        view = self.views.get(key)
        if view is None:
            n = shape[0]
            room = 1 << (n - 1).bit_length() if n else 0
            buf = self.tensor(name, (room, *shape[1:]), device, dtype)
            start = buf.data_ptr()
            if len(self.views) >= 4096:
                self.views.clear()
            view = self.views[key] = buf[:n], start, start + buf.numel() * buf.element_size()
        return view

    def bytes(self):
        return sum(x.numel() * x.element_size() for x in self.entries.values())
