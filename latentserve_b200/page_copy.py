"""Copying pages inside a cache's pools -- host side.

`copy_pages` is the device half of forking a sequence and of compacting a pool
(`cache.fork`, `cache.compact`): page dst[i] becomes a copy of page src[i] in every pool it is
given, all layers, one launch. The reference shares whole pages by reference counts only
(cache/block_allocator.py:40-162) and never moves one.
"""

from __future__ import annotations

import ctypes
from typing import Sequence

import numpy as np
import torch

from latentserve_b200 import _lib


class _Pool(ctypes.Structure):
    _fields_ = [("base", ctypes.c_void_p), ("layer_stride", ctypes.c_int64), ("page_stride", ctypes.c_int64),
                ("page_bytes", ctypes.c_int32), ("layers", ctypes.c_int32)]


def _describe(t: torch.Tensor, block_dim: int) -> _Pool:
    if not t.is_cuda:
        raise RuntimeError("latentserve_b200 has no CPU path: tensors must be on a CUDA device")
    if t.dim() <= block_dim:
        raise ValueError(f"a pool needs a page axis {block_dim}")
    run = 1
    for size, stride in zip(reversed(t.shape[block_dim + 1:]), reversed(t.stride()[block_dim + 1:])):
        if size != 1 and stride != run:
            raise ValueError("a page must be one dense run of memory")
        run *= size
    size = t.element_size()
    return _Pool(t.data_ptr(), t.stride(0) * size if block_dim else 0, t.stride(block_dim) * size, run * size,
                 t.shape[0] if block_dim else 1)


def _ids(x, what: str) -> np.ndarray:
    """Page ids as int32, refused where they would not survive the conversion."""
    a = np.asarray(x)
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise ValueError(f"{what} must be a flat sequence of whole numbers")
    if a.size and (a.min() < 0 or a.max() >= 2 ** 31):
        raise ValueError(f"{what} holds a page id outside the pool")
    return np.ascontiguousarray(a, dtype=np.int32)


def copy_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int], block_dim: int = 0) -> None:
    """pool[dst[i]] = pool[src[i]] for every tensor of `pools`, whose axis `block_dim` (0, or 1
    behind an axis of layers) counts the pages; any type, each page one dense run. src and dst are
    host sequences of page ids: they are read before the call returns, and a captured call
    replays with the same ids. A source may serve several destinations; a destination given
    twice, or that is a source as well, is refused."""
    if block_dim not in (0, 1):
        raise ValueError("block_dim must be 0 or 1")
    if not pools:
        return
    blocks, device = pools[0].shape[block_dim] if pools[0].dim() > block_dim else 0, pools[0].device
    table = (_Pool * len(pools))(*(_describe(t, block_dim) for t in pools))
    if any(t.shape[block_dim] != blocks or t.device != device for t in pools):
        raise ValueError("the pools must have one number of pages, on one device")
    s, d = _ids(src, "src"), _ids(dst, "dst")
    if s.size != d.size:
        raise ValueError(f"{s.size} source pages for {d.size} destinations")
    if s.size == 0:
        return
    if max(int(s.max()), int(d.max())) >= blocks:
        raise ValueError(f"a page id lies outside the pool of {blocks} pages")
    rc = _lib.lib().ls_copy_pages(table, len(pools), s.ctypes.data, d.ctypes.data, int(s.size), blocks,
                                  _lib.raw_stream(device.index))
    _lib.check(rc, "copy_pages")
