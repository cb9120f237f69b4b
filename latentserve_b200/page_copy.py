"""Copying pages inside a cache's pools -- host side.

`copy_pages` is the device half of forking a sequence and of compacting a pool
(`cache.fork`, `cache.compact`): page dst[i] becomes a copy of page src[i] in every pool it is
given, all layers, one launch. The reference shares whole pages by reference counts only
(cache/block_allocator.py:40-162) and never moves one.
"""

from __future__ import annotations

import ctypes
from array import array
from typing import Sequence

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


def _ids(x, what: str) -> array:
    """Page ids as int32, refused where they would not survive the conversion."""
    try:
        return array("i", x)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{what} must be a flat sequence of page ids (whole numbers): {e}") from None


class PagePools:
    """The pools one kind of copy goes through, described once: for who copies again and again
    (a cache). Keeps the tensors alive."""

    def __init__(self, pools: Sequence[torch.Tensor], block_dim: int = 0):
        if block_dim not in (0, 1):
            raise ValueError("block_dim must be 0 or 1")
        self.pools = list(pools)
        self.table = (_Pool * len(self.pools))(*[_describe(t, block_dim) for t in self.pools])
        self.blocks = self.pools[0].shape[block_dim] if self.pools else 0
        self.index = self.pools[0].get_device() if self.pools else -1
        if any(t.shape[block_dim] != self.blocks or t.get_device() != self.index for t in self.pools):
            raise ValueError("the pools must have one number of pages, on one device")

    def copy(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """pool[dst[i]] = pool[src[i]] in every pool; see `copy_pages`."""
        s, d = _ids(src, "src"), _ids(dst, "dst")
        if len(s) != len(d):
            raise ValueError(f"{len(s)} source pages for {len(d)} destinations")
        if not s or not self.pools:
            return
        rc = _lib.lib().ls_copy_pages(self.table, len(self.pools), s.buffer_info()[0], d.buffer_info()[0], len(s),
                                      self.blocks, _lib.raw_stream(self.index))
        _lib.check(rc, "copy_pages")


def copy_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int], block_dim: int = 0) -> None:
    """pool[dst[i]] = pool[src[i]] for every tensor of `pools`, whose axis `block_dim` (0, or 1
    behind an axis of layers) counts the pages; any type, each page one dense run. src and dst are
    host sequences of page ids: they are read before the call returns, and a captured call
    replays with the same ids. A source may serve several destinations; a destination given
    twice, or that is a source as well, is refused."""
    if _lib.binding().copy_pages(pools, src, dst, block_dim) is None:
        PagePools(pools, block_dim).copy(src, dst)
