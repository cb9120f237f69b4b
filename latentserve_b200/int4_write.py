"""Writing into a KV cache held in 4 bits, and reading it back -- host side.

One pool per layer, `kv_pool` uint8 [num_blocks, H, record]: everything a page (16 tokens)
holds of one KV head (head_dim 128) is one record of `record_bytes(group)` bytes, K and V
codes and their scales (csrc/int4_page.cuh has the order). A value stands for
`lo + step * code`, code 0..15, with fp16 lo and step per (token, head, group of channels):
`lo` the group's minimum, `step` fp16((max - lo) / 15). Groups of 32, 64 or 128 channels
cost 5, 4.5 or 4.25 bits a value.

Nothing of a token is shared with another token, so a page can be partly filled, rewound,
forked and moved as plain bytes, and there is no full-precision residual beside the pool.
The reference has no 4-bit cache; its INT8 one is cache/int8_paged_cache.py:143-1028.
"""

from __future__ import annotations

from typing import Optional

import torch

from latentserve_b200 import _lib

GROUPS = {32: 4, 64: 2, 128: 1}            # channels a scale covers -> scales per row


def record_bytes(group: int) -> int:
    """Bytes one page takes per KV head."""
    if group not in GROUPS:
        raise ValueError(f"group must be 32, 64 or 128 channels, not {group}")
    return 2048 + 128 * GROUPS[group]


_GROUPS_OF_RECORD = {record_bytes(g): n for g, n in GROUPS.items()}


def pool_ok(kv_pool: torch.Tensor) -> bool:
    """A pool of page records whose strides keep rows 16-byte aligned and apart. (The address is
    checked by every call.)"""
    return (kv_pool.dim() == 3 and kv_pool.dtype == torch.uint8 and kv_pool.shape[2] in _GROUPS_OF_RECORD
            and kv_pool.shape[0] > 0 and kv_pool.shape[1] > 0 and kv_pool.stride(2) == 1
            and all(s % 16 == 0 and s >= kv_pool.shape[2] for s in kv_pool.stride()[:2]))


def groups_of(kv_pool: torch.Tensor) -> int:
    """Scales per row (4, 2 or 1), from the record's size."""
    return _GROUPS_OF_RECORD[kv_pool.shape[2]]


def check_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, batch: int, device) -> torch.Tensor:
    """Block tables [>= batch, pages] and lengths [>= batch], int32; the tables' rows are
    made dense (a copy) where they are not."""
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block tables and sequence lengths must be int32")
    if (block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.shape[0] < batch
            or seq_lens.shape[0] < batch or block_tables.shape[1] < 1):
        raise ValueError("block tables must be [batch, pages] and sequence lengths [batch]")
    if seq_lens.shape[0] > 1 and seq_lens.stride(0) != 1:
        raise ValueError("sequence lengths must be contiguous")
    if block_tables.device != device or seq_lens.device != device:
        raise ValueError("block tables and sequence lengths must be on the queries' or rows' device")
    return block_tables if block_tables.is_contiguous() else block_tables.contiguous()


def _vector(t: torch.Tensor, batch: int, device, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < batch or t.device != device or (
            t.shape[0] > 1 and t.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous int32 vector with one entry per sequence, on the rows' device")
    return t


def _strides(t: torch.Tensor) -> list[int]:
    """Batch, head and token stride; 0 for an axis of one, whose stride says nothing."""
    return [st if n > 1 else 0 for n, st in zip(t.shape[:3], t.stride()[:3])]


def _check_rows(k: torch.Tensor, v: torch.Tensor, kv_pool: torch.Tensor) -> None:
    if not k.is_cuda:
        raise RuntimeError("latentserve_b200 has no CPU path: tensors must be on a CUDA device")
    if not pool_ok(kv_pool):
        raise ValueError("kv_pool must be uint8 [num_blocks, H, record_bytes(group)] with 16-byte aligned rows")
    if v.device != k.device or kv_pool.device != k.device:
        raise ValueError("rows and pool must be on one device")
    for t in (k, v):
        if t.dtype != torch.float16 or t.dim() != 4 or t.shape != k.shape or t.shape[3] != 128:
            raise ValueError("K and V rows must be fp16 [B, H, n, 128] of one shape")
        if t.stride(3) != 1 or any(s % 8 for s in _strides(t)):
            raise ValueError("K and V rows must have unit-stride channels and 16-byte alignment")
    if k.shape[1] != kv_pool.shape[1]:
        raise ValueError(f"the rows have {k.shape[1]} KV heads, the pool {kv_pool.shape[1]}")


def write(k: torch.Tensor, v: torch.Tensor, kv_pool: torch.Tensor, block_tables: torch.Tensor,
          seq_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None) -> None:
    """Quantise k, v [B, H, n, 128] fp16 (any strides with unit-stride channels) into the pages
    of the batch's block tables, one launch. `seq_lens` [B] already count the new tokens: rows
    0 .. m-1 of sequence b go to positions seq_lens[b] - m .. seq_lens[b] - 1, m = n or, with
    `new_lens` [B] int32, min(new_lens[b], n); rows past m are not read. Positions below zero,
    past the table or in a block outside the pool are dropped. Bytes of other tokens stay as
    they are. Sequences of one call must not write the same token of the same block (pages that are
    shared are full): which of the rows' bytes it then holds is not defined.

    NaN is stored as 0 and an infinity as the largest fp16 of its sign."""
    if _lib.binding().write(k, v, kv_pool, block_tables, seq_lens, new_lens) is not None:
        return
    _check_rows(k, v, kv_pool)
    b, h, n, d = k.shape
    block_tables = check_tables(block_tables, seq_lens, b, k.device)
    if new_lens is not None:
        _vector(new_lens, b, k.device, "new_lens")
    if b == 0 or n == 0:
        return
    sp = kv_pool.stride()
    rc = _lib.lib().ls_int4_write(
        k.data_ptr(), v.data_ptr(), kv_pool.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
        _lib.ptr(new_lens), b, h, n, groups_of(kv_pool), d, 16, block_tables.shape[1], kv_pool.shape[0],
        *_strides(k), *_strides(v), sp[0], sp[1], _lib.raw_stream(k.device.index))
    _lib.check(rc, "int4 write")


def read(kv_pool: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, length: int,
         start: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V as the cache holds them, fp16 [B, H, length, 128] each: positions
    start[b] .. start[b] + length - 1 (`start` [B] int32, not negative; zeros if not given).
    Rows at or past seq_lens[b], or of a block outside the pool, are zeros. For what attends a
    cached prefix densely: a prompt's next chunk, a check."""
    got = _lib.binding().read(kv_pool, block_tables, seq_lens, length, start)
    if got is not None:
        return got
    if not kv_pool.is_cuda:
        raise RuntimeError("latentserve_b200 has no CPU path: tensors must be on a CUDA device")
    if length < 0:
        raise ValueError(f"cannot read {length} positions")
    if not pool_ok(kv_pool):
        raise ValueError("kv_pool must be uint8 [num_blocks, H, record_bytes(group)] with 16-byte aligned rows")
    b, h, dev = seq_lens.shape[0] if seq_lens.dim() else 0, kv_pool.shape[1], kv_pool.device
    block_tables = check_tables(block_tables, seq_lens, b, dev)
    if start is not None:
        _vector(start, b, dev, "start")
    k = torch.empty(b, h, length, 128, dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    rows, sp = (h * length * 128, length * 128, 128), kv_pool.stride()
    rc = _lib.lib().ls_int4_read(
        kv_pool.data_ptr(), k.data_ptr(), v.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
        _lib.ptr(start), b, h, length, groups_of(kv_pool), 128, 16, block_tables.shape[1], kv_pool.shape[0],
        *rows, *rows, sp[0], sp[1], _lib.raw_stream(dev.index))
    _lib.check(rc, "int4 read")
    return k, v


def rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                q_out: torch.Tensor, kv_pool: torch.Tensor, q_heads: int) -> None:
    """One decode token per sequence from the fused projection row qkv [B, (q_heads + 2 H) * 128]
    (q, k, v head order): rotated q into `q_out` [B, q_heads * 128], rotated k and v quantised
    into the page of flat slot slots[b]. cos, sin [max_pos, 128] fp16, halves duplicated;
    positions, slots [B] int64. The rotation rounds as `fused_elementwise.rope_append_fp16`'s.
    A sequence whose position lies outside the tables or whose slot lies outside the pool gets nothing."""
    if not qkv.is_cuda:
        raise RuntimeError("latentserve_b200 has no CPU path: tensors must be on a CUDA device")
    if not pool_ok(kv_pool):
        raise ValueError("kv_pool must be uint8 [num_blocks, H, record_bytes(group)] with 16-byte aligned rows")
    b, heads = qkv.shape[0], kv_pool.shape[1]
    if qkv.dim() != 2 or qkv.shape[1] != (q_heads + 2 * heads) * 128 or q_out.shape != (b, q_heads * 128):
        raise ValueError("qkv must be [B, (q_heads + 2 kv_heads) * 128] and q_out [B, q_heads * 128]")
    if any(t.dtype != torch.float16 or t.stride(-1) != 1 for t in (qkv, cos, sin, q_out)):
        raise ValueError("qkv, q_out, cos and sin must be fp16 with unit-stride channels")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != 128 or cos.stride(0) != sin.stride(0):
        raise ValueError("cos and sin must be [max_pos, 128] tables of one layout")
    if any(t.dtype != torch.int64 or t.dim() != 1 or t.shape[0] < b or (t.shape[0] > 1 and t.stride(0) != 1)
           for t in (positions, slots)):
        raise ValueError("positions and slots must be contiguous int64 vectors with one entry per sequence")
    if any(t.device != qkv.device for t in (cos, sin, positions, slots, q_out, kv_pool)):
        raise ValueError("all tensors must be on one device")
    if b == 0:
        return
    rc = _lib.lib().ls_rope_append_int4(
        qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), slots.data_ptr(), q_out.data_ptr(),
        kv_pool.data_ptr(), b, q_heads, heads, groups_of(kv_pool), 128, 16, cos.shape[0], kv_pool.shape[0],
        qkv.stride(0), cos.stride(0), q_out.stride(0), kv_pool.stride(0), kv_pool.stride(1),
        _lib.raw_stream(qkv.device.index))
    _lib.check(rc, "int4 rope_append")
