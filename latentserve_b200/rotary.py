"""Rotary positions of queries and keys on the sm_100a kernels -- host side.

`apply_rotary` turns any number of tokens at once (a prompt, a decode batch), in the half or the
interleaved layout, the whole head or the first part of it, fp16, bf16 or fp32;
`rotary_tables` makes the tables it reads, with the frequencies scaled for contexts longer than
the trained ones. The reference has one form, `rope_qk` (kernels/fused_elementwise.py:229-252): half
layout, whole head. `fused_elementwise.rope_append_*` are that form fused with the cache append.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from latentserve_b200 import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None) -> tuple[torch.Tensor, float]:
    """Angles per position, fp64 [rotary_dim / 2] on the CPU, and the factor on cos and sin.
    theta ** (-2 i / rotary_dim), changed by `scaling`:

        {"type": "linear", "factor": f}   every frequency divided by f
        {"type": "ntk", "factor": f}      theta multiplied by f ** (n / (n - 2)), n = rotary_dim
        {"type": "yarn", "factor": f, "original_max_pos": L, "beta_fast": 32, "beta_slow": 1,
         "attention_factor": 0.1 ln f + 1}
            frequencies that turn more than beta_fast times in L positions stay, those that
            turn less than beta_slow times are divided by f, linearly blended between
    """
    n = rotary_dim
    if n < 2 or n % 2:
        raise ValueError(f"rotary_dim must be even and positive, not {n}")
    scaling = dict(scaling or {"type": "none"})
    kind = scaling.pop("type", None)
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_max_pos", "beta_fast", "beta_slow", "attention_factor")}
    if kind not in known or any(key not in known[kind] for key in scaling):
        raise ValueError(f"unknown rotary scaling {kind!r} with {sorted(scaling)}")
    factor = float(scaling.get("factor", 1.0))
    if not factor > 0 or not theta > 0:
        raise ValueError("theta and the scaling factor must be positive")
    if kind == "ntk":
        if n <= 2:
            raise ValueError("ntk scaling needs more than two rotated channels")
        theta = theta * factor ** (n / (n - 2))
    inv = theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if kind == "linear":
        inv = inv / factor
    if kind != "yarn":
        return inv, 1.0
    if "original_max_pos" not in scaling:
        raise ValueError("yarn scaling needs original_max_pos")

    def dim_of(turns: float) -> float:
        return n * math.log(scaling["original_max_pos"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

    first = max(math.floor(dim_of(scaling.get("beta_fast", 32.0))), 0)
    last = min(math.ceil(dim_of(scaling.get("beta_slow", 1.0))), n - 1)
    ramp = ((torch.arange(n // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0, 1)
    magnitude = scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    return inv / factor * ramp + inv * (1 - ramp), float(magnitude)


def rotary_tables(rotary_dim: int, max_pos: int, theta: float = 10000.0, scaling: Optional[dict] = None,
                  device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin fp32 [max_pos, rotary_dim / 2] for `apply_rotary`. Angles are formed in 64 bits:
    in 32 a position of a million is already off by a tenth of a radian."""
    inv, magnitude = rotary_frequencies(rotary_dim, theta, scaling)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def _check(x: torch.Tensor, tokens: int, dim: int, like: torch.Tensor, what: str) -> None:
    if x.dim() != 3 or x.shape[0] != tokens or x.shape[2] != dim:
        raise ValueError(f"{what} must be [tokens, heads, head_dim]")
    if x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{what} must have the queries' type and device")
    if x.shape[2] > 1 and x.stride(2) != 1:
        raise ValueError(f"{what} needs unit-stride channels")


def _strides(x: torch.Tensor) -> tuple[int, int]:
    """Token and head stride; 0 for an axis of one, whose stride says nothing."""
    return tuple(x.stride(i) if x.shape[i] > 1 else 0 for i in (0, 1))


def apply_rotary(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                 interleaved: bool = False, inverse: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """q [tokens, q_heads, head_dim], k [tokens, k_heads, head_dim] (views of a fused projection are
    fine) rotated by positions [tokens] int64; returns (q_out, k_out), new dense tensors unless
    given. Either may be given as the input itself (in place), but must not overlap it otherwise.

    cos, sin fp32 [max_pos, r / 2] say how much of a head turns: its first r channels, in pairs
    (i, i + r / 2), or (2 i, 2 i + 1) with `interleaved`; the rest is copied. `inverse` turns the
    other way, which is also the gradient. A position outside the tables comes out as NaN."""
    got = _lib.binding().rotary(q, k, cos, sin, positions, interleaved, inverse, q_out, k_out)
    if got is not None:
        return got
    if not q.is_cuda:
        raise RuntimeError("latentserve_b200 has no CPU path: tensors must be on a CUDA device")
    if q.dtype not in _DTYPES:
        raise ValueError("queries must be fp16, bf16 or fp32")
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    tokens, _, dim = q.shape
    _check(q, tokens, dim, q, "q")
    _check(k, tokens, dim, q, "k")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be fp32 [max_pos, rotary_dim / 2]")
    rot = 2 * cos.shape[1]
    if not 0 < rot <= dim or cos.shape[0] < 1:
        raise ValueError(f"tables for {rot} rotated channels do not fit a head of {dim}")
    if cos.device != q.device or sin.device != q.device or cos.stride() != sin.stride() or (
            cos.shape[1] > 1 and cos.stride(1) != 1) or (cos.shape[0] > 1 and cos.stride(0) < cos.shape[1]):
        raise ValueError("cos and sin must share one row layout with dense entries, on the queries' device")
    if positions.dtype != torch.int64 or positions.shape != (tokens,) or positions.device != q.device or (
            tokens > 1 and positions.stride(0) != 1):
        raise ValueError("positions must be a contiguous int64 vector with one entry per token")
    outs = []
    for x, out, what in ((q, q_out, "q_out"), (k, k_out, "k_out")):
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        _check(out, tokens, dim, q, what)
        if out.shape != x.shape:
            raise ValueError(f"{what} must have its input's shape")
        if any(size > 1 and stride == 0 for size, stride in zip(out.shape, out.stride())):
            raise ValueError(f"{what} must not be broadcast")
        if x.numel() and out.data_ptr() == x.data_ptr() and _strides(out) != _strides(x):
            raise ValueError(f"{what} in place needs its input's strides")
        outs.append(out)
    q_out, k_out = outs
    if tokens == 0 or q.shape[1] + k.shape[1] == 0:
        return q_out, k_out
    rc = _lib.lib().ls_rotary(
        q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        positions.data_ptr(), tokens, q.shape[1], k.shape[1], dim, rot, _DTYPES[q.dtype], int(interleaved), int(inverse),
        cos.shape[0], cos.stride(0) if cos.shape[0] > 1 else cos.shape[1], *_strides(q), *_strides(k), *_strides(q_out),
        *_strides(k_out), _lib.raw_stream(q.device.index))
    _lib.check(rc, "apply_rotary")
    return q_out, k_out
