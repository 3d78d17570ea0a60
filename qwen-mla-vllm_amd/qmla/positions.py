"""Rotary positions of query and key heads on their own (libqmla.so, `qmla_rotary`): half and interleaved
pairs, any part of the head, tables scaled for long contexts.

`mla_decode_prep` rotates inside its fused launch, half layout and bf16 arithmetic as the reference does
(qwen_mla/qwen3_5_mla.py:341-354). This is the operator beside it for what does not pass through it: a tree's
drafted tokens, whose positions repeat, prefill chunks, models with interleaved pairs. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16}


def rotary_table(rot: int, max_pos: int, theta: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                 original_max_pos: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 low_freq_factor: float = 1.0, high_freq_factor: float = 4.0, mscale: float | None = None,
                 device=None) -> torch.Tensor:
    """The fp32 table [max_pos, rot] = cos | sin that `rotary` reads, angles in float64. Built once per model.

    Pair i turns by theta^(-2i/rot) a position. `scaling` stretches that to a context `factor` times the
    trained one:
      "linear"  positions interpolated: every frequency / factor
      "ntk"     the base grows: theta * factor^(rot / (rot - 2)), so the fastest pair keeps its frequency and
                the slowest is interpolated (rot > 2)
      "yarn"    pairs that turn more than beta_fast times over original_max_pos keep their frequency, those
                below beta_slow turns are interpolated, a linear ramp over the pair index between; cos and sin
                times `mscale`, by default 0.1 ln(factor) + 1 (YaRN, arXiv:2309.00071)
      "llama3"  the same with the ramp over turns: kept above high_freq_factor turns, interpolated below
                low_freq_factor
    """
    if rot <= 0 or rot % 2 or max_pos <= 0:
        raise ValueError("rotary_table: rot must be even and positive, max_pos positive")
    if not theta > 1.0:
        raise ValueError("rotary_table: theta must be above 1")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    inv = theta ** (-i / rot)
    scale = 1.0
    if scaling is not None:
        if not factor >= 1.0:
            raise ValueError("rotary_table: factor must be at least 1")
        if scaling in ("yarn", "llama3") and not (original_max_pos and original_max_pos > 0):
            raise ValueError(f"rotary_table: {scaling} needs original_max_pos")
        if scaling == "linear":
            inv = inv / factor
        elif scaling == "ntk":
            if rot <= 2:
                raise ValueError("rotary_table: ntk needs more than one pair")
            inv = (theta * factor ** (rot / (rot - 2))) ** (-i / rot)
        elif scaling == "yarn":
            def pair_of(turns):   # the pair index that turns so often over the trained context
                return rot * math.log(original_max_pos / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rot - 1)
            ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            inv = inv * (1 - ramp) + inv / factor * ramp
            scale = 0.1 * math.log(factor) + 1.0
        elif scaling == "llama3":
            if not high_freq_factor > low_freq_factor:
                raise ValueError("rotary_table: high_freq_factor must exceed low_freq_factor")
            turns = original_max_pos * inv / (2 * math.pi)
            keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
            inv = inv * keep + inv / factor * (1 - keep)
        else:
            raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    if mscale is not None:
        scale = mscale
    angle = torch.outer(torch.arange(max_pos, dtype=torch.float64), inv)
    return (torch.cat([angle.cos(), angle.sin()], dim=-1) * scale).to(device=device, dtype=torch.float32)


def _span(t: torch.Tensor):
    """[first, last) byte address of a tensor's elements."""
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _check_out(name: str, x: torch.Tensor, out: torch.Tensor) -> None:
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError(f"rotary: {name}_out must have {name}'s shape and dtype")
    if out.numel() and out.stride(-1) != 1:
        raise ValueError(f"rotary: {name}_out's last dimension must be contiguous")
    extent = 1
    for st, size in sorted((st, size) for st, size in zip(out.stride(), out.shape) if size > 1):
        if st < extent:
            raise ValueError(f"rotary: elements of {name}_out lie on one another")
        extent += (size - 1) * st
    if out.numel() == 0 or (out.data_ptr() == x.data_ptr() and out.stride() == x.stride()):
        return
    (a0, a1), (b0, b1) = _span(x), _span(out)
    if a0 < b1 and b0 < a1:
        raise ValueError(f"rotary: {name}_out overlaps {name} without being it")


def rotary(positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None, cos_sin: torch.Tensor, *,
           layout: str = "half", offset: int = 0, inverse: bool = False, q_out: torch.Tensor | None = None,
           k_out: torch.Tensor | None = None):
    """Rotate columns [offset, offset + rot) of q [n, heads, dim] and k [n, key heads, dim] (or None) by the
    angles of positions [n], rot = cos_sin.shape[1] (see `rotary_table`); returns (q_out, k_out).

    layout "half" pairs columns (i, i + rot/2) of that part, "interleaved" (2i, 2i + 1). inverse turns back. bf16,
    fp16 or fp32 heads with any token and head strides, fp32 arithmetic rounded once. The other columns are
    copied; with q_out=q (k_out=k) the heads are rotated in place. A position outside the table gives NaN in the
    rotated columns. q_out and k_out must not overlap other inputs or each other."""
    if layout not in ("half", "interleaved"):
        raise ValueError(f"rotary: layout must be 'half' or 'interleaved', got {layout!r}")
    if positions.dim() != 1 or positions.dtype not in (torch.int64, torch.int32):
        raise TypeError("rotary: positions must be a 1-D int64 or int32 tensor")
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.stride(-1) != 1 or cos_sin.shape[0] == 0:
        raise TypeError("rotary: cos_sin must be an fp32 [max_pos, rot] table with contiguous rows")
    rot, n = cos_sin.shape[1], positions.shape[0]
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if t.dim() != 3 or t.shape[0] != n or t.dtype not in _DT:
            raise TypeError(f"rotary: {name} must be [{n}, heads, dim] in bf16, fp16 or fp32")
        if t.numel() and t.stride(-1) != 1:
            raise ValueError(f"rotary: {name}'s last dimension must be contiguous")
        if offset < 0 or rot % 2 or offset + rot > t.shape[-1]:
            raise ValueError(f"rotary: columns [{offset}, {offset + rot}) are not an even part of {name}'s {t.shape[-1]}")
    if k is not None and (k.dtype != q.dtype or k.shape[-1] != q.shape[-1]):
        raise TypeError("rotary: q and k must share dtype and head dim")
    if k is None and k_out is not None:
        raise ValueError("rotary: k_out without k")
    for name, t, t_out in (("q", q, q_out), ("k", k, k_out)):
        if t_out is not None:
            _check_out(name, t, t_out)
    _lib.same_device("rotary", "positions", positions, "q", q, "k", k, "cos_sin", cos_sin, "q_out", q_out,
                     "k_out", k_out)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    keep = ()
    if positions.dtype != torch.int64:
        positions = positions.to(torch.int64)
        keep = (positions,)
    p = _lib.RotaryParams()
    p.q, (p.q_token_stride, p.q_head_stride, _) = q.data_ptr(), q.stride()
    p.q_out, (p.q_out_token_stride, p.q_out_head_stride, _) = q_out.data_ptr(), q_out.stride()
    if k is not None:
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        p.k, (p.k_token_stride, p.k_head_stride, _) = k.data_ptr(), k.stride()
        p.k_out, (p.k_out_token_stride, p.k_out_head_stride, _) = k_out.data_ptr(), k_out.stride()
        p.k_heads = k.shape[1]
    p.positions, p.pos_stride = positions.data_ptr(), positions.stride(0)
    p.cos_sin, p.max_pos, p.cos_sin_stride = cos_sin.data_ptr(), cos_sin.shape[0], cos_sin.stride(0)
    p.n, p.q_heads, p.head_dim = q.shape
    p.offset, p.rot = offset, rot
    p.interleaved, p.inverse, p.dtype = layout == "interleaved", inverse, _DT[q.dtype]
    _lib.check("qmla_rotary", _lib.lib().qmla_rotary(ctypes.byref(p), _lib.stream()))
    if keep:
        _lib.keep_alive(keep)
    return q_out, k_out
