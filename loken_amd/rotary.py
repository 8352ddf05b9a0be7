"""Norms of the query and key heads and their rotation in one pass (``lk_qk_norm_rope`` in ``include/loken_gfx950.h``, which states the
formulas), and the same with keys and values going straight into the 4-bit cache. All of it can be recorded into a graph.
"""
from __future__ import annotations

import math

import torch

from . import lib as _lib
from .kv import HEAD_DIMS, KvCacheMxfp4, _on_device, _rows, _vector
from .ops import _X_TYPES, _stream

MAX_AXES = 4


class Rotary:
    """A model's rotation: ``frequencies`` f32 [pairs], radians a position, scaled as the model wants them; ``axis`` uint8 [pairs], which
    run of the positions turns a pair (time, height, width); pairs of ``neighbours`` (2 i, 2 i + 1) instead of (i, i + pairs); ``factor`` on
    what is turned. Other tensors are another rotation: these two are not assigned anew."""

    def __init__(self, frequencies: torch.Tensor, axis: torch.Tensor | None = None, neighbours: bool = False, factor: float = 1.0):
        _vector("rotary", "frequencies", frequencies, torch.float32)
        if frequencies.numel() % 4 or frequencies.numel() > max(HEAD_DIMS) // 2:
            raise ValueError(f"rotary: a multiple of 4 pairs, up to {max(HEAD_DIMS) // 2}")
        if axis is not None:
            _vector("rotary", "axis", axis, torch.uint8, frequencies.numel())
            if axis.device != frequencies.device:
                raise ValueError("rotary: its tensors are on several devices")
        if not math.isfinite(factor):
            raise ValueError("rotary: the factor is a number")
        self._tensors, self.neighbours, self.factor = (frequencies, axis), int(bool(neighbours)), float(factor)

    frequencies = property(lambda self: self._tensors[0])
    axis = property(lambda self: self._tensors[1])


def _arguments(what, q, k, positions, rotary, q_weight, k_weight, eps):
    """Head dimension and sizes, what is checked of both calls' arguments, and the arguments that they share."""
    if q.dim() != 3 or q.shape[2] not in HEAD_DIMS:
        raise ValueError(f"{what}: heads of {HEAD_DIMS} values")
    dim = q.shape[2]
    rows, heads, qs = _rows(what, "q", q, None, dim)
    of_k, kv_heads, ks = _rows(what, "k", k, None, dim)
    if of_k != rows or k.dtype is not q.dtype or heads == 0 or kv_heads == 0:
        raise ValueError(f"{what}: queries and keys are of one type and number of rows")
    frequencies, axis = rotary._tensors
    pairs = frequencies.numel()
    if 2 * pairs > dim:
        raise ValueError(f"{what}: more pairs than a head has")
    shape = positions.shape
    axes = 1 if len(shape) == 1 else shape[0] if len(shape) == 2 else 0
    if positions.dtype is not torch.int32 or axes == 0 or shape[-1] != rows:
        raise ValueError(f"{what}: positions are int32 [rows] or [axes, rows]")
    if axes > 1 and axis is None:
        raise ValueError(f"{what}: positions of several axes go with a rotation whose axis says which of them turns a pair")
    across = rows
    if not positions.is_contiguous():
        if rows > 1 and positions.stride(-1) != 1:
            raise ValueError(f"{what}: an axis of positions stands together")
        across = positions.stride(0) if axes > 1 else rows
    if axes > MAX_AXES or across < rows:
        raise ValueError(f"{what}: up to {MAX_AXES} axes of positions, which do not overlap")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"{what}: eps is a number from zero on")
    on = [q, k, positions, frequencies]
    qw = kw = of_axis = None
    if q_weight is not None:
        _vector(what, "q_weight", q_weight, torch.float32, dim)
        qw = q_weight.data_ptr()
        on.append(q_weight)
    if k_weight is not None:
        _vector(what, "k_weight", k_weight, torch.float32, dim)
        kw = k_weight.data_ptr()
        on.append(k_weight)
    if axis is not None:
        of_axis = axis.data_ptr()
        on.append(axis)
    tail = (qw, kw, eps, positions.data_ptr(), across, axes, frequencies.data_ptr(), of_axis, pairs, rotary.neighbours, rotary.factor)
    return dim, rows, heads, kv_heads, qs, ks, on, tail


def _output(what, name, out, like, rows, heads, dim):
    if out is None:
        return like.new_empty((rows, heads, dim)), heads * dim
    of_out, _, stride = _rows(what, name, out, heads, dim)
    if out.dtype is not like.dtype or of_out != rows:
        raise ValueError(f"{what}: {name} has the type and shape of {name[0]}")
    return out, stride


def rotate(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, *, q_weight: torch.Tensor | None = None,
           k_weight: torch.Tensor | None = None, eps: float = 1e-6, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """``q`` [rows, heads, head_dim] and ``k`` [rows, kv_heads, head_dim] (f32, f16 or bf16; rows may be parts of wider ones), normed head by
    head where there is a weight (f32 [head_dim]) and turned by ``positions`` (int32 [rows], or [axes, rows] for a rotation with ``axis``); into ``q_out`` and ``k_out``
    (new ones without; ``q`` and ``k`` themselves may be given)."""
    dim, rows, heads, kv_heads, qs, ks, on, tail = _arguments("rotate", q, k, positions, rotary, q_weight, k_weight, eps)
    q_out, qo = _output("rotate", "q_out", q_out, q, rows, heads, dim)
    k_out, ko = _output("rotate", "k_out", k_out, k, rows, kv_heads, dim)
    _on_device("rotate", *on, q_out, k_out)
    _lib.check("lk_qk_norm_rope", _lib.load().lk_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), _X_TYPES[q.dtype], qs, ks, q_out.data_ptr(), k_out.data_ptr(), qo, ko, rows, heads, kv_heads, dim, *tail,
        _stream()))
    return q_out, k_out


def rotate_into(cache: KvCacheMxfp4, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                rotary: Rotary, *, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """``rotate`` whose keys go into ``cache`` at ``slots`` (int64 [rows], as ``kv_plan`` gives them), and the values ``v`` with them; returns
    the queries."""
    if not isinstance(cache, KvCacheMxfp4):
        raise ValueError("rotate_into: a 4-bit cache (for another: rotate, then kv_write)")
    dim, rows, heads, kv_heads, qs, ks, on, tail = _arguments("rotate_into", q, k, positions, rotary, q_weight, k_weight, eps)
    if dim != cache.head_dim or kv_heads != cache.kv_heads:
        raise ValueError("rotate_into: heads of the cache")
    of_v, _, vs = _rows("rotate_into", "v", v, kv_heads, dim)
    if v.dtype is not q.dtype or of_v != rows:
        raise ValueError("rotate_into: queries, keys and values are of one type and number of rows")
    _vector("rotate_into", "slots", slots, torch.int64, rows)
    q_out, qo = _output("rotate_into", "q_out", q_out, q, rows, heads, dim)
    _on_device("rotate_into", *on, v, slots, q_out, cache.k)
    _lib.check("lk_qk_norm_rope_kv_mxfp4", _lib.load().lk_qk_norm_rope_kv_mxfp4(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _X_TYPES[q.dtype], qs, ks, vs, q_out.data_ptr(), qo, slots.data_ptr(), rows, heads, kv_heads,
        dim, *tail, cache.page_tokens, cache.pages, *cache._at(), _stream()))
    return q_out
