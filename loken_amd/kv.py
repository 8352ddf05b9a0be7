"""The paged 8-bit key / value cache of a served step, and attention over it.

Torch holds device memory and the current stream only; every computation goes through ``libloken_gfx950.so``
(``lk_kv_*`` in ``include/loken_gfx950.h``, which states the formulas and what is done with absent pages). Per step:

    plan = kv_plan(past, fresh, table, free_pages, page_tokens, plan)     # once a step
    kv_write(cache, k, v, plan.slots)                                      # per layer
    out = kv_attention(q, cache, table, plan.lens, plan.starts, max_fresh=..., max_len=...)

All of it can be recorded into a graph.
"""
from __future__ import annotations

import math

import torch

from . import lib as _lib
from .ops import _X_TYPES, _stream

PAGE_TOKENS = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
PLAN_SEQS = 8192


def _on_device(what: str, *tensors: torch.Tensor) -> None:
    """The launches go to the current device's current stream: the tensors have to be there."""
    device = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != device:
            raise ValueError(f"{what}: tensors on several devices")
    if device < 0 or device != torch._C._cuda_getDevice():
        raise ValueError(f"{what}: a tensor is not on the current device")


def _vector(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, n: int | None = None) -> None:
    if t.dtype is not dtype or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{what}: {name} is a contiguous {dtype} vector" + (f" of {n}" if n is not None else ""))


def _rows(what: str, name: str, t: torch.Tensor, heads: int | None, head_dim: int):
    """``[rows, heads, head_dim]`` with a token's values together: rows, heads, the distance between tokens."""
    if t.dim() != 3 or t.dtype not in _X_TYPES:
        raise ValueError(f"{what}: {name} is [rows, heads, {head_dim}] of f32, f16 or bf16")
    n, h, d = t.shape
    if d != head_dim or (heads is not None and h != heads):
        raise ValueError(f"{what}: {name} is [rows, {'heads' if heads is None else heads}, {head_dim}]")
    if t.is_contiguous():
        return n, h, h * d
    across, of_head, of_value = t.stride()
    if n and (of_value != 1 or (h > 1 and of_head != d)):
        raise ValueError(f"{what}: the values of a token of {name} have to stand together")
    if n <= 1:
        return n, h, h * d
    if across < h * d:
        raise ValueError(f"{what}: rows of {name} overlap")
    return n, h, across


def _table(what: str, table: torch.Tensor, seqs: int):
    """int32 ``[sequences, columns]``: columns, the distance between rows."""
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != seqs:
        raise ValueError(f"{what}: table is int32 [sequences, columns]")
    cols = table.shape[1]
    if table.is_contiguous():
        return cols, cols
    across, of_col = table.stride()
    if (cols > 1 and of_col != 1) or (seqs > 1 and across < cols):
        raise ValueError(f"{what}: table is int32 [sequences, columns], a row together")
    return cols, across if seqs > 1 else cols


class KvCacheQ8:
    """Pages of one layer's cache: codes ``k`` int8 [pages, kv_heads, page_tokens, head_dim] and ``v`` int8
    [pages, kv_heads, page_tokens / 16, head_dim, 16], scales f32 [pages, kv_heads]. Other tensors are another cache: these four are not
    assigned anew."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        if k.dim() != 4 or k.dtype != torch.int8 or v.dtype != torch.int8:
            raise ValueError("kv cache: k is int8 [pages, kv_heads, page_tokens, head_dim], v int8 [pages, kv_heads, page_tokens / 16, head_dim, 16]")
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        if self.page_tokens not in PAGE_TOKENS or self.head_dim not in HEAD_DIMS or self.pages < 1 or self.kv_heads < 1:
            raise ValueError(f"kv cache: pages of {PAGE_TOKENS} tokens, heads of {HEAD_DIMS} values")
        if tuple(v.shape) != (self.pages, self.kv_heads, self.page_tokens // 16, self.head_dim, 16):
            raise ValueError("kv cache: v is [pages, kv_heads, page_tokens / 16, head_dim, 16]")
        for s in (k_scales, v_scales):
            if s.dtype != torch.float32 or tuple(s.shape) != (self.pages, self.kv_heads):
                raise ValueError("kv cache: scales are f32 [pages, kv_heads]")
        if len({t.device for t in (k, v, k_scales, v_scales)}) != 1:
            raise ValueError("kv cache: its tensors are on several devices")
        if not all(t.is_contiguous() for t in (k, v, k_scales, v_scales)):
            raise ValueError("kv cache: its tensors are contiguous")
        self._tensors = (k, v, k_scales, v_scales)
        if (k.data_ptr() | v.data_ptr()) & 15:
            raise ValueError("kv cache: codes start on 16 bytes")

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    def _at(self):
        """Where the tensors are now: a program may have given one other memory since."""
        k, v, k_scales, v_scales = self._tensors
        return k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr()

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 16, device="cuda") -> "KvCacheQ8":
        if page_tokens not in PAGE_TOKENS:
            raise ValueError(f"kv cache: pages of {PAGE_TOKENS} tokens")
        return cls(torch.zeros((pages, kv_heads, page_tokens, head_dim), dtype=torch.int8, device=device),
                   torch.zeros((pages, kv_heads, page_tokens // 16, head_dim, 16), dtype=torch.int8, device=device),
                   torch.zeros((pages, kv_heads), dtype=torch.float32, device=device),
                   torch.zeros((pages, kv_heads), dtype=torch.float32, device=device))


class KvPlan:
    """What ``kv_plan`` writes for ``seqs`` sequences and a batch of ``rows`` rows; kept from step to step (a recorded step
    holds its addresses)."""

    def __init__(self, seqs: int, rows: int, device="cuda"):
        if seqs < 0 or rows < 0:
            raise ValueError("kv plan: sizes below zero")
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.starts = torch.zeros(seqs + 1, dtype=torch.int32, device=device)
        self.slots = torch.full((rows,), -1, dtype=torch.int64, device=device)
        self.positions = torch.zeros(rows, dtype=torch.int32, device=device)
        self.taken = torch.zeros(1, dtype=torch.int32, device=device)


def kv_plan(past: torch.Tensor, fresh: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page_tokens: int, plan: KvPlan,
            taken: torch.Tensor | None = None) -> KvPlan:
    """Pages for the tokens that each sequence brings (into ``table`` [seqs, columns], in place) and, in ``plan``, lengths, first
    rows, the slot and position of every row, and how many pages of ``free_pages`` are gone by then; ``taken``: how many were before.
    None of what it reads is the plan's own: the next step's ``past`` is a copy of ``plan.lens``, or two plans are used in turn."""
    seqs = past.numel()
    _vector("kv_plan", "past", past, torch.int32)
    _vector("kv_plan", "fresh", fresh, torch.int32, seqs)
    _vector("kv_plan", "free_pages", free_pages, torch.int32)
    cols, across = _table("kv_plan", table, seqs)
    if page_tokens not in PAGE_TOKENS:
        raise ValueError(f"kv_plan: pages of {PAGE_TOKENS} tokens")
    if plan.lens.numel() != seqs:
        raise ValueError("kv_plan: the plan is for another number of sequences")
    if taken is not None:
        _vector("kv_plan", "taken", taken, torch.int32, 1)
        if taken.data_ptr() == plan.taken.data_ptr():
            raise ValueError("kv_plan: taken is the plan's own")
    if past.data_ptr() == plan.lens.data_ptr() and seqs:
        raise ValueError("kv_plan: past is the plan's own")
    _on_device("kv_plan", past, fresh, table, free_pages, plan.slots, *(() if taken is None else (taken,)))
    _lib.check("lk_kv_plan", _lib.load().lk_kv_plan(
        past.data_ptr(), fresh.data_ptr(), seqs, page_tokens, free_pages.data_ptr(), free_pages.numel(),
        None if taken is None else taken.data_ptr(), table.data_ptr(), across, cols, plan.lens.data_ptr(),
        plan.starts.data_ptr(), plan.slots.data_ptr(), plan.positions.data_ptr(), plan.slots.numel(), plan.taken.data_ptr(), _stream()))
    return plan


def kv_write(cache: KvCacheQ8, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """New keys and values ``[tokens, kv_heads, head_dim]`` (f32, f16 or bf16; rows may be parts of wider ones) into the cache."""
    tokens, _, ks = _rows("kv_write", "k", k, cache.kv_heads, cache.head_dim)
    of_v, _, vs = _rows("kv_write", "v", v, cache.kv_heads, cache.head_dim)
    if k.dtype is not v.dtype or of_v != tokens:
        raise ValueError("kv_write: keys and values are of one type and shape")
    _vector("kv_write", "slots", slots, torch.int64, tokens)
    _on_device("kv_write", k, v, slots, cache.k)
    _lib.check("lk_kv_write_q8", _lib.load().lk_kv_write_q8(
        k.data_ptr(), v.data_ptr(), _X_TYPES[k.dtype], ks, vs, slots.data_ptr(), tokens, cache.kv_heads, cache.head_dim,
        cache.page_tokens, cache.pages, *cache._at(), _stream()))


def kv_read(cache: KvCacheQ8, slots: torch.Tensor, dtype: torch.dtype = torch.float32):
    """Rows of the cache as values: keys and values ``[tokens, kv_heads, head_dim]``; zeros where a slot is absent."""
    if dtype not in _X_TYPES:
        raise ValueError("kv_read: f32, f16 or bf16")
    _vector("kv_read", "slots", slots, torch.int64)
    _on_device("kv_read", slots, cache.k)
    k = torch.empty((slots.numel(), cache.kv_heads, cache.head_dim), dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    _lib.check("lk_kv_read_q8", _lib.load().lk_kv_read_q8(
        slots.data_ptr(), slots.numel(), cache.kv_heads, cache.head_dim, cache.page_tokens, cache.pages, *cache._at(), k.data_ptr(),
        v.data_ptr(), _X_TYPES[dtype], _stream()))
    return k, v


def kv_attention(q: torch.Tensor, cache: KvCacheQ8, table: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor, *, max_fresh: int,
                 max_len: int, scale: float | None = None, window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the rows ``q`` ``[rows, heads, head_dim]`` over the cache, causal, each sequence's rows being its last positions;
    ``window`` > 0: that many positions, the row's own among them. Rows behind the last sequence stay as they are in ``out``
    (without one: zeros). ``max_fresh``, ``max_len``: the most rows and tokens of a sequence as far as the caller knows them."""
    seqs = lens.numel()
    rows, heads, stride = _rows("kv_attention", "q", q, None, cache.head_dim)
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("kv_attention: the heads of q are a multiple of the cache's")
    _vector("kv_attention", "lens", lens, torch.int32)
    _vector("kv_attention", "starts", starts, torch.int32, seqs + 1)
    cols, across = _table("kv_attention", table, seqs)
    if max_fresh < 0 or max_len < 0 or window < 0:
        raise ValueError("kv_attention: sizes below zero")
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("kv_attention: the scale is a number above zero")
    if out is None:
        out = torch.zeros((rows, heads, cache.head_dim), dtype=q.dtype, device=q.device)
    of_out, _, out_stride = _rows("kv_attention", "out", out, heads, cache.head_dim)
    if out.dtype is not q.dtype or of_out != rows:
        raise ValueError("kv_attention: out has the type and shape of q")
    _on_device("kv_attention", q, out, table, lens, starts, cache.k)
    _lib.check("lk_kv_attention_q8", _lib.load().lk_kv_attention_q8(
        q.data_ptr(), _X_TYPES[q.dtype], stride, out.data_ptr(), out_stride, *cache._at(), cache.pages, cache.page_tokens, table.data_ptr(),
        across, cols, lens.data_ptr(), starts.data_ptr(), seqs, rows, min(max_fresh, 0x7FFFFFFF),
        min(max_len, 0x7FFFFFFF), heads, cache.kv_heads, cache.head_dim, scale, min(window, 0x7FFFFFFF), _stream()))
    return out
