"""The next token of each sequence from its logits (``lk_sample``; the header states the rules and their order)."""
from __future__ import annotations

import torch

from . import lib as _lib
from .kv import _on_device, _vector
from .ops import _X_TYPES, _stream

MAX_VOCAB = 1 << 20


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None):
    """``logits`` [rows, vocab] (f32, f16 or bf16; rows may be parts of wider ones), one uniform number in [0, 1) and one
    temperature a row; ``top_k`` int32, ``top_p``, ``min_p`` f32 per row -> (tokens int32, probabilities f32), [rows] each."""
    if logits.dtype not in _X_TYPES or logits.dim() != 2 or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("sample: logits are [rows, vocab] of f32, f16 or bf16")
    rows, vocab = logits.shape
    if vocab > MAX_VOCAB:
        raise ValueError(f"sample: up to {MAX_VOCAB} words")
    stride = logits.stride(0) if rows > 1 else vocab
    if stride < vocab:
        raise ValueError("sample: rows of logits overlap")
    given = [("uniform", uniform, torch.float32), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
             ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)]
    given = [g for g in given if g[1] is not None]
    for name, t, dtype in given:
        _vector("sample", name, t, dtype, rows)
    _on_device("sample", logits, *(t for _, t, _ in given))
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    probs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    at = [None if t is None else t.data_ptr() for t in (top_k, top_p, min_p)]
    _lib.check("lk_sample", _lib.load().lk_sample(
        logits.data_ptr(), _X_TYPES[logits.dtype], stride, rows, vocab, uniform.data_ptr(), temperature.data_ptr(), *at,
        tokens.data_ptr(), probs.data_ptr(), _stream()))
    return tokens, probs
