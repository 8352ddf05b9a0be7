"""The next token of each sequence from its logits (``lk_sample``), and drafted tokens against the target's distribution (``lk_verify``);
the header states the rules and their order."""
from __future__ import annotations

import torch

from . import lib as _lib
from .kv import _on_device, _vector
from .ops import _X_TYPES, _stream

MAX_VOCAB = 1 << 20


def _words(what: str, name: str, t: torch.Tensor) -> int:
    """``[rows, vocab]`` with a row's words together: the distance between rows."""
    if t.dtype not in _X_TYPES or t.dim() != 2 or t.shape[1] < 1 or (t.numel() and t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what}: {name} are [rows, vocab] of f32, f16 or bf16")
    rows, vocab = t.shape
    if vocab > MAX_VOCAB:
        raise ValueError(f"{what}: up to {MAX_VOCAB} words")
    stride = t.stride(0) if rows > 1 else vocab
    if stride < vocab:
        raise ValueError(f"{what}: rows of {name} overlap")
    return stride


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None):
    """``logits`` [rows, vocab] (f32, f16 or bf16; rows may be parts of wider ones), one uniform number in [0, 1) and one
    temperature a row; ``top_k`` int32, ``top_p``, ``min_p`` f32 per row -> (tokens int32, probabilities f32), [rows] each."""
    stride = _words("sample", "logits", logits)
    rows, vocab = logits.shape
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


def verify(logits: torch.Tensor, drafted: torch.Tensor, starts: torch.Tensor, uniform: torch.Tensor, draw: torch.Tensor, temperature: torch.Tensor,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           draft: torch.Tensor | None = None):
    """``logits`` [rows, vocab], ``starts`` int32 [sequences + 1]: each sequence's rows are its drafted tokens and one more; ``drafted`` int32
    [rows], ``draft`` [rows, vocab] the distributions that they came from (f32, f16 or bf16; none: for certain), ``uniform`` [rows] and ``draw``
    [sequences] numbers in [0, 1), rules by row as ``sample`` has them -> (tokens int32 [rows]: accepted drafts, the next token, -1; accepted
    int32 [sequences]; the tokens' probabilities f32 [rows])."""
    stride = _words("verify", "logits", logits)
    rows, vocab = logits.shape
    seqs = starts.numel() - 1
    if seqs < 0:
        raise ValueError("verify: starts has one entry more than there are sequences")
    _vector("verify", "starts", starts, torch.int32)
    given = [("drafted", drafted, torch.int32, rows), ("uniform", uniform, torch.float32, rows), ("draw", draw, torch.float32, seqs),
             ("temperature", temperature, torch.float32, rows), ("top_k", top_k, torch.int32, rows), ("top_p", top_p, torch.float32, rows),
             ("min_p", min_p, torch.float32, rows)]
    given = [g for g in given if g[1] is not None]
    for name, t, dtype, n in given:
        _vector("verify", name, t, dtype, n)
    draft_stride, more = 0, []
    if draft is not None:
        draft_stride, more = _words("verify", "draft", draft), [draft]
        if draft.shape != logits.shape:
            raise ValueError("verify: draft has the shape of logits")
    _on_device("verify", logits, starts, *(g[1] for g in given), *more)
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    accepted = torch.empty(seqs, dtype=torch.int32, device=logits.device)
    probs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    if seqs == 0:
        tokens.fill_(-1)
        probs.zero_()
    elif rows == 0:
        accepted.zero_()
    at = [None if t is None else t.data_ptr() for t in (top_k, top_p, min_p)]
    _lib.check("lk_verify", _lib.load().lk_verify(
        logits.data_ptr(), _X_TYPES[logits.dtype], stride, rows, vocab, drafted.data_ptr(), starts.data_ptr(), seqs,
        None if draft is None else draft.data_ptr(), 0 if draft is None else _X_TYPES[draft.dtype], draft_stride, uniform.data_ptr(),
        draw.data_ptr(), temperature.data_ptr(), *at, tokens.data_ptr(), accepted.data_ptr(), probs.data_ptr(), _stream()))
    return tokens, accepted, probs
