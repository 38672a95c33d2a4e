"""Scores of tokens over torch tensors (include/faie2fn.h, fn_logprobs): the log probability and rank of a given token, the
entropy and the best alternatives of every row of logits, in one pass. The reference answers with the argmax alone
(k_argmax, engine/faie2fn.cu:1910-1935).

    fn = FN()
    r = token_logprobs(fn, logits, tokens, top=5)    # logits [rows][vocab] fp32 or bf16, tokens int32 [rows]
    r.logprob, r.rank, r.entropy                     # [rows]; r.top_ids, r.top_logprobs [rows][top]

Runs on the current stream and returns at once.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from kv4 import _TYPE, _ints, _stream

MAX_TOP = 32


class Logprobs(NamedTuple):
    """Device tensors, fp32 or int32. logprob, rank: None if no tokens were given."""
    logprob: torch.Tensor | None
    rank: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def _make(rows, top, dev, tokens):
    # one allocation: an empty tensor costs the host as much as two views of one
    f = torch.empty(rows * (3 + 2 * top), dtype=torch.float32, device=dev)
    i = f.view(torch.int32)
    one, wide, at = (rows,), (rows, top), 3 * rows
    return Logprobs(f.as_strided(one, (1,), 0) if tokens else None, i.as_strided(one, (1,), rows) if tokens else None,
                    f.as_strided(one, (1,), 2 * rows), i.as_strided(wide, (top, 1), at), f.as_strided(wide, (top, 1), at + rows * top))


def token_logprobs(fn, logits, tokens=None, top: int = 0, out: Logprobs | None = None) -> Logprobs:
    """logits: fp32 or bf16 [rows][vocab] on a CUDA device, any row stride; tokens: int32 [rows] (< 0: none) or None; top: how many
    alternatives (0..32). out: buffers of an earlier call of the same sizes, written again."""
    shape, dtype, dev = logits.shape, logits.dtype, logits.get_device()
    if len(shape) != 2 or dtype not in _TYPE or dev < 0 or shape[1] < 1 or (logits.stride(1) != 1 and shape[1] > 1):
        raise ValueError(f"logits: fp32 or bf16 [rows][vocab] on a CUDA device with adjacent entries is wanted, got {dtype} {tuple(shape)} "
                         f"on {logits.device}")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top: 0..{MAX_TOP} is wanted")
    rows, vocab = shape
    if tokens is not None:
        _ints("tokens", tokens, (rows,), dev)
    if out is None:
        out = _make(rows, top, logits.device, tokens is not None)
    else:
        for name, t, want, kind in (("logprob", out.logprob, (rows,), torch.float32), ("rank", out.rank, (rows,), torch.int32),
                                    ("entropy", out.entropy, (rows,), torch.float32), ("top_ids", out.top_ids, (rows, top), torch.int32),
                                    ("top_logprobs", out.top_logprobs, (rows, top), torch.float32)):
            if (t is None) != (tokens is None and name in ("logprob", "rank")) or t is not None and (
                    t.shape != want or t.dtype is not kind or not t.is_contiguous() or t.get_device() != dev):
                raise ValueError(f"out.{name}: not of this call's sizes, type and device")
    token = logprob = rank = None
    if tokens is not None:
        token, logprob, rank = tokens.data_ptr(), out.logprob.data_ptr(), out.rank.data_ptr()
    fn.logprobs(_TYPE[dtype], logits.data_ptr(), logits.stride(0), rows, vocab, token, logprob, rank, out.entropy.data_ptr(), top,
                out.top_ids.data_ptr(), out.top_logprobs.data_ptr(), _stream(logits.device))
    return out
