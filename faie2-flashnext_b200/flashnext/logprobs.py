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


def _make(rows, top, dev, tokens=True):
    f = torch.empty(rows * (2 + top), dtype=torch.float32, device=dev).split([rows, rows, rows * top])
    i = torch.empty(rows * (1 + top), dtype=torch.int32, device=dev).split([rows, rows * top])
    return Logprobs(f[0] if tokens else None, i[0] if tokens else None, f[1], i[1].view(rows, top), f[2].view(rows, top))


def token_logprobs(fn, logits, tokens=None, top: int = 0, out: Logprobs | None = None) -> Logprobs:
    """logits: fp32 or bf16 [rows][vocab] on a CUDA device, any row stride; tokens: int32 [rows] (< 0: none) or None; top: how many
    alternatives (0..32). out: buffers of an earlier call of the same sizes, written again."""
    if logits.dim() != 2 or logits.dtype not in _TYPE or not logits.is_cuda or (logits.stride(1) != 1 and logits.shape[1] > 1) or \
            logits.shape[1] < 1:
        raise ValueError(f"logits: fp32 or bf16 [rows][vocab] on a CUDA device with adjacent entries is wanted, got {logits.dtype} "
                         f"{tuple(logits.shape)} on {logits.device}")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top: 0..{MAX_TOP} is wanted")
    rows, vocab = logits.shape
    dev = logits.get_device()
    if tokens is not None:
        _ints("tokens", tokens, (rows,), dev)
    if out is None:
        out = _make(rows, top, logits.device, tokens is not None)
    else:
        for name, t, shape, dtype in (("logprob", out.logprob, (rows,), torch.float32), ("rank", out.rank, (rows,), torch.int32),
                                      ("entropy", out.entropy, (rows,), torch.float32), ("top_ids", out.top_ids, (rows, top), torch.int32),
                                      ("top_logprobs", out.top_logprobs, (rows, top), torch.float32)):
            if (t is None) != (tokens is None and name in ("logprob", "rank")) or t is not None and (
                    t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != dev):
                raise ValueError(f"out.{name}: not of this call's sizes, type and device")
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    fn.logprobs(_TYPE[logits.dtype], logits.data_ptr(), logits.stride(0), rows, vocab, p(tokens), p(out.logprob), p(out.rank),
                p(out.entropy), top, p(out.top_ids), p(out.top_logprobs), _stream(logits.device))
    return out
