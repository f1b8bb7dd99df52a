"""Drawing the next tokens from logits, on the GPU.

``sample_logits`` draws a token for each row from random numbers that the caller gives, with
temperature, top-k, top-p and min-p, for the batch or for each row.  No counterpart in the reference,
whose generation is the host library's.
"""
from __future__ import annotations

import math

import torch

from .. import _hip

__all__ = ["sample_logits"]

_CODES = {torch.float32: _hip.LS_F32, torch.bfloat16: _hip.LS_BF16, torch.float16: _hip.LS_F16}
_MAX_VOCAB = 1 << 19


def check_settings(rows: int, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> tuple[list, list]:
    """The settings' tensors and their numbers (None for the other kind), or ``ValueError`` for what
    ``sample_logits`` does not take for ``rows`` rows."""
    each = []
    numbers = []
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if torch.is_tensor(value):
            if value.dtype is not dtype or value.shape != (rows,):
                raise ValueError(f"{name} must be a number or {dtype} [{rows}]")
            each.append(value)
            numbers.append(None)
        else:
            each.append(None)
            numbers.append(value)
    t, k, p, m = numbers
    if t is not None and not 0.0 <= t < math.inf:
        raise ValueError(f"temperature must be 0 or more and finite (got {t})")
    if k is not None and (not math.isfinite(k) or k != int(k)):
        raise ValueError(f"top_k must be a whole number (got {k})")
    if p is not None and not p > 0.0:
        raise ValueError(f"top_p must be above 0 (got {p})")
    if m is not None and not 0.0 <= m <= 1.0:
        raise ValueError(f"min_p must be 0 to 1 (got {m})")
    return each, numbers


def sample_logits(logits: torch.Tensor, u: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
                  min_p: float | torch.Tensor = 0.0, return_logprob: bool = False):
    """int32 ``tokens [rows]`` drawn from ``logits [rows, vocab]`` (float32, bf16 or fp16) by the numbers ``u
    [rows]`` (float32, in [0, 1)), and with ``return_logprob`` their log-probabilities (float32) in the
    distribution they were drawn from.

    A token's weight is ``exp((x - max x) / temperature)``.  Ordered by logit, ties to the lower index,
    the first ``top_k`` are kept (0 or less: all), of these the shortest run, of one at least, whose
    weights reach ``top_p`` of their sum (from 1: all), of these those of at least ``min_p`` of the
    largest.  The draw is the lowest index at which the running sum of the kept weights, in the
    vocabulary's order, exceeds ``u`` times their sum.  ``temperature`` 0 takes the largest logit (the
    lowest index; log-probability 0).

    NaN counts as -inf, which is never drawn; a row of nothing else gives -1 (and -inf); where the
    largest is +inf only such are drawn.  Each setting may be one number or one of each row (``top_k``
    int32, the others float32); a row's own numbers are not looked at on the host: a temperature
    that is not above 0 counts as 0.  A row's token does not depend on the other rows."""
    code = _CODES.get(logits.dtype)
    if code is None or logits.ndim != 2:
        raise ValueError("logits must be float32, bf16 or fp16 [rows, vocab]")
    rows, vocab = logits.shape
    if not 1 <= vocab <= _MAX_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {_MAX_VOCAB} tokens (got {vocab})")
    if u.dtype is not torch.float32 or u.shape != (rows,):
        raise ValueError(f"u must be float32 [{rows}]")
    each, (t, k, p, m) = check_settings(rows, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    index = _hip.gpu_index(logits, u, *each)
    if vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    u, each = u.contiguous(), [None if x is None else x.contiguous() for x in each]
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device) if return_logprob else None
    _hip.launch(index, "ls_sample_logits", logits.data_ptr(), logits.stride(0), rows, vocab, code,
                u.data_ptr(), 1.0 if t is None else float(t), 0 if k is None else max(-1, min(int(k), _MAX_VOCAB)),
                1.0 if p is None else float(p), 0.0 if m is None else float(m), *map(_hip.ptr, each),
                tokens.data_ptr(), _hip.ptr(logprob))
    return (tokens, logprob) if return_logprob else tokens
