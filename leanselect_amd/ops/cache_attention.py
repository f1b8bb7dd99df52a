"""Attention over dense 16-bit caches with capped, biased or windowed scores, and for a batch that
shares a prefix, on the GPU.

- ``shared_prefix_attention``: rows of a batch whose sequences begin with the same keys, kept once,
  and go on in caches of their own; the prefix is read once for the batch;
- ``scored_attention`` (reached through ``dense_attention_kvcache``): one cache per sequence, with
  the options below.

A sequence with ``n`` query rows and ``len`` keys, the prefix's ``P`` included, has its row ``i`` at position
``p = len - n + i``.  Key ``j < len`` is visible where, with ``causal``, ``j <= p`` and, with ``window = (left,
right)``, ``p - left <= j <= p + right`` (a negative side is open).  A score is ``x = scale * q.k``, then
``softcap * tanh(x / softcap)`` (0: not capped; at most 512; the cap's float32 form, and with it ``lse``, is
within ``softcap * 2^-21``), then less ``alibi_slopes[h] * |p - j|``: the options of
``infllmv2_attn_with_kvcache`` (third_party/infllmv2/paper1.patch:2511-2615).  The reference has no
call for a shared prefix.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch

from .. import _hip

__all__ = ["shared_prefix_attention", "scored_attention"]

HEAD_DIM = 128
_CODES = {torch.bfloat16: _hip.LS_BF16, torch.float16: _hip.LS_F16}
_SCALE = HEAD_DIM ** -0.5
_MAX_SPLITS = 128
_STEP = 128


def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k_cache: torch.Tensor, v_cache: torch.Tensor,
                            cache_seqlens: torch.Tensor, cu_seqlens_q: torch.Tensor, max_len: int, *,
                            causal: bool = False, softmax_scale: float | None = None,
                            softcap: float = 0.0, alibi_slopes: torch.Tensor | None = None,
                            window: tuple[int, int] = (-1, -1), n_splits: int | None = None,
                            return_lse: bool = False, out: torch.Tensor | None = None):
    """``out [total_q, H, 128]`` of the rows ``q [total_q, H, 128]`` (bf16 or fp16; sequence ``b``'s are
    ``cu_seqlens_q[b]:cu_seqlens_q[b+1]``) over the keys every sequence begins with, ``k_prefix / v_prefix
    [P, G, 128]``, and its own ``cache_seqlens[b]`` in ``k_cache / v_cache [batch, capacity, G, 128]`` (and ``lse
    [H, total_q]`` float32 with ``return_lse``).  Positions count the prefix: own key ``j`` stands at
    ``P + j``.  ``max_len`` is the longest ``cache_seqlens`` (it only decides how the work is cut).
    A row that sees no key gives zeros and ``lse = +inf``.  Rows at and after
    ``cu_seqlens_q[-1]`` are left as they are."""
    if k_prefix.ndim != 3 or v_prefix.shape != k_prefix.shape:
        raise ValueError("k_prefix and v_prefix must be [prefix_len, num_kv_heads, head_dim]")
    return _attend(q, k_prefix, v_prefix, k_cache, v_cache, cache_seqlens, cu_seqlens_q, max_len,
                   causal, softmax_scale, softcap, alibi_slopes, window, n_splits, return_lse, out)


def scored_attention(q, k_cache, v_cache, cache_seqlens, cu_seqlens_q, max_len, *, causal=False,
                     softmax_scale=None, softcap=0.0, alibi_slopes=None, window=(-1, -1),
                     n_splits=None, return_lse=False, out=None):
    """``shared_prefix_attention`` without a prefix."""
    return _attend(q, None, None, k_cache, v_cache, cache_seqlens, cu_seqlens_q, max_len, causal,
                   softmax_scale, softcap, alibi_slopes, window, n_splits, return_lse, out)


def check_scores(softmax_scale, softcap, alibi_slopes, batch: int, num_heads: int) -> tuple[float, float]:
    """The scale and the cap as numbers, or ``ValueError`` for options that no call takes."""
    scale = _SCALE if softmax_scale is None else ctypes.c_float(float(softmax_scale)).value
    softcap = float(softcap)
    if not 0.0 < scale < math.inf or not 0.0 <= softcap < math.inf:
        raise ValueError("softmax_scale must be positive and softcap not negative, both finite (in float32)")
    if softcap and not 1e-20 <= softcap <= 512.0:
        raise ValueError(f"softcap must be 0 or from 1e-20 to 512 (got {softcap})")
    if alibi_slopes is not None and (alibi_slopes.dtype is not torch.float32
                                     or alibi_slopes.shape not in ((num_heads,), (batch, num_heads))):
        raise ValueError(f"alibi_slopes must be float32 [{num_heads}] or [{batch}, {num_heads}]")
    return scale, softcap


@lru_cache(maxsize=4096)
def _workspace_bytes(total_q: int, batch: int, H: int, G: int, prefix_len: int, max_len: int,
                     left: int, n_splits: int) -> int:
    return _hip.lib().ls_cache_attn_workspace_size(total_q, batch, H, G, prefix_len, max_len, left, n_splits)


def _key_strides(k: torch.Tensor, v: torch.Tensor, name: str) -> tuple[int, ...]:
    """The strides of ``[.., rows, G, 128]`` keys and values in front of the heads, as the kernels read
    both."""
    if k.is_contiguous() and v.is_contiguous():
        row, ok = k.shape[-2] * HEAD_DIM, True
        strides = (k.shape[-3] * row, row, 0, 0) if k.ndim == 4 else (row, 0, 0)
    else:  # a dimension of one may have any stride
        step, strides, ok = 1, [], True
        for i, (n, ks, vs) in enumerate(reversed(tuple(zip(k.shape, k.stride(), v.stride())))):
            if n > 1:
                ok = ok and ks == vs and (ks == step if i < 2 else ks % 8 == 0)
                strides.append(ks)
            else:
                strides.append(step)
            step = strides[-1] * n
        strides = tuple(reversed(strides))
    if not ok or (k.data_ptr() | v.data_ptr()) & 15 or strides[-3] >= 1 << 24:
        raise ValueError(f"{name} rows must be dense, 16-byte aligned and less than 2^24 elements apart, k and v with the "
                         "same strides")
    return strides[:-2]


def check_attention(q, k_cache, v_cache, softmax_scale, softcap, alibi_slopes, window) -> tuple:
    """The numbers of a call on ``q`` and the cache (scale, cap, window and the cache's strides), or ``ValueError``
    for what no call takes, whatever the lengths."""
    dtype, q_shape, c_shape = q.dtype, q.shape, k_cache.shape
    if dtype not in _CODES or len(q_shape) != 3 or q_shape[2] != HEAD_DIM:
        raise ValueError(f"q must be bf16 or fp16 [total_q, H, {HEAD_DIM}]")
    if len(c_shape) != 4 or c_shape[3] != HEAD_DIM or v_cache.shape != c_shape:
        raise ValueError(f"k_cache and v_cache must be [batch, capacity, num_kv_heads, {HEAD_DIM}]")
    H, (B, capacity, G, _) = q_shape[1], c_shape
    if B < 1 or G < 1 or H % G or not G <= H <= 16 * G:
        raise ValueError(f"q's {H} heads must be a multiple of the cache's {G}, at most 16 times")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError("q and the cache must share a dtype")
    if q_shape[0] * H >= 1 << 23 or capacity >= 1 << 30:
        raise ValueError("a call takes fewer than 2^23 rows and heads, and fewer than 2^30 keys a sequence")
    left, right = (min(max(int(x), -1), 1 << 30) for x in window)
    scale, softcap = check_scores(softmax_scale, softcap, alibi_slopes, B, H)
    return scale, softcap, left, right, *_key_strides(k_cache, v_cache, "the cache's")


def _attend(q, k_prefix, v_prefix, k_cache, v_cache, cache_seqlens, cu_seqlens_q, max_len, causal,
            softmax_scale, softcap, alibi_slopes, window, n_splits, return_lse, out):
    scale, softcap, left, right, c_batch, c_row = check_attention(q, k_cache, v_cache, softmax_scale, softcap,
                                                                  alibi_slopes, window)
    dtype, (total_q, H, _), (B, capacity, G, _) = q.dtype, q.shape, k_cache.shape
    if cache_seqlens.dtype is not torch.int32 or cache_seqlens.shape != (B,) \
            or cu_seqlens_q.dtype is not torch.int32 or cu_seqlens_q.shape != (B + 1,):
        raise ValueError("cache_seqlens must be int32 [batch] and cu_seqlens_q int32 [batch + 1]")
    P, p_row = 0, 0
    if k_prefix is not None:
        P = k_prefix.shape[0]
        if k_prefix.shape[1:] != (G, HEAD_DIM) or k_prefix.dtype is not dtype or v_prefix.dtype is not dtype:
            raise ValueError(f"the prefix must be [prefix_len, {G}, {HEAD_DIM}] in q's dtype")
        if P:
            p_row, = _key_strides(k_prefix, v_prefix, "the prefix's")
    slopes_stride = 0
    if alibi_slopes is not None:
        alibi_slopes = alibi_slopes.contiguous()
        slopes_stride = H if alibi_slopes.ndim == 2 else 0
    given = out is not None
    if given:
        _hip.check_out(out, (total_q, H, HEAD_DIM), dtype, q.device)
    index = _hip.gpu_index(q, k_cache, v_cache, cache_seqlens, cu_seqlens_q, k_prefix, v_prefix, alibi_slopes)
    cache_seqlens, cu_seqlens_q = cache_seqlens.contiguous(), cu_seqlens_q.contiguous()
    if given and total_q:
        _check_apart(out, q, k_cache, v_cache, k_prefix, v_prefix)
    row, q_ptr = q.stride(), q.data_ptr()
    if q_ptr & 15 or row[0] & 7 or row[1] != HEAD_DIM or row[2] != 1:  # rows the kernels do not read
        q = q.clone(memory_format=torch.contiguous_format)
        row, q_ptr = (H * HEAD_DIM,), q.data_ptr()
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((H, total_q), dtype=torch.float32, device=q.device) if return_lse else None
    splits = 0 if n_splits is None else max(1, min(int(n_splits), _MAX_SPLITS))
    max_len = -(-max(0, min(int(max_len), capacity)) // _STEP) * _STEP
    nbytes = _workspace_bytes(total_q, B, H, G, P, max_len, left, splits)
    ws = q.new_empty((nbytes + 1) >> 1) if nbytes else None  # counted in q's 16-bit elements
    _hip.launch(index, "ls_cache_attn", q_ptr, row[0], cu_seqlens_q.data_ptr(), total_q,
                k_prefix.data_ptr() if P else None, v_prefix.data_ptr() if P else None, p_row, P,
                k_cache.data_ptr(), v_cache.data_ptr(), c_batch, c_row, capacity,
                cache_seqlens.data_ptr(), B, H, G, HEAD_DIM, _CODES[dtype], max_len, scale, 1 if causal else 0,
                softcap, None if alibi_slopes is None else alibi_slopes.data_ptr(), slopes_stride,
                left, right, splits, out.data_ptr(), lse.data_ptr() if return_lse else None,
                ws.data_ptr() if nbytes else None, nbytes)
    return (out, lse) if return_lse else out


def _check_apart(out, q, *caches):
    """A given output must be 16-byte aligned and lie apart from what the kernels read."""
    at, nbytes = out.data_ptr(), out.numel() * 2
    row = out.shape[1] * HEAD_DIM * 2
    apart = not at & 15
    if q.stride(1) == HEAD_DIM and q.stride(2) == 1:
        apart = apart and not _hip.rows_overlap(at, row, out.shape[0], row, q.data_ptr(), 2 * q.stride(0),
                                                q.shape[0] if q.stride(0) else 1, row)
        tensors = caches
    else:
        tensors = (q, *caches)
    for t in tensors:
        if t is not None and t.numel():
            span = 2 * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            apart = apart and (at + nbytes <= t.data_ptr() or t.data_ptr() + span <= at)
    if not apart:
        raise ValueError("out must be 16-byte aligned and must not overlap q, the cache or the prefix")
