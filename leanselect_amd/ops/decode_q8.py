"""Decode over a KV cache held in 8 bits, on the GPU.

The counterparts of ``ops.decode``'s append and attention for a cache of e4m3
pages (64 tokens of one KV head) with one power-of-two scale each:

- ``new_kvcache_q8``: the tensors of an empty cache;
- ``kvcache_append_q8``: packed new keys/values into it, plus the compressed key
  windows they complete;
- ``sparse_attention_kvcache_q8`` / ``dense_attention_kvcache_q8``: attention of
  decode rows over the pages of their plans, or over every cached page.

Layout: keys ``k8 [batch, pages, G, 64, 128]`` and values ``v8 [batch, pages, G,
128, 64]`` as ``torch.float8_e4m3fn`` (a value channel's 64 tokens lie together,
token ``16 t + 4 q + i`` at place ``16 q + 4 t + i``), scale codes ``k_scale /
v_scale [batch, pages, G]`` as ``torch.uint8``, code ``c`` standing for ``2 ** (c -
127)``.  A page's code is the least ``c >= 1`` with ``max |x| <= 448 * 2 ** (c -
127)`` over the finite rows it has held since its first token; rows already there
are brought under a raised code.  Infinities and NaN are kept as NaN.

The reference's cache is 16-bit (leanselect/models/minicpm.py:1188-1490).
"""
from __future__ import annotations

import torch

from .. import _hip
from .decode import _lengths, n_windows

__all__ = ["new_kvcache_q8", "kvcache_append_q8", "sparse_attention_kvcache_q8",
           "dense_attention_kvcache_q8"]

PAGE, HEAD_DIM = 64, 128
_PAGE_BYTES = PAGE * HEAD_DIM
_MAX_SPLITS = 256


def new_kvcache_q8(batch: int, capacity: int, num_kv_heads: int, head_dim: int = 128, *,
                   device="cuda") -> tuple[torch.Tensor, ...]:
    """``(k8, v8, k_scale, v_scale)`` of an empty cache for ``batch`` sequences of up to
    ``capacity`` tokens (rounded up to the 64-token page)."""
    if batch < 1 or capacity < 1 or num_kv_heads < 1:
        raise ValueError("batch, capacity and num_kv_heads must be positive")
    if head_dim != HEAD_DIM:
        raise ValueError(f"the 8-bit cache holds heads of {HEAD_DIM} channels (got {head_dim})")
    pages = -(-int(capacity) // PAGE)
    shape = (batch, pages, num_kv_heads)
    k8 = torch.empty((*shape, PAGE, HEAD_DIM), dtype=torch.float8_e4m3fn, device=device)
    v8 = torch.empty((*shape, HEAD_DIM, PAGE), dtype=torch.float8_e4m3fn, device=device)
    return (k8, v8, torch.empty(shape, dtype=torch.uint8, device=device),
            torch.empty(shape, dtype=torch.uint8, device=device))


def _check_cache_q8(k8, v8, k_scale, v_scale) -> tuple[int, int, int]:
    if k8.ndim != 5 or k8.shape[3:] != (PAGE, HEAD_DIM) or k8.dtype != torch.float8_e4m3fn:
        raise ValueError(f"k8 must be float8_e4m3fn [batch, pages, num_kv_heads, {PAGE}, {HEAD_DIM}]")
    B, P, G = k8.shape[:3]
    if v8.shape != (B, P, G, HEAD_DIM, PAGE) or v8.dtype != torch.float8_e4m3fn:
        raise ValueError(f"v8 must be float8_e4m3fn [batch, pages, num_kv_heads, {HEAD_DIM}, {PAGE}]")
    if k_scale.shape != (B, P, G) or v_scale.shape != (B, P, G) \
            or k_scale.dtype != torch.uint8 or v_scale.dtype != torch.uint8:
        raise ValueError("k_scale and v_scale must be uint8 [batch, pages, num_kv_heads]")
    row = (G * _PAGE_BYTES, _PAGE_BYTES)
    ks, vs = k8.stride(), v8.stride()
    if ks[1:] != (*row, HEAD_DIM, 1) or vs[1:] != (*row, PAGE, 1) or ks[0] != vs[0] \
            or k_scale.stride()[1:] != (G, 1) or v_scale.stride() != k_scale.stride():
        raise ValueError("each sequence's pages and scales must be dense, k and v with the same "
                         "batch strides")
    return B, P, G


def kvcache_append_q8(k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor,
                      v_scale: torch.Tensor, cache_seqlens: torch.Tensor, k_new: torch.Tensor,
                      v_new: torch.Tensor, cu_seqlens_new: torch.Tensor, *,
                      kc_cache: torch.Tensor | None = None, kernel_size: int = 32,
                      kernel_stride: int = 16, cache_seqlens_host: list[int] | None = None,
                      cu_seqlens_new_host: list[int] | None = None) -> None:
    """Write ``k_new / v_new [total_new, G, 128]`` (bf16 or fp16; sequence ``b``'s rows
    are ``cu_seqlens_new[b]:cu_seqlens_new[b+1]``) at positions ``cache_seqlens[b] + i`` of
    the 8-bit cache and, with ``kc_cache [batch, kc_capacity, G, 128]`` (``k_new``'s dtype),
    the compressed windows the new tokens complete: means of the 32 keys as the cache
    holds them.  ``cache_seqlens`` is left as it is (advance it after)."""
    B, P, G = _check_cache_q8(k8, v8, k_scale, v_scale)
    if k_new.ndim != 3 or v_new.shape != k_new.shape or k_new.shape[1:] != (G, HEAD_DIM):
        raise ValueError("k_new and v_new must be [total_new, num_kv_heads, head_dim] like the cache")
    if k_new.dtype not in (torch.bfloat16, torch.float16) or v_new.dtype != k_new.dtype:
        raise ValueError("new keys/values must be bf16 or fp16, k and v alike")
    lens = _lengths(cache_seqlens, cache_seqlens_host, "cache_seqlens")
    cu = _lengths(cu_seqlens_new, cu_seqlens_new_host, "cu_seqlens_new")
    if len(lens) != B or cache_seqlens.numel() != B or len(cu) != B + 1 \
            or cu_seqlens_new.numel() != B + 1 or cu[0] != 0 or cu[-1] != k_new.shape[0]:
        raise ValueError("cache_seqlens must be [batch] and cu_seqlens_new [batch + 1] offsets "
                         "of the packed new rows")
    windows = 0
    for b, before in enumerate(lens):
        after = before + cu[b + 1] - cu[b]
        if before < 0 or after < before or after > P * PAGE:
            raise ValueError(f"appending {cu[b + 1] - cu[b]} tokens to {before} of sequence {b} "
                             f"exceeds the capacity {P * PAGE}")
        if kc_cache is not None and after > before:
            nw = n_windows(after)
            if nw > kc_cache.shape[1]:
                raise ValueError(f"{nw} compressed windows exceed kc_capacity {kc_cache.shape[1]}")
            windows += nw - n_windows(before)
    if kc_cache is not None:
        if (kernel_size, kernel_stride) != (32, 16):
            raise ValueError("the 8-bit cache forms windows of 32 keys at stride 16")
        if kc_cache.ndim != 4 or kc_cache.shape[0] != B or kc_cache.shape[2:] != (G, HEAD_DIM) \
                or kc_cache.dtype != k_new.dtype or kc_cache.stride()[2:] != (HEAD_DIM, 1):
            raise ValueError("kc_cache must be [batch, kc_capacity, num_kv_heads, head_dim] in "
                             "k_new's dtype with dense rows")
    dev = _hip.require_gpu(k8, v8, k_scale, v_scale, cache_seqlens, k_new, v_new, cu_seqlens_new,
                           kc_cache)
    # One row stride serves both: dense 16-byte aligned rows with equal strides, else copies.
    if k_new.stride()[1:] != (HEAD_DIM, 1) or v_new.stride() != k_new.stride() \
            or k_new.stride(0) % 8 or k_new.data_ptr() % 16 or v_new.data_ptr() % 16:
        k_new = k_new.clone(memory_format=torch.contiguous_format)
        v_new = v_new.clone(memory_format=torch.contiguous_format)
    kc = (kc_cache.data_ptr(), kc_cache.stride(0), kc_cache.stride(1), kc_cache.shape[1]) \
        if kc_cache is not None else (None, 0, 0, 0)
    _hip.launch(dev, "ls_kvcache_append_q8", k8.data_ptr(), v8.data_ptr(), k8.stride(0),
                k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), P,
                cache_seqlens.contiguous().data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
                k_new.stride(0), cu_seqlens_new.contiguous().data_ptr(), k_new.shape[0], B, G,
                HEAD_DIM, _hip.dtype_code(k_new.dtype), *kc, windows)


def sparse_attention_kvcache_q8(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor,
                                k_scale: torch.Tensor, v_scale: torch.Tensor,
                                cache_seqlens: torch.Tensor, topk_idx: torch.Tensor,
                                cu_seqlens_q: torch.Tensor, *, causal: bool = False,
                                softmax_scale: float | None = None, n_splits: int | None = None,
                                return_lse: bool = False, out: torch.Tensor | None = None):
    """``out [total_q, H, 128]`` of the rows ``q [total_q, H, 128]`` (bf16 or fp16) over the
    8-bit cache, restricted to each row's plan ``topk_idx [G, total_q, k]`` (and ``lse [H,
    total_q]`` float32 with ``return_lse``): ``ops.sparse_attention_kvcache`` over the values
    the cache stands for.  Ids below 0, past the sequence or repeated are ignored; a row that
    sees no key gives zeros and ``lse = +inf``.  Rows of ``out`` and ``lse`` at and after
    ``cu_seqlens_q[-1]`` are left as they are."""
    if topk_idx is None or topk_idx.ndim != 3:
        raise ValueError("topk_idx must be [G, total_q, k]")
    return _attend(q, k8, v8, k_scale, v_scale, cache_seqlens, topk_idx, cu_seqlens_q, 0, causal,
                   softmax_scale, n_splits, return_lse, out)


def dense_attention_kvcache_q8(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor,
                               k_scale: torch.Tensor, v_scale: torch.Tensor,
                               cache_seqlens: torch.Tensor, cu_seqlens_q: torch.Tensor,
                               max_len: int, *, causal: bool = False,
                               softmax_scale: float | None = None, n_splits: int | None = None,
                               return_lse: bool = False, out: torch.Tensor | None = None):
    """``sparse_attention_kvcache_q8`` over every cached page; ``max_len`` is the longest
    sequence's length (it only decides how the work is cut)."""
    return _attend(q, k8, v8, k_scale, v_scale, cache_seqlens, None, cu_seqlens_q,
                   max(1, -(-int(max_len) // PAGE)), causal, softmax_scale, n_splits, return_lse, out)


def _attend(q, k8, v8, k_scale, v_scale, cache_seqlens, topk_idx, cu_seqlens_q, n_pages, causal,
            softmax_scale, n_splits, return_lse, out):
    B, P, G = _check_cache_q8(k8, v8, k_scale, v_scale)
    if q.ndim != 3 or q.shape[2] != HEAD_DIM or q.shape[1] % G or q.shape[1] > 16 * G \
            or q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"q must be bf16 or fp16 [total_q, H, {HEAD_DIM}], H a multiple of the "
                         f"cache's {G} heads and at most 16 times it")
    total_q, H, _ = q.shape
    if cache_seqlens.dtype != torch.int32 or cache_seqlens.shape != (B,) \
            or cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.shape != (B + 1,):
        raise ValueError("cache_seqlens must be int32 [batch] and cu_seqlens_q int32 [batch + 1]")
    if topk_idx is not None:
        if topk_idx.shape[:2] != (G, total_q) or not 1 <= topk_idx.shape[2] <= 256:
            raise ValueError(f"topk_idx must be [{G}, {total_q}, k] with 1 <= k <= 256")
        topk_idx = topk_idx.to(torch.int32).contiguous()
        n_pages = topk_idx.shape[2]
    if out is not None:
        _hip.check_out(out, (total_q, H, HEAD_DIM), q.dtype, q.device)
    dev = _hip.require_gpu(q, k8, v8, k_scale, v_scale, cache_seqlens, topk_idx, cu_seqlens_q)
    if q.stride()[1:] != (HEAD_DIM, 1) or q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if n_splits is None:
        # Workgroups of four waves per (row, group): enough of them to cover the
        # device when there are few rows, at least one page per wave.
        n_splits = max(1, min(-(-n_pages // 4), -(-256 // max(1, total_q * G))))
    n_splits = max(1, min(int(n_splits), _MAX_SPLITS))
    if out is None:
        out = torch.empty((total_q, H, HEAD_DIM), dtype=q.dtype, device=dev)
    lse = torch.empty((H, total_q), dtype=torch.float32, device=dev) if return_lse else None
    nbytes = _hip.lib().ls_attn_kvcache_q8_workspace_size(total_q, G, n_splits)
    ws = _hip.workspace(nbytes, dev) if nbytes else None
    _hip.launch(dev, "ls_attn_kvcache_q8", q.data_ptr(), q.stride(0),
                cu_seqlens_q.contiguous().data_ptr(), total_q, k8.data_ptr(), v8.data_ptr(),
                k8.stride(0), k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), P,
                cache_seqlens.contiguous().data_ptr(), B, H, G, HEAD_DIM, _hip.dtype_code(q.dtype),
                _hip.ptr(topk_idx), n_pages if topk_idx is not None else 0,
                HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale),
                1 if causal else 0, n_splits, out.data_ptr(), _hip.ptr(lse), _hip.ptr(ws), nbytes)
    return (out, lse) if return_lse else out
