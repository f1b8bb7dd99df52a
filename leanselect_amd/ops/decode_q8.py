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

from operator import gt

import torch

from .. import _hip

__all__ = ["new_kvcache_q8", "kvcache_append_q8", "sparse_attention_kvcache_q8",
           "dense_attention_kvcache_q8"]

PAGE, HEAD_DIM = 64, 128
_E4M3 = torch.float8_e4m3fn
_CODES = {torch.bfloat16: _hip.LS_BF16, torch.float16: _hip.LS_F16}
_PAGE_BYTES = PAGE * HEAD_DIM
_MAX_SPLITS = 256
_SCALE = HEAD_DIM ** -0.5
_WORKGROUPS = 256


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


def _cache_dims(k8, v8, k_scale, v_scale) -> tuple[int, int, int, int, int]:
    """``(batch, pages, num_kv_heads, batch stride, scale batch stride)`` of a well-formed cache."""
    if k8.ndim != 5 or k8.dtype is not _E4M3 or v8.dtype is not _E4M3 \
            or k_scale.dtype is not torch.uint8 or v_scale.dtype is not torch.uint8:
        _refuse_cache()
    B, P, G, rows, cols = k8.shape
    scales = (B, P, G)
    if rows != PAGE or cols != HEAD_DIM or v8.shape != (B, P, G, HEAD_DIM, PAGE) \
            or k_scale.shape != scales or v_scale.shape != scales:
        _refuse_cache()
    if k8.is_contiguous() and v8.is_contiguous() and k_scale.is_contiguous() \
            and v_scale.is_contiguous():
        return B, P, G, P * G * _PAGE_BYTES, P * G
    ks, vs, row = k8.stride(), v8.stride(), (G * _PAGE_BYTES, _PAGE_BYTES)
    if ks[1:] != (*row, HEAD_DIM, 1) or vs[1:] != (*row, PAGE, 1) or ks[0] != vs[0] \
            or k_scale.stride()[1:] != (G, 1) or v_scale.stride() != k_scale.stride():
        raise ValueError("each sequence's pages and scales must be dense, k and v with the same "
                         "batch strides")
    return B, P, G, ks[0], k_scale.stride(0)


def _refuse_cache():
    raise ValueError(f"the cache must be k8 float8_e4m3fn [batch, pages, num_kv_heads, {PAGE}, "
                     f"{HEAD_DIM}], v8 float8_e4m3fn [batch, pages, num_kv_heads, {HEAD_DIM}, "
                     f"{PAGE}] and k_scale, v_scale uint8 [batch, pages, num_kv_heads]")


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
    B, P, G, cache_stride, scale_stride = _cache_dims(k8, v8, k_scale, v_scale)
    shape, dtype = k_new.shape, k_new.dtype
    if len(shape) != 3 or shape[1] != G or shape[2] != HEAD_DIM or v_new.shape != shape:
        raise ValueError("k_new and v_new must be [total_new, num_kv_heads, head_dim] like the cache")
    code = _CODES.get(dtype)
    if code is None or v_new.dtype is not dtype:
        raise ValueError("new keys/values must be bf16 or fp16, k and v alike")
    total = shape[0]
    if cache_seqlens.dtype is not torch.int32 or cu_seqlens_new.dtype is not torch.int32:
        raise ValueError("cache_seqlens and cu_seqlens_new must be int32")
    lens = cache_seqlens.tolist() if cache_seqlens_host is None else cache_seqlens_host
    cu = cu_seqlens_new.tolist() if cu_seqlens_new_host is None else cu_seqlens_new_host
    if B < 1 or cache_seqlens.shape != (B,) or cu_seqlens_new.shape != (B + 1,) \
            or len(lens) != B or len(cu) != B + 1 or cu[0] != 0 or cu[-1] != total:
        raise ValueError("cache_seqlens must be [batch] and cu_seqlens_new [batch + 1] offsets "
                         "of the packed new rows")
    if B > 1 and (cache_stride < P * G * _PAGE_BYTES or scale_stride < P * G
                  or kc_cache is not None and kc_cache.stride(0) == 0):
        raise ValueError("sequences that share pages or windows cannot be appended to")
    k8_ptr, v8_ptr = k8.data_ptr(), v8.data_ptr()
    ks_ptr, vs_ptr = k_scale.data_ptr(), v_scale.data_ptr()
    if abs(k8_ptr - v8_ptr) < B * cache_stride or abs(ks_ptr - vs_ptr) < B * scale_stride:
        pages, scales = P * G * _PAGE_BYTES, P * G
        if _hip.rows_overlap(k8_ptr, cache_stride, B, pages, v8_ptr, cache_stride, B, pages) \
                or _hip.rows_overlap(ks_ptr, scale_stride, B, scales, vs_ptr, scale_stride, B, scales):
            raise ValueError("keys and values must not share pages or scales")
    after = [n + b - a for n, a, b in zip(lens, cu, cu[1:])]
    longest = max(after)
    if min(lens) < 0 or longest > P * PAGE or any(map(gt, lens, after)):
        raise ValueError(f"sequences of {lens} tokens cannot become {after} in a cache with a "
                         f"capacity of {P * PAGE}")
    kc = (None, 0, 0, 0)
    if kc_cache is not None:
        if kernel_size != 32 or kernel_stride != 16:
            raise ValueError("the 8-bit cache forms windows of 32 keys at stride 16")
        kc_shape, kc_stride = kc_cache.shape, kc_cache.stride()
        if len(kc_shape) != 4 or kc_shape[0] != B or kc_shape[2] != G or kc_shape[3] != HEAD_DIM \
                or kc_stride[2] != HEAD_DIM or kc_stride[3] != 1 or kc_cache.dtype is not dtype:
            raise ValueError("kc_cache must be [batch, kc_capacity, num_kv_heads, head_dim] in "
                             "k_new's dtype with dense rows")
        if longest >= 32 and (longest - 32) // 16 + 1 > kc_shape[1]:
            raise ValueError(f"{(longest - 32) // 16 + 1} compressed windows exceed kc_capacity "
                             f"{kc_shape[1]}")
        if kc_stride[1] < G * HEAD_DIM or kc_stride[0] < kc_shape[1] * kc_stride[1]:
            _check_windows(kc_shape, kc_stride)
        kc = (kc_cache.data_ptr(), kc_stride[0], kc_stride[1], kc_shape[1])
    index = _hip.gpu_index(k8, v8, k_scale, v_scale, cache_seqlens, k_new, v_new, cu_seqlens_new,
                           kc_cache)
    cache_seqlens, cu_seqlens_new = cache_seqlens.contiguous(), cu_seqlens_new.contiguous()
    # One row stride serves both: dense 16-byte aligned rows with equal strides, else copies.
    row, k_ptr, v_ptr = k_new.stride(), k_new.data_ptr(), v_new.data_ptr()
    if (k_ptr | v_ptr) & 15 or row[0] & 7 or row[1] != HEAD_DIM or row[2] != 1 or v_new.stride() != row:
        k_new = k_new.clone(memory_format=torch.contiguous_format)
        v_new = v_new.clone(memory_format=torch.contiguous_format)
        row, k_ptr, v_ptr = (G * HEAD_DIM,), k_new.data_ptr(), v_new.data_ptr()
    _hip.launch(index, "ls_kvcache_append_q8", k8_ptr, v8_ptr, cache_stride, ks_ptr, vs_ptr,
                scale_stride, P, cache_seqlens.data_ptr(), k_ptr, v_ptr, row[0],
                cu_seqlens_new.data_ptr(), total, B, G, HEAD_DIM, code, *kc)


def _check_windows(shape, stride) -> None:
    """Refuses compressed windows that overlap (sequences may lie within windows or around them)."""
    width = shape[2] * HEAD_DIM
    for step, n in sorted((step, n) for step, n in zip(stride[:2], shape) if n > 1):
        if step < width:
            raise ValueError("kc_cache's windows must not overlap")
        width += (n - 1) * step


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
                   -(-int(max_len) // PAGE), causal, softmax_scale, n_splits, return_lse, out)


def _attend(q, k8, v8, k_scale, v_scale, cache_seqlens, topk_idx, cu_seqlens_q, n_pages, causal,
            softmax_scale, n_splits, return_lse, out):
    B, P, G, cache_stride, scale_stride = _cache_dims(k8, v8, k_scale, v_scale)
    code, q_shape = _CODES.get(q.dtype), q.shape
    if code is None or len(q_shape) != 3:
        _refuse_queries(G)
    total_q, H, cols = q_shape
    if cols != HEAD_DIM or H % G or not G <= H <= 16 * G:
        _refuse_queries(G)
    if cache_seqlens.dtype is not torch.int32 or cache_seqlens.shape != (B,) \
            or cu_seqlens_q.dtype is not torch.int32 or cu_seqlens_q.shape != (B + 1,):
        raise ValueError("cache_seqlens must be int32 [batch] and cu_seqlens_q int32 [batch + 1]")
    ids = None
    if topk_idx is not None:
        g, t, n_pages = topk_idx.shape
        if g != G or t != total_q or not 1 <= n_pages <= 256:
            raise ValueError(f"topk_idx must be [{G}, {total_q}, k] with 1 <= k <= 256")
    else:
        n_pages = max(1, min(n_pages, P))
    given = out is not None
    if given:
        _hip.check_out(out, (total_q, H, HEAD_DIM), q.dtype, q.device)
        if out.data_ptr() % 16 or out.data_ptr() == q.data_ptr() and total_q:
            raise ValueError("out must be 16-byte aligned and must not overlap q")
    index = _hip.gpu_index(q, k8, v8, k_scale, v_scale, cache_seqlens, cu_seqlens_q, topk_idx)
    cache_seqlens, cu_seqlens_q = cache_seqlens.contiguous(), cu_seqlens_q.contiguous()
    if topk_idx is not None:
        if topk_idx.dtype is not torch.int32 or not topk_idx.is_contiguous():
            topk_idx = _hip.page_ids(topk_idx)
        ids = topk_idx.data_ptr()
    row, q_ptr = q.stride(), q.data_ptr()
    if q_ptr & 15 or row[0] & 7 or row[1] != HEAD_DIM or row[2] != 1:  # rows the kernels do not read
        q = q.clone(memory_format=torch.contiguous_format)
        row, q_ptr = (H * HEAD_DIM,), q.data_ptr()
    elif given and _hip.rows_overlap(out.data_ptr(), 2 * H * HEAD_DIM, total_q, 2 * H * HEAD_DIM, q_ptr,
                                     2 * row[0], total_q if row[0] else 1, 2 * H * HEAD_DIM):
        raise ValueError("out must be 16-byte aligned and must not overlap q")
    if n_splits is None:
        # Slices of a row: as many as leave every workgroup its compute unit, at least a page a wave.
        # One slice (eight waves, no join) up to three pages a wave, a launch less for the host (us,
        # replayed and called, one slice and several: 1 row of 16 pages 9.6 / 10.2, 8.8 / 14.6, of 24
        # pages 12.2 / 12.4, 9.0 / 15.0, of 32 pages 14.6 / 14.7, 9.0 / 14.7), up to 32 pages from 48
        # workgroups (24 rows of two heads 15.7 / 15.9, 14.0 / 19.8; 48 rows 16.6, 18.1 replayed), and
        # where the rows nearly fill the device meanwhile (63 pages, replayed: 48 rows 29.8, 26.7, 56
        # rows 33.6, 30.5, 64 rows 35.1, 34.6, 72 rows 36.3, 46.0).  More workgroups than units: 48
        # rows of 63 pages in 2 slices 26.7, in 3 31.9; 65 rows of 469 in 1 slice 203, in 2 259, in 3 202.
        pairs = total_q * G
        n_splits = 1 if n_pages <= max(24, min(32, 2 * pairs // 3), pairs // 2) \
            else min(-(-n_pages // 4), _WORKGROUPS // max(1, pairs))
    n_splits = max(1, min(int(n_splits), _MAX_SPLITS))
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((H, total_q), dtype=torch.float32, device=q.device) if return_lse else None
    # The slices' partial sums, maxima and weights, ls_attn_kvcache_q8_workspace_size bytes, counted
    # in q's 16-bit elements (the cheapest tensor to make here).
    nbytes = 4 * total_q * H * n_splits * (HEAD_DIM + 2) if n_splits > 1 else 0
    ws = q.new_empty(nbytes >> 1) if nbytes else None
    _hip.launch(index, "ls_attn_kvcache_q8", q_ptr, row[0], cu_seqlens_q.data_ptr(), total_q,
                k8.data_ptr(), v8.data_ptr(), cache_stride, k_scale.data_ptr(), v_scale.data_ptr(),
                scale_stride, P, cache_seqlens.data_ptr(), B, H, G, HEAD_DIM, code, ids, n_pages,
                _SCALE if softmax_scale is None else float(softmax_scale), 1 if causal else 0,
                n_splits, out.data_ptr(), lse.data_ptr() if return_lse else None,
                ws.data_ptr() if nbytes else None, nbytes)
    return (out, lse) if return_lse else out


def _refuse_queries(G: int):
    raise ValueError(f"q must be bf16 or fp16 [total_q, H, {HEAD_DIM}], H a multiple of the cache's "
                     f"{G} heads and at most 16 times it")
