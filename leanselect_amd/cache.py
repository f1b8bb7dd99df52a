"""Decode KV cache in HBM: the counterpart of the reference's ``InfLLMv2Cache``
(leanselect/models/minicpm.py:1188-1490) for the LeanSelect model.

All layers' keys (after RoPE), values and 32/16 compressed keys live in
preallocated device tensors ``[layers, batch, capacity, G, D]`` (capacity
rounded up to the 64-token page), so appending a token writes in place
instead of concatenating, and the compressed keys are extended by the windows
each step completes (``ls_kvcache_append``) instead of being kept as Python
lists.  A step of new tokens is written layer by layer between ``begin`` and
``end``; during the step ``seqlens_after`` holds the lengths including it.

``kv_format="q8"`` holds keys and values in 8 bits (e4m3 pages with a power-of-two
scale per page and head, ``ops.decode_q8``): half the memory and half the bytes a
step reads.  The compressed keys stay in ``dtype``; those the cache forms are means
of the keys as it holds them.

``fork`` makes a :class:`SharedPrefixKVCache` of a cache with one sequence: several sequences that
go on from it, its keys and values kept once.
"""
from __future__ import annotations

import torch

from .ops.cache_attention import shared_prefix_attention
from .ops.decode import kvcache_append, n_windows, sparse_attention_kvcache
from .ops.decode_q8 import kvcache_append_q8, new_kvcache_q8, sparse_attention_kvcache_q8

__all__ = ["LeanSelectKVCache", "SharedPrefixKVCache"]


class LeanSelectKVCache:
    def __init__(self, num_layers: int, batch: int, capacity: int, num_kv_heads: int,
                 head_dim: int = 128, *, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 kernel_size: int = 32, kernel_stride: int = 16, kv_format: str = "native"):
        if num_layers < 1 or batch < 1 or capacity < 1:
            raise ValueError("num_layers, batch and capacity must be positive")
        if kv_format not in ("native", "q8"):
            raise ValueError(f"unknown kv_format {kv_format!r}; expected 'native' or 'q8'")
        if kv_format == "q8" and ((kernel_size, kernel_stride) != (32, 16)
                                  or dtype not in (torch.bfloat16, torch.float16)):
            raise ValueError("the 8-bit cache forms windows of 32 keys at stride 16, in bf16 or fp16")
        self.kv_format = kv_format
        cap = -(-int(capacity) // 64) * 64
        self.num_layers, self.batch, self.capacity = int(num_layers), int(batch), cap
        self.kernel_size, self.kernel_stride = int(kernel_size), int(kernel_stride)
        self.device = torch.device(device)
        shape = (num_layers, batch, cap, num_kv_heads, head_dim)
        if kv_format == "q8":  # per layer [batch, pages, ...], see ops.decode_q8
            flat = new_kvcache_q8(num_layers * batch, cap, num_kv_heads, head_dim, device=self.device)
            self.k8, self.v8, self.k_scale, self.v_scale = (
                t.view(num_layers, batch, *t.shape[1:]) for t in flat)
        else:
            self.k = torch.empty(shape, dtype=dtype, device=self.device)
            self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self.kc = self._compressed_keys((num_layers, batch, num_kv_heads, head_dim), dtype)
        self.lengths = [0] * batch  # tokens held before the open step
        self.seqlens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self._step = None

    def _compressed_keys(self, shape: tuple[int, ...], dtype: torch.dtype) -> torch.Tensor | None:
        layers, batch, *rest = shape
        cap_c = max(1, n_windows(self.capacity, self.kernel_size, self.kernel_stride))
        return torch.empty((layers, batch, cap_c, *rest), dtype=dtype, device=self.device)

    # -- step protocol --------------------------------------------------------
    def begin(self, n_new: list[int]) -> None:
        """Open a step that appends ``n_new[b]`` tokens to sequence ``b``."""
        if self._step is not None:
            raise RuntimeError("a cache step is already open")
        if len(n_new) != self.batch or any(n < 0 for n in n_new):
            raise ValueError(f"n_new must hold {self.batch} non-negative counts")
        after = [l + n for l, n in zip(self.lengths, n_new)]
        if max(after) > self.capacity:
            raise ValueError(f"the step would exceed the cache capacity {self.capacity}")
        cu = [0]
        for n in n_new:
            cu.append(cu[-1] + int(n))
        self._step = dict(
            cu_host=cu, cu=torch.tensor(cu, dtype=torch.int32, device=self.device),
            after_host=after, after=torch.tensor(after, dtype=torch.int32, device=self.device))

    def update(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Write layer ``layer``'s packed new keys / values ``[sum n_new, G, D]``
        (and the compressed windows they complete) into the cache."""
        st = self._require_step()
        append = kvcache_append_q8 if self.kv_format == "q8" else kvcache_append
        append(*self.layer(layer), self.seqlens, k_new, v_new, st["cu"], kc_cache=self.kc[layer],
               kernel_size=self.kernel_size, kernel_stride=self.kernel_stride,
               cache_seqlens_host=self.lengths, cu_seqlens_new_host=st["cu_host"])

    def attend(self, layer: int, q: torch.Tensor, topk_idx: torch.Tensor, cu_seqlens_q: torch.Tensor,
               **kw) -> torch.Tensor:
        """Attention of the open step's rows over layer ``layer``, restricted to their page
        plans: ``ops.sparse_attention_kvcache`` (or its 8-bit form; ``kw`` are its options)."""
        st = self._require_step()
        attention = sparse_attention_kvcache_q8 if self.kv_format == "q8" else sparse_attention_kvcache
        return attention(q, *self.layer(layer), st["after"], topk_idx, cu_seqlens_q, **kw)

    def layer(self, layer: int) -> tuple[torch.Tensor, ...]:
        """Layer ``layer``'s cache tensors: ``(k, v)``, or ``(k8, v8, k_scale, v_scale)``."""
        if self.kv_format == "q8":
            return self.k8[layer], self.v8[layer], self.k_scale[layer], self.v_scale[layer]
        return self.k[layer], self.v[layer]

    def end(self) -> None:
        """Close the step: the appended tokens count from now on."""
        st = self._require_step()
        self.lengths = list(st["after_host"])
        self.seqlens = st["after"]
        self._step = None

    @property
    def seqlens_after(self) -> torch.Tensor:
        """int32 ``[batch]`` lengths including the open step."""
        return self._require_step()["after"]

    @property
    def lengths_after(self) -> list[int]:
        return list(self._require_step()["after_host"])

    @property
    def positions(self) -> list[int]:
        """The positions that the next token of each sequence takes (outside a step)."""
        return list(self.lengths)

    def fork(self, batch: int, capacity: int) -> "SharedPrefixKVCache":
        """``batch`` sequences that go on from this cache's one, for up to ``capacity`` tokens each.
        The cache is the prefix of them all and must not change while they are in use."""
        return SharedPrefixKVCache(self, batch, capacity)

    def get_seq_length(self) -> int:
        """Tokens of the longest sequence, a shared prefix included (outside a step)."""
        return max(self.lengths)

    def _require_step(self):
        if self._step is None:
            raise RuntimeError("no cache step is open (call begin first)")
        return self._step


class SharedPrefixKVCache(LeanSelectKVCache):
    """Sequences that begin with what ``prefix`` (a cache of one sequence, 16-bit) holds, each with a
    cache of its own behind it.  The step protocol is that of :class:`LeanSelectKVCache`, lengths
    counting the own tokens; ``attend`` is dense, over the prefix and the own tokens (no page plans,
    and no compressed keys are formed)."""

    def __init__(self, prefix: LeanSelectKVCache, batch: int, capacity: int):
        if prefix.kv_format != "native" or isinstance(prefix, SharedPrefixKVCache):
            raise ValueError("only a 16-bit cache without a prefix of its own can be shared")
        if prefix.batch != 1 or prefix.lengths[0] < 1 or prefix._step is not None:
            raise ValueError("a shared prefix is one sequence, prefilled, with no step open")
        super().__init__(prefix.num_layers, batch, capacity, prefix.k.shape[3], prefix.k.shape[4],
                         dtype=prefix.k.dtype, device=prefix.device, kernel_size=prefix.kernel_size,
                         kernel_stride=prefix.kernel_stride)
        self.prefix_len = prefix.lengths[0]
        self.k_prefix = prefix.k[:, 0, :self.prefix_len]
        self.v_prefix = prefix.v[:, 0, :self.prefix_len]

    def _compressed_keys(self, shape, dtype):
        return None

    def update(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        st = self._require_step()
        kvcache_append(*self.layer(layer), self.seqlens, k_new, v_new, st["cu"],
                       cache_seqlens_host=self.lengths, cu_seqlens_new_host=st["cu_host"])

    def attend(self, layer: int, q: torch.Tensor, cu_seqlens_q: torch.Tensor, **kw) -> torch.Tensor:
        """Attention of the open step's rows over the prefix and their own tokens
        (``ops.shared_prefix_attention``; ``kw`` are its options)."""
        st = self._require_step()
        return shared_prefix_attention(q, self.k_prefix[layer], self.v_prefix[layer], *self.layer(layer),
                                       st["after"], cu_seqlens_q, max(st["after_host"]), **kw)

    @property
    def positions(self) -> list[int]:
        return [self.prefix_len + n for n in self.lengths]

    def get_seq_length(self) -> int:
        return max(self.positions)

    def fork(self, batch: int, capacity: int):
        raise ValueError("only a 16-bit cache without a prefix of its own can be shared")
