"""Attention over a cache (capped, biased, windowed scores; a shared prefix) and sampling, in 64 bits,
from their definitions (test infrastructure only).

No reference output covers these; each function states the definition one row at a time."""
from __future__ import annotations

import math

import numpy as np
import torch

__all__ = ["cache_attention", "sample_row"]


def cache_attention(q, k_cache, v_cache, lens, cu, *, k_prefix=None, v_prefix=None, causal=False,
                    softmax_scale=None, softcap=0.0, alibi_slopes=None, window=(-1, -1)):
    """``(out, lse, out_bound, lse_bound)`` float64 of CPU tensors: the results, and how far a kernel's
    float32 sums, 16-bit inputs and split softmax weights may be off before its one rounding.

    Score: 128 exact products summed in float32 are off by 128 * 2^-24 sum |q k| at most; the scale, the
    bias, the base-2 exponent and its difference from the maximum a few 2^-24 of what they hold;
    the cap cap * 2^-20 (exp2 and reciprocal of one unit each, of values up to 2 cap).  A weight's
    relative error is the score's; its two 16-bit parts hold 2^-17 of it (fp16: and 2^-35 of the
    largest weight).  Sums: 2^-24 of the sum of magnitudes for each of n / 32 + 64 additions."""
    total, H, D = q.shape
    G = k_cache.shape[2]
    P = 0 if k_prefix is None else k_prefix.shape[0]
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    out = torch.zeros(total, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((H, total), math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    for b, length in enumerate(lens):
        length = max(0, min(length, k_cache.shape[1]))
        for t in range(cu[b], cu[b + 1]):
            p = P + length - (cu[b + 1] - cu[b]) + t - cu[b]
            j = torch.arange(P + length)
            see = torch.ones(P + length, dtype=torch.bool)
            if causal:
                see &= j <= p
            if window[0] >= 0:
                see &= j >= p - window[0]
            if window[1] >= 0:
                see &= j <= p + window[1]
            if not bool(see.any()):
                continue
            j = j[see]
            for h in range(H):
                g = h // (H // G)
                k, v = k_cache[b, :length, g], v_cache[b, :length, g]
                if P:
                    k, v = torch.cat((k_prefix[:, g], k)), torch.cat((v_prefix[:, g], v))
                k, v = k[see].double(), v[see].double()
                x = k @ q[t, h].double() * scale
                off = 130 * 2.0 ** -24 * scale * (k.abs() @ q[t, h].double().abs())
                if softcap > 0:
                    x = softcap * torch.tanh(x / softcap)
                    off = off + softcap * 2.0 ** -20
                if alibi_slopes is not None:
                    slope = alibi_slopes[h] if alibi_slopes.ndim == 1 else alibi_slopes[b, h]
                    bias = float(slope) * (p - j).abs().double()
                    x = x - bias
                    off = off + 2.0 ** -22 * bias
                off = float((off + 2.0 ** -22 * (x.abs() + x.abs().max())).max())
                top = x.max()
                if top == -math.inf:
                    continue
                w = torch.exp(x - top)
                lse[h, t] = top + torch.log(w.sum())
                w = w / w.sum()
                out[t, h] = w @ v
                size = w @ v.abs()
                n = j.numel()
                rel = 2 * off + 2.0 ** -16 + (n / 32 + 64) * 2.0 ** -23
                bound[t, h] = rel * size
                if q.dtype == torch.float16:
                    bound[t, h] += n * 2.0 ** -35 * w.max() * v.abs().amax(0)
                lse_bound[h, t] = off + (n / 32 + 64) * 2.0 ** -23 + 2.0 ** -22 * lse[h, t].abs()
    return out, lse, bound, lse_bound


def sample_row(logits, u, temperature, top_k, top_p, min_p):
    """``(token, logprob, sure, off)`` of one row of float logits, in 64 bits.

    ``off``: the share of the sums by which a kernel's may be off: 2^-43 of each weight, and 2^-41, as they are
    whole numbers of 2^-40.  ``sure``: whether the token is the same with ``top_p`` and ``u`` moved
    by that much either way (equal weights are exact)."""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, -math.inf, True, 0.0
    if not temperature > 0:
        return int(order[0]), 0.0, True, 0.0
    with np.errstate(invalid="ignore"):
        y = np.where(x == top, 0.0, (x - top) / temperature)
    weight = np.exp(y)
    if 0 < top_k < order.size:
        order = order[:top_k]
    run = weight[order]
    total = run.sum()
    off = 2.0 ** -43 + run.size * 2.0 ** -41 / total

    def draw(p, u):
        n = order.size
        if top_p < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(run), p * total, side="left")))
        keep = run[:n] >= min_p
        kept = np.sort(order[:n][keep])
        w = weight[kept]
        upto = np.cumsum(w)
        i = int(np.searchsorted(upto, u * upto[-1], side="right"))
        if i >= kept.size:
            i = int(np.nonzero(w > 0)[0][-1])
        return int(kept[i]), math.log(w[i] / upto[-1])

    token, logprob = draw(top_p, u)
    if np.ptp(run[run > 0]) == 0:
        return token, logprob, True, off
    near = {draw(top_p + a * off, max(0.0, u + b * off) if u > 0 else 0.0)[0] for a in (-1, 0, 1) for b in (-1, 0, 1)}
    return token, logprob, near == {token}, off
