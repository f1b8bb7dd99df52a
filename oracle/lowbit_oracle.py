"""Plain CPU forms, in 64 bits, of decoding in 8 and 4 bits: the e4m3 cache append,
attention over the cache and products with E2M1 weights.  Layouts and rules are
written out here from their definitions; nothing is shared with the kernels.
"""
from __future__ import annotations

import math

import torch

PAGE, D = 64, 128
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def e4m3_values() -> torch.Tensor:
    """The 127 finite e4m3 magnitudes, by code: 0, seven subnormals of 2^-9, then 1.m 2^(e-7)."""
    v = [m * 2.0 ** -9 for m in range(8)]
    v += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64)


def _nearest(y: torch.Tensor, values: torch.Tensor) -> torch.Tensor:
    """Code (index) of the nearest of ascending ``values`` to ``y >= 0``, ties to the even code."""
    middle = (values[1:] + values[:-1]) / 2
    low = torch.searchsorted(middle, y.contiguous())
    tie = (low < len(middle)) & (middle[low.clamp(max=len(middle) - 1)] == y)
    return low + (tie & (low % 2 == 1)).long()


def e4m3_round(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value; non-finite becomes NaN (callers keep |y| <= 448)."""
    values = e4m3_values()
    ok = torch.isfinite(y)
    z = torch.where(ok, y, 0.0).double()
    return torch.where(ok, torch.copysign(values[_nearest(z.abs(), values)], z), math.nan)


def scale_code(top: float, largest: float, low: int) -> int:
    """The least c >= low with top <= largest * 2^(c - 127)."""
    c = low
    while top > largest * 2.0 ** (c - 127):
        c += 1
    return c


def place(token: int) -> int:
    """Where a page's value of this token lies among its channel's 64."""
    t, q, i = token // 16, token // 4 % 4, token % 4
    return 16 * q + 4 * t + i


class Q8Cache:
    """The values and codes of an 8-bit cache, by token: ``k, v [B, P, G, 64, 128]`` float64
    e4m3 values (unscaled), ``kcode, vcode [B, P, G]``."""

    def __init__(self, k8, v8, k_scale, v_scale):
        order = torch.tensor([place(t) for t in range(PAGE)])
        self.k = k8.cpu().double()
        self.v = v8.cpu().double()[..., order].transpose(-1, -2).contiguous()
        self.kcode, self.vcode = k_scale.cpu().long(), v_scale.cpu().long()

    def append(self, lens, k_new, v_new, cu):
        for x, code, new in ((self.k, self.kcode, k_new), (self.v, self.vcode, v_new)):
            new = new.cpu().double()
            for b, before in enumerate(lens):
                n = cu[b + 1] - cu[b]
                for p in range(before // PAGE, -(-(before + n) // PAGE) if n else 0):
                    lo, hi = max(before, p * PAGE), min(before + n, p * PAGE + PAGE)
                    rows = new[cu[b] + lo - before:cu[b] + hi - before]  # [rows, G, D]
                    for g in range(rows.shape[1]):
                        r = rows[:, g]
                        finite = r[torch.isfinite(r)]
                        top = float(finite.abs().max()) if finite.numel() else 0.0
                        c = scale_code(top, 448.0, 1)
                        old = int(code[b, p, g])
                        held = lo - p * PAGE
                        if held:
                            c = max(c, old)
                            x[b, p, g, :held] = e4m3_round(x[b, p, g, :held] * 2.0 ** (old - c))
                        x[b, p, g, held:hi - p * PAGE] = e4m3_round(r * 2.0 ** (127 - c))
                        code[b, p, g] = c

    def keys(self, b, g):
        """``[P * 64, 128]`` the values the cache stands for."""
        return self._values(self.k, self.kcode, b, g)

    def values(self, b, g):
        return self._values(self.v, self.vcode, b, g)

    @staticmethod
    def _values(x, code, b, g):
        return (x[b, :, g] * (2.0 ** (code[b, :, g].double() - 127))[:, None, None]).reshape(-1, D)

    def window(self, b, g, w):
        return self.keys(b, g)[16 * w:16 * w + 32].mean(0)


def attend(cache: Q8Cache, q, lens, cu_q, ids=None, causal=False, scale=None):
    """``(out, lse, bound)`` of decode rows over the cache; rows past ``cu_q[-1]`` NaN.

    ``bound`` is what the kernel's own roundings may move an output by, before its rounding
    to 16 bits: weights held as an fp16 head and remainder (2^-22 of each, or 2^-40 of the
    largest where either is subnormal), scores formed in float32, and float32 sums (a page
    of 64 keys an addition, the joins' beside)."""
    total, H, _ = q.shape
    G = cache.k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((total, H, D), math.nan, dtype=torch.float64)
    lse = torch.full((H, total), math.nan, dtype=torch.float64)
    bound = torch.zeros(total, H, D, dtype=torch.float64)
    for b, n in enumerate(lens):
        for t in range(cu_q[b], cu_q[b + 1]):
            limit = n - (cu_q[b + 1] - cu_q[b]) + (t - cu_q[b]) + 1 if causal else n
            for g in range(G):
                if ids is None:
                    keep = list(range(max(0, limit)))
                else:
                    plan = {int(p) for p in ids[g, t] if p >= 0}
                    keep = [j for p in sorted(plan) for j in range(PAGE * p, min(PAGE * p + PAGE, limit))]
                rows = slice(g * (H // G), (g + 1) * (H // G))
                if not keep:
                    out[t, rows], lse[rows, t] = 0.0, math.inf
                    continue
                k, v = cache.keys(b, g)[keep], cache.values(b, g)[keep]
                x = q[t, rows].double()
                s = x @ k.t() * scale
                p = torch.softmax(s, -1)
                out[t, rows] = p @ v
                lse[rows, t] = torch.logsumexp(s, -1)
                size = (x.abs() @ k.abs().t() * abs(scale)).amax(-1, keepdim=True)
                e = 2.0 ** -22 + 2.0 ** -17 * size + 2.0 ** -22 * (1 + s.abs().amax(-1, keepdim=True)) \
                    + 2.0 ** -24 * (len(keep) / PAGE + PAGE)
                lost = 2 * len(keep) * 2.0 ** -40 * p.amax(-1, keepdim=True)
                bound[t, rows] = 2 * e * (p @ v.abs()) + lost * v.abs().amax(0)
    return out, lse, bound


def e2m1_codes(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values 0..15 [N, K], scale codes [N, ceil(K / 32)])`` of a weight.  Codes end at 252
    (6 * 2^125 is the last product bf16 holds): magnitudes above it saturate."""
    n, k = weight.shape
    w = torch.nn.functional.pad(weight.double(), (0, -k % 32)).view(n, -1, 32)
    top = w.abs().amax(-1)
    codes = torch.tensor([[127 if t == 0 else min(252, scale_code(t, 6.0, 8)) for t in row]
                          for row in top.tolist()])
    y = w * (2.0 ** (127 - codes.double()))[..., None]
    mag = _nearest(y.abs(), torch.tensor(E2M1, dtype=torch.float64))
    mag = mag | (torch.signbit(w).long() << 3)
    return mag.view(n, -1)[:, :k].to(torch.uint8), codes.to(torch.uint8)


def e2m1_weight(values: torch.Tensor, codes: torch.Tensor) -> torch.Tensor:
    """The float64 weight of values 0..15 and scale codes."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float64)
    per_input = (2.0 ** (codes.double() - 127)).repeat_interleave(32, 1)[:, :values.shape[1]]
    return table[values.long()] * per_input


def tile_bytes(values: torch.Tensor, codes: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The kernel's order, one element at a time."""
    n, k = values.shape
    nt, kc = -(-n // 16), -(-k // 128)
    kc4 = -(-kc // 4)
    out = torch.zeros(nt, kc, 64, 16, dtype=torch.uint8)
    scales = torch.full((nt, kc4, 64, 4), 127, dtype=torch.uint8)
    for row in range(n):
        for col in range(k):
            lane = 16 * (col % 128 // 32) + row % 16
            out[row // 16, col // 128, lane, col % 32 // 2] |= int(values[row, col]) << 4 * (col % 2)
        for group in range(codes.shape[1]):
            lane = 16 * (group % 4) + row % 16
            scales[row // 16, group // 16, lane, group // 4 % 4] = codes[row, group]
    return out, scales
