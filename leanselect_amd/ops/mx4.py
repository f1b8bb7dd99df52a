"""Products of a few rows with 4-bit weights, on the GPU.

A weight ``[out_features, in_features]`` is held as E2M1 values (0, 0.5, 1, 1.5, 2,
3, 4, 6 and their negatives) with one power-of-two scale for every 32 inputs of an
output, laid out once by ``quantize_mx4`` (or ``lay_out_mx4`` from a checkpoint's
values) in the order the kernel reads:

- ``codes`` uint8 ``[ceil(out / 16), ceil(in / 128), 64, 16]``: tiles of 16 outputs by
  128 inputs; lane ``16 q + r`` holds inputs ``32 q`` to ``32 q + 31`` of output ``r``, the
  even input in a byte's low half;
- ``scales`` uint8 ``[ceil(out / 16), ceil(in / 512), 64, 4]``: the same lanes, byte ``i``
  for the ``i``-th of four tiles; code ``c`` in 8..252 stands for ``2 ** (c - 127)``.

Sizes are padded with value 0 and scale 1.  ``linear_mx4`` multiplies rows of bf16 or
fp16 with the values in that type (exact in bf16; in fp16 exact for codes 104 to 140,
rounded and at most infinite outside), sums in float32 and rounds once.

No counterpart in the reference, whose projections are 16-bit.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from .. import _hip

_CODES = {torch.bfloat16: _hip.LS_BF16, torch.float16: _hip.LS_F16}

__all__ = ["quantize_mx4", "lay_out_mx4", "dequantize_mx4", "linear_mx4", "linear_mx4_silu_mul"]


@lru_cache(maxsize=4096)
def _shapes(out_features: int, in_features: int) -> tuple[tuple, tuple]:
    if out_features < 1 or in_features < 8 or in_features % 8:
        raise ValueError(f"need out_features >= 1 and in_features a multiple of 8 "
                         f"(got {out_features} x {in_features})")
    nt, kc = (out_features + 15) // 16, (in_features + 127) // 128
    return (nt, kc, 64, 16), (nt, (kc + 3) // 4, 64, 4)


def _check_weight(codes, scales, out_features: int, in_features: int) -> None:
    cs, ss = _shapes(out_features, in_features)
    if codes.shape != cs or scales.shape != ss or codes.dtype is not torch.uint8 \
            or scales.dtype is not torch.uint8 or not codes.is_contiguous() \
            or not scales.is_contiguous():
        raise ValueError(f"a {out_features} x {in_features} weight needs contiguous uint8 codes "
                         f"{cs} and scales {ss} (got {tuple(codes.shape)} and "
                         f"{tuple(scales.shape)})")


def quantize_mx4(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``weight [out_features, in_features]`` (float32, bf16 or fp16;
    finite).  A group's scale is the least power of two, from 2^-119, under which none of its
    values exceeds 6 (1 for a group of zeros), and at most 2^125, whose 6 is the last product
    that bf16 holds (larger magnitudes become that); values go to the nearest E2M1 value, ties
    to the even code.  Reads the weight's finiteness on the host (laying out is done once)."""
    if weight.ndim != 2 or weight.stride(1) != 1 and weight.shape[1] > 1:
        raise ValueError("weight must be [out_features, in_features] with unit column stride")
    n, k = weight.shape
    cs, ss = _shapes(n, k)
    code = _hip.dtype_code(weight.dtype)
    index = _hip.gpu_index(weight)
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("weight must be finite: E2M1 has no infinity and no NaN")
    codes = torch.empty(cs, dtype=torch.uint8, device=weight.device)
    scales = torch.empty(ss, dtype=torch.uint8, device=weight.device)
    _hip.launch(index, "ls_quantize_mx4", weight.data_ptr(), weight.stride(0), n, k, code,
                codes.data_ptr(), scales.data_ptr())
    return codes, scales


def lay_out_mx4(values: torch.Tensor, scale_codes: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` in the kernel's order from 4-bit values ``uint8 [out_features,
    in_features]`` (0..15: sign, two exponent bits, one mantissa bit) and scale codes ``uint8
    [out_features, ceil(in_features / 32)]`` in 8..252."""
    if values.ndim != 2 or values.dtype != torch.uint8 or scale_codes.dtype != torch.uint8:
        raise ValueError("values and scale_codes must be uint8, values [out_features, in_features]")
    n, k = values.shape
    cs, ss = _shapes(n, k)
    if scale_codes.shape != (n, -(-k // 32)) or scale_codes.device != values.device:
        raise ValueError(f"scale_codes must be [{n}, {-(-k // 32)}] on {values.device}")
    if bool((values > 15).any()) or bool(((scale_codes < 8) | (scale_codes > 252)).any()):
        raise ValueError("values must be 0..15 and scale codes 8..252")
    full = values.new_zeros(cs[0] * 16, cs[1] * 128)
    full[:n, :k] = values
    packed = (full[:, 0::2] | full[:, 1::2] << 4).view(cs[0], 16, cs[1], 4, 16)
    s = values.new_full((cs[0] * 16, ss[1] * 16), 127)
    s[:n, :scale_codes.shape[1]] = scale_codes
    s = s.view(cs[0], 16, ss[1], 4, 4)
    return (packed.permute(0, 2, 3, 1, 4).reshape(cs).contiguous(),
            s.permute(0, 2, 4, 1, 3).reshape(ss).contiguous())


def dequantize_mx4(codes: torch.Tensor, scales: torch.Tensor, out_features: int, in_features: int,
                   dtype: torch.dtype = torch.bfloat16,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The weight's values ``[out_features, in_features]`` in bf16 (exact) or fp16 (rounded)."""
    _check_weight(codes, scales, out_features, in_features)
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("the values are given in bf16 or fp16")
    index = _hip.gpu_index(codes, scales)
    if out is None:
        out = torch.empty((out_features, in_features), dtype=dtype, device=codes.device)
    else:
        _hip.check_out(out, (out_features, in_features), dtype, codes.device)
    _hip.launch(index, "ls_dequantize_mx4", codes.data_ptr(), scales.data_ptr(), out_features,
                in_features, _hip.dtype_code(dtype), out.data_ptr(), in_features)
    return out


def linear_mx4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out_features: int, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T`` for ``x [rows, in_features]`` (bf16 or fp16): ``[rows, out_features]`` in
    ``x``'s dtype.  Made for the few rows of a decode step; every 64 rows read the weight
    again.  ``out`` must not overlap ``x`` (rows of one buffer side by side do not).  A row's
    bits do not depend on what the other rows hold, but may on how many there are.  No gradient
    passes."""
    return _linear(x, codes, scales, out_features, 0, out)


def linear_mx4_silu_mul(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                        out_features: int, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x @ gate.T) * (x @ up.T)`` for a weight ``[gate; up]`` of ``out_features`` rows in
    all (a multiple of 32): ``[rows, out_features / 2]``, float32 up to the one rounding."""
    if out_features % 32:
        raise ValueError(f"out_features must be a multiple of 32 (got {out_features})")
    return _linear(x, codes, scales, out_features, 1, out)


@lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, k: int, out_features: int, silu: int) -> int:
    return _hip.lib().ls_linear_mx4_workspace_size(rows, k, out_features, silu)


def _linear(x, codes, scales, out_features, silu, out):
    dtype, shape = x.dtype, x.shape
    code = _CODES.get(dtype)
    if code is None or len(shape) != 2:
        raise ValueError("x must be bf16 or fp16 [rows, in_features]")
    rows, k = shape
    _check_weight(codes, scales, out_features, k)
    n = out_features // 2 if silu else out_features
    index = _hip.gpu_index(x, codes, scales, out)
    given = out is not None
    if not given:
        out = x.new_empty((rows, n))
        out_stride = n
    else:
        if out.shape != (rows, n) or out.stride(1) != 1 or out.dtype is not dtype:
            raise ValueError(f"out must be ({rows}, {n}) {x.dtype} with unit column stride, "
                             f"got {tuple(out.shape)} {out.dtype}")
        out_stride = out.stride(0)
        if rows > 1 and out_stride < n or out.data_ptr() == x.data_ptr() and rows:
            raise ValueError("out's rows must not overlap each other or x")
    x_stride, x_ptr = x.stride(), x.data_ptr()
    if x_ptr & 15 or x_stride[1] != 1 or x_stride[0] & 7:  # rows the kernels do not read
        x = x.clone(memory_format=torch.contiguous_format)
        x_stride, x_ptr = (k,), x.data_ptr()
    elif given and _hip.rows_overlap(out.data_ptr(), 2 * out_stride, rows, 2 * n, x_ptr,
                                       2 * x_stride[0], rows if x_stride[0] else 1, 2 * k):
        raise ValueError("out's rows must not overlap each other or x")
    nbytes = _workspace_bytes(rows, k, out_features, silu)
    ws = x.new_empty((nbytes + 1) >> 1) if nbytes else None  # counted in x's 16-bit elements
    _hip.launch(index, "ls_linear_mx4", x_ptr, x_stride[0], rows, k, codes.data_ptr(),
                scales.data_ptr(), out_features, silu, code, out.data_ptr(), out_stride,
                ws.data_ptr() if nbytes else None, nbytes)
    return out
