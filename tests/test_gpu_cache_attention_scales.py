"""Capped scores under scales whose ratio to the cap float32 does not hold: the cap's ends and its middle."""
import pytest
import torch

from leanselect_amd.ops import dense_attention_kvcache
from test_gpu_cache_attention import BF16, FP16, D, DEV, _i32, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("scale,cap", [(1e20, 1e-20), (3e38, 1e-3), (3e38, 512.0), (1e-45, 512.0), (1e-40, 0.5), (1e-30, 1e-20)])
def test_scales_far_from_the_cap(dtype, rows, scale, cap):
    n = 200
    q, k, v, _, _ = _inputs([n], [rows], 4, 2, dtype, 31)
    q[0, :2] = 0.0  # products of 0 stay 0 under any scale
    out, lse = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32([n]), _i32([0, rows]), n, softcap=cap,
                                       softmax_scale=scale, return_lse=True)
    kd, vd = (t[0].double().repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))  # [H, n, D]
    x = cap * torch.tanh((q.double().transpose(0, 1) @ kd.transpose(1, 2)) * scale / cap)
    w = torch.softmax(x, -1)
    exact, size = (w @ vd).transpose(0, 1), (w @ vd.abs()).transpose(0, 1)
    # A capped score is off by cap 2^-20, a weight by that and 2^-16 (in fp16 2^-35 of the largest: less), sums by 2^-23
    # for each of n / 32 + 64 additions; then the output's rounding.
    off = cap * 2.0 ** -20
    bound = (2 * off + 2.0 ** -16 + (n / 32 + 64) * 2.0 ** -23) * size
    allowed = torch.finfo(dtype).eps / 2 * (exact.abs() + bound) + bound + (2.0 ** -25 if dtype == FP16 else 0.0)
    assert bool(((out.cpu().double() - exact).abs() <= allowed).all())
    want = torch.logsumexp(x, -1)
    lse_off = off + (n / 32 + 64) * 2.0 ** -23 + 2.0 ** -22 * (want.abs() + cap)
    assert bool(((lse.cpu().double() - want).abs() <= lse_off).all())
