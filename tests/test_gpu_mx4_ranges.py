"""4-bit products at the ends of their types' ranges, on the GPU."""
import pytest
import torch

from leanselect_amd.ops import lay_out_mx4, linear_mx4, linear_mx4_silu_mul
from oracle import lowbit_oracle as lo
from test_gpu_mx4 import DEV, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("silu,n,k,m", [
    (False, 16640, 512, 1), (False, 16640, 1536, 5), (False, 48, 8704, 33), (False, 48, 9728, 17),
    (True, 20480, 512, 1), (True, 2048, 8704, 33)])
def test_fp16_weights_near_the_largest_stay_finite(silu, n, k, m):
    """Sums of 512 inputs of which the first three quarters have code 141 and values up to 3 (49152
    in fp16) and the last a small code and values up to 6: every weight is finite in fp16, but a
    value of the last under a scale of the first would not be, and no product may meet one, not
    even as a padding whose rows of x are zero."""
    g = torch.Generator().manual_seed(n + k + m)
    values = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    low = torch.arange(k) % 512 < 384
    values[:, low] = values[:, low] % 6 | values[:, low] & 8
    codes = torch.randint(104, 111, (n, k // 32), generator=g, dtype=torch.uint8)
    codes[:, low[::32]] = 141
    laid, w = lay_out_mx4(values.to(DEV), codes.to(DEV)), lo.e2m1_weight(values, codes)
    assert torch.equal(w.half().double(), w)
    spread = 2.0 ** (-14 if silu else -10) / (k / 512) ** 0.5
    x = (torch.randn(m, k, generator=g) * spread).half()
    product = linear_mx4_silu_mul if silu else linear_mx4
    got = product(x.to(DEV), *laid, n)
    assert bool(torch.isfinite(got).all())
    _check(got, x, w, silu=silu)
