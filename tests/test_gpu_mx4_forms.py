"""Every form of the 4-bit products in both types: which one a size takes is ``mx4_cut``'s choice
in csrc/ls_mx4.hip, named beside it (waves and tiles of the weight a workgroup, or shared rows of x
in blocks of 16 and the slices of the inputs)."""
import pytest
import torch

from leanselect_amd.ops import linear_mx4, linear_mx4_silu_mul
from test_gpu_mx4 import DEV, _check, _values

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])


def _rows(m, k, dtype):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(m + k)).to(dtype)


@TYPES
@pytest.mark.parametrize("n,k,m", [
    (40, 520, 3), (200, 136, 20),                    # eight waves, one tile; 17 to 32 rows of them
    (4624, 264, 9), (4608, 1032, 17),                # eight waves, two tiles
    (4620, 4096, 32),
    (32790, 520, 1), (33000, 136, 16),               # four waves, four tiles
    (20480, 520, 16), (20480, 264, 20),              # shared rows: one block of 16, two
    (20488, 264, 40), (20470, 264, 60),              # three, four
    (100, 12296, 15), (40, 4104, 20),                # the same in slices
    (2048, 8192, 40), (2048, 2056, 130)])
def test_linear(dtype, n, k, m):
    (codes, scales), w = _values(n, k, n + k + m)
    x = _rows(m, k, dtype)
    _check(linear_mx4(x.to(DEV), codes, scales, n), x, w)


@TYPES
@pytest.mark.parametrize("n,k,m", [
    (64, 136, 3), (64, 136, 20),                     # eight waves, a tile and its other half
    (33024, 72, 1), (33024, 520, 7),                 # four waves, two and two
    (20480, 520, 1), (20480, 264, 20),               # shared rows: one block of 16, two
    (20480, 520, 32), (20480, 520, 40),              # two, three
    (20480, 264, 50), (20512, 264, 130),             # four
    (2048, 16392, 5), (512, 4104, 17),               # the same in slices
    (2048, 8200, 33), (2048, 2056, 200)])
def test_silu_mul(dtype, n, k, m):
    (codes, scales), w = _values(n, k, n + 2 * k + m, 112, 120)
    x = _rows(m, k, dtype)
    _check(linear_mx4_silu_mul(x.to(DEV), codes, scales, n), x, w, silu=True)
