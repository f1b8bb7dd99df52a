"""4-bit weights laid out from a checkpoint's values and scale codes (torch operations: CPU)."""
import pytest
import torch

from leanselect_amd.ops import lay_out_mx4
from oracle import lowbit_oracle as lo


def _checkpoint(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    values = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    values[:, ::32] |= 1  # no group of zeros
    return values, torch.randint(8, 253, (n, -(-k // 32)), generator=g, dtype=torch.uint8)


@pytest.mark.parametrize("n,k", [(1, 8), (17, 136), (33, 1048)])
@pytest.mark.parametrize("code", [0, 1, 7, 253, 254])
def test_a_group_of_zeros_may_have_any_scale(n, k, code):
    values, codes = _checkpoint(n, k, n + k)
    groups = codes.shape[1]
    for row, group in ((0, 0), (n - 1, groups - 1), (n // 2, groups // 2)):
        at = slice(32 * group, 32 * group + 32)
        values[row, at] = values[row, at] & 8  # zeros of either sign
        codes[row, group] = code
    got = lay_out_mx4(values, codes)
    for row, group in ((0, 0), (n - 1, groups - 1), (n // 2, groups // 2)):
        codes[row, group] = 127
    want = lo.tile_bytes(values, codes)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("code", [0, 7, 253, 254, 255])
def test_scales_that_the_kernels_do_not_hold_are_refused(code):
    values, codes = _checkpoint(5, 72, 1)
    codes[2, 1] = code
    with pytest.raises(ValueError, match="scale codes"):
        lay_out_mx4(values, codes)
    values[2, 32:64] = 0
    if code == 255:  # not a number, of zeros too
        with pytest.raises(ValueError, match="scale codes"):
            lay_out_mx4(values, codes)
    else:
        lay_out_mx4(values, codes)


def test_its_arguments_are_left_as_they_are():
    values, codes = _checkpoint(5, 72, 2)
    values[0], codes[0] = 0, 0
    before = values.clone(), codes.clone()
    lay_out_mx4(values, codes)
    assert torch.equal(values, before[0]) and torch.equal(codes, before[1])
