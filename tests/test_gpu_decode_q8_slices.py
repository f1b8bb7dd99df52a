"""Long rows in many slices: the join of more than 64 of them, with lanes and parts that hold none,
one and several, against the 64-bit form."""
import pytest
import torch

from leanselect_amd.ops import dense_attention_kvcache_q8
from oracle import lowbit_oracle as lo
from test_gpu_decode_q8 import D, DEV, _check, _cu, _filled, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slices,n,H", [(64, 16384, 16), (65, 16640, 3), (128, 32750, 16), (129, 33024, 5),
                                        (200, 51190, 8), (256, 65536, 16)])
def test_a_long_row_in_many_slices(dtype, slices, n, H):
    """A page a wave, so ``slices`` slices; a row that ends in its second page (the other slices
    hold nothing), one without a key, and one of a few slices beside it."""
    lens = [n, 100, 0, 1500]
    cache = _filled(lens, 1, dtype, slices)
    ref = lo.Q8Cache(*cache)
    cu = _cu([1, 1, 1, 1])
    q = torch.randn(4, H, D, generator=torch.Generator().manual_seed(n)).to(dtype)
    want, want_lse, bound = lo.attend(ref, q, lens, cu)
    out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), _i32(cu), n, n_splits=slices,
                                          return_lse=True)
    _check(out, lse, want, want_lse, bound, dtype)
    assert bool((out[2] == 0).all()) and bool(torch.isinf(lse[:, 2]).all())


def test_the_slices_of_one_long_row_as_they_are_chosen():
    """One row of one head over 70000 keys: 256 slices, the rows behind it left as they were."""
    n, H = 70000, 16
    cache = _filled([n], 1, torch.bfloat16, 41)
    q = torch.randn(2, H, D, generator=torch.Generator().manual_seed(42)).bfloat16()
    out = torch.full((2, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
    _, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), _i32([0, 1]), n, out=out,
                                        n_splits=256, return_lse=True)
    want, want_lse, bound = lo.attend(lo.Q8Cache(*cache), q, [n], [0, 1])
    _check(out, lse, want, want_lse, bound, torch.bfloat16, slice(0, 1))
    assert bool((out[1] == 3.0).all())
    alone = dense_attention_kvcache_q8(q[:1].to(DEV), *cache, _i32([n]), _i32([0, 1]), n)
    assert torch.equal(alone, out[:1])
