"""What the softmax weights of the 8-bit cache's attention hold, on the GPU: scores that are exact
in float32 (one channel, powers of two and small e4m3 values), so that the outputs show the weights."""
import pytest
import torch

from leanselect_amd.ops import (dense_attention_kvcache_q8, kvcache_append_q8,
                                sparse_attention_kvcache_q8)
from oracle import lowbit_oracle as lo
from test_gpu_decode_q8 import D, DEV, _check, _garbage, _i32

pytestmark = pytest.mark.gpu


def _one_channel_keys(values, v, dtype):
    """A cache of one sequence: key j is ``values[j]`` in channel 0 (each exact in e4m3 under its
    page's scale), value j is ``v[j]``."""
    n, G = len(values), 1
    k = torch.zeros(n, G, D)
    k[:, 0, 0] = values
    cache = _garbage(1, n, G, 1)
    kvcache_append_q8(*cache, _i32([0]), k.to(dtype).to(DEV), v.to(dtype).to(DEV), _i32([0, n]))
    ref = lo.Q8Cache(*cache)
    assert torch.equal(ref.keys(0, 0)[:n, 0], values.double())
    assert torch.equal(ref.values(0, 0)[:n], v[:, 0].double())
    return cache, ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,first,second", [(2, 0, 1), (300, 0, 299), (300, 250, 3), (1000, 64, 700)])
def test_two_values_that_nearly_cancel(dtype, n, first, second):
    """Weights 1 and e^-x of values of opposite signs (the other keys' are 0): where the values nearly
    cancel, the output's own rounding is small and the weights' shows."""
    rows, H = 8, 16
    keys = torch.zeros(n)
    keys[second] = -1.0
    v = torch.zeros(n, 1, D)
    c = torch.arange(D)
    v[first, 0] = 1 + c % 8 / 8.0
    v[second, 0] = -(1 + c // 8 % 8 / 8.0) * (1 + c // 64)
    cache, ref = _one_channel_keys(keys, v, dtype)
    q = torch.zeros(rows, H, D)
    q[..., 0] = (1 + torch.arange(rows * H).view(rows, H)) / 256.0
    q = q.to(dtype)
    want, want_lse, bound = lo.attend(ref, q, [n], [0, rows], scale=1.0)
    # About a hundred outputs of each kind are so small that a half step of theirs is below 2^-16.
    assert int((want.abs() * (n / 2) < 2.0 ** -8).sum()) > 100
    ids = torch.arange(16, dtype=torch.int32, device=DEV).expand(1, rows, 16).contiguous()
    for n_splits in (1, 3, None):
        out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), _i32([0, rows]), n,
                                              softmax_scale=1.0, n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)
        assert bool(((lse.cpu().double() - want_lse).abs() <= 2.0 ** -16 * (1 + want_lse.abs())).all())
        out, lse = sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), ids, _i32([0, rows]),
                                               softmax_scale=1.0, n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [0, 700, 16383])
def test_many_keys_far_below_one(dtype, at):
    """A key that draws nearly all the weight and whose value is 0, among 16383 keys 20 to 30 bits
    below it: the output is theirs alone, so what is lost of their weights is lost of it."""
    n, H = 16384, 16
    keys = torch.zeros(n)
    keys[at] = 20.0
    g = torch.Generator().manual_seed(40)
    v = (torch.randint(8, 16, (n, 1, D), generator=g) / 8.0)
    v[at] = 0.0
    cache, ref = _one_channel_keys(keys, v, dtype)
    q = torch.zeros(1, H, D)
    q[0, :, 0] = (88 + 3 * torch.arange(H)) / 128.0  # scores of 13.75 to 20.8
    q = q.to(dtype)
    want, want_lse, bound = lo.attend(ref, q, [n], [0, 1], scale=1.0)
    ids = torch.arange(256, dtype=torch.int32, device=DEV).view(1, 1, 256)
    for n_splits in (1, 7, None):
        out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), _i32([0, 1]), n,
                                              softmax_scale=1.0, n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)
        out, lse = sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), ids, _i32([0, 1]),
                                               softmax_scale=1.0, n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)
