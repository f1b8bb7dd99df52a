"""Attention with biased scores in caches of more than 2^24 keys, against its 64-bit form over the keys in the
window (oracle/serving_oracle.py): a bias goes by the distance, wherever the two stand."""
import pytest
import torch

from leanselect_amd.ops import dense_attention_kvcache, shared_prefix_attention
from oracle import serving_oracle as so
from test_gpu_cache_attention import BF16, D, DEV, _check, _i32, _inputs

pytestmark = pytest.mark.gpu
_FAR = 1 << 24
_SLOPES = torch.tensor([0.8, 0.3, 0.05, 2.0])


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("rows", [1, 70])
def test_a_far_row(odd, rows):
    n, cap = 300, _FAR + 400 + odd
    k = torch.empty(1, cap, 1, D, dtype=BF16, device=DEV)
    v = torch.empty(1, cap, 1, D, dtype=BF16, device=DEV)
    q, ks, vs, _, _ = _inputs([n], [rows], 4, 1, BF16, 21)
    k[0, cap - n:], v[0, cap - n:] = ks[0].to(DEV), vs[0].to(DEV)
    options = dict(causal=True, window=(n - rows, -1))
    got = dense_attention_kvcache(q.to(DEV), k, v, _i32([cap]), _i32([0, rows]), cap, return_lse=True,
                                  alibi_slopes=_SLOPES.to(DEV), **options)
    _check(got, so.cache_attention(q, ks, vs, [n], [0, rows], alibi_slopes=_SLOPES, **options), BF16)


@pytest.mark.parametrize("odd", [0, 1])
def test_behind_a_far_prefix(odd):
    """Some of the keys in the window are the prefix's, some the sequence's own."""
    n, own, P = 300, 100, _FAR + 400 + odd
    kp = torch.empty(P, 1, D, dtype=BF16, device=DEV)
    vp = torch.empty(P, 1, D, dtype=BF16, device=DEV)
    q, ks, vs, _, _ = _inputs([n], [1], 4, 1, BF16, 22)
    kp[P - n + own:], vp[P - n + own:] = ks[0, :n - own].to(DEV), vs[0, :n - own].to(DEV)
    got = shared_prefix_attention(q.to(DEV), kp, vp, ks[:, n - own:].to(DEV), vs[:, n - own:].to(DEV), _i32([own]),
                                  _i32([0, 1]), own, return_lse=True, alibi_slopes=_SLOPES.to(DEV), window=(n - 1, -1))
    _check(got, so.cache_attention(q, ks, vs, [n], [0, 1], alibi_slopes=_SLOPES), BF16)
