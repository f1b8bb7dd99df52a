"""A refused call with new keys and options leaves the cache as it was."""
import pytest
import torch

from leanselect_amd.infllm_v2 import infllmv2_attn_with_kvcache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("H,G,D,options", [
    (8, 2, 64, dict(softcap=5.0)), (17, 1, 128, dict(softcap=5.0)), (8, 2, 128, dict(window_size=(1, 2, 3))),
    (8, 2, 128, dict(softcap=5.0, softmax_scale=1e-50)), (8, 2, 128, dict(alibi_slopes=torch.ones(8)))], ids=str)
def test_nothing_is_appended(H, G, D, options):
    q, new = (torch.ones(2, 1, n, D, dtype=torch.bfloat16, device=DEV) for n in (H, G))
    k, v = (torch.zeros(2, 64, G, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    with pytest.raises((ValueError, RuntimeError)):
        infllmv2_attn_with_kvcache(q, k, v, new, new, cache_seqlens=5, **options)
    assert not bool(k.any()) and not bool(v.any())
