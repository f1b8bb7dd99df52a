"""Calls with new keys and options that the attention does not take are refused before the keys are appended (here: with
ValueError, not by the append, which wants a GPU)."""
import pytest
import torch

from leanselect_amd.infllm_v2 import infllmv2_attn_with_kvcache

BF16 = torch.bfloat16


def _call(H=8, G=2, D=128, kv=None, **kw):
    q, new = torch.zeros(1, 1, H, D, dtype=BF16), torch.zeros(1, 1, G, D, dtype=BF16)
    k, v = kv or (torch.zeros(1, 64, G, D, dtype=BF16),) * 2
    infllmv2_attn_with_kvcache(q, k, v, new, new, cache_seqlens=3, **{"softcap": 5.0, **kw})


@pytest.mark.parametrize("change,match", [
    (dict(D=64), "128"), (dict(H=34), "at most 16"), (dict(H=7), "multiple"), (dict(softmax_scale=1e-50), "softmax_scale"),
    (dict(softmax_scale=1e39), "softmax_scale"), (dict(window_size=(3, 3, 3)), "unpack"), (dict(window_size=(3,)), "unpack"),
    (dict(kv=(torch.zeros(1, 64, 2, 130, dtype=BF16)[..., :128],) * 2), "dense"),
    (dict(kv=(torch.zeros(1 + 64 * 256, dtype=BF16)[1:].view(1, 64, 2, 128),) * 2), "aligned"),
    (dict(kv=(torch.zeros(1, dtype=BF16).expand(1, 1 << 30, 2, 128),) * 2), "2\\^30")], ids=lambda x: None)
def test_refused_before_the_append(change, match):
    with pytest.raises(ValueError, match=match):
        _call(**change)


def test_what_is_taken_reaches_the_device_check():
    with pytest.raises(RuntimeError, match="GPU"):
        _call()
    with pytest.raises(RuntimeError, match="GPU"):
        _call(softcap=0.0, window_size=[3, -1])
