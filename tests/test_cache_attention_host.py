"""Refusals of the scored and shared-prefix attention, before any GPU call (CPU only)."""
import math

import pytest
import torch

from leanselect_amd import _hip
from leanselect_amd.infllm_v2 import infllmv2_attn_with_kvcache
from leanselect_amd.ops import dense_attention_kvcache, shared_prefix_attention

BF16 = torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _kv(*shape, dtype=BF16):
    return torch.zeros(*shape, 2, 128, dtype=dtype)


def _call(**kw):
    a = dict(q=torch.zeros(3, 8, 128, dtype=BF16), kp=_kv(5), vp=_kv(5), k=_kv(2, 9), v=_kv(2, 9), lens=_i32([3, 9]),
             cu=_i32([0, 1, 3]))
    more = {n: o for n, o in kw.items() if n not in a}
    a.update({n: o for n, o in kw.items() if n in a})
    shared_prefix_attention(a["q"], a["kp"], a["vp"], a["k"], a["v"], a["lens"], a["cu"], 9, **more)


def test_well_formed_cpu_arguments_reach_the_device_check():
    for more in (dict(), dict(alibi_slopes=torch.zeros(8)), dict(alibi_slopes=torch.zeros(2, 8)),
                 dict(window=(0, 3), softcap=5.0), dict(kp=_kv(0), vp=_kv(0)),
                 dict(k=_kv(2, 9).transpose(2, 3).contiguous().transpose(2, 3)[:, :, :1],
                      v=_kv(2, 9)[:, :, :1], kp=_kv(5)[:, :1], vp=_kv(5)[:, :1])):
        with pytest.raises((RuntimeError, ValueError), match="GPU|same strides"):
            _call(**more)
    with pytest.raises(RuntimeError, match="GPU"):
        _call()
    with pytest.raises(RuntimeError, match="GPU"):
        dense_attention_kvcache(torch.zeros(3, 8, 128, dtype=BF16), _kv(2, 9), _kv(2, 9), _i32([3, 9]),
                                _i32([0, 1, 3]), 9, softcap=1.0)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(3, 8, 64, dtype=BF16)), "q must be"),
    (dict(q=torch.zeros(3, 8, 128)), "q must be"),
    (dict(q=torch.zeros(3, 8 * 128, dtype=BF16)), "q must be"),
    (dict(q=torch.zeros(3, 7, 128, dtype=BF16)), "multiple of the cache's"),
    (dict(q=torch.zeros(3, 34, 128, dtype=BF16)), "multiple of the cache's"),
    (dict(k=_kv(2, 9, dtype=torch.float16), v=_kv(2, 9, dtype=torch.float16)), "share a dtype"),
    (dict(v=_kv(2, 8)), "k_cache and v_cache"),
    (dict(k=_kv(9), v=_kv(9)), "k_cache and v_cache"),
    (dict(k=_kv(2, 9), v=_kv(9, 2).transpose(0, 1)), "same strides"),
    (dict(k=torch.zeros(2, 9, 2, 132, dtype=BF16)[..., 2:130], v=torch.zeros(2, 9, 2, 132, dtype=BF16)[..., 2:130]),
     "same strides"),
    (dict(kp=_kv(5), vp=_kv(4)), "k_prefix and v_prefix"),
    (dict(kp=_kv(1, 5), vp=_kv(1, 5)), "k_prefix and v_prefix"),
    (dict(kp=_kv(5)[:, :1], vp=_kv(5)[:, :1]), "prefix must be"),
    (dict(kp=_kv(5, dtype=torch.float16), vp=_kv(5, dtype=torch.float16)), "prefix must be"),
    (dict(kp=_kv(10)[::2], vp=_kv(5)), "prefix's rows"),
    (dict(lens=torch.tensor([3, 9])), "int32"),
    (dict(lens=_i32([3])), "int32"),
    (dict(cu=_i32([0, 3])), "int32"),
    (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.nan), "softcap"),
    (dict(softcap=math.inf), "softcap"),
    (dict(softcap=1e-30), "softcap"),
    (dict(softcap=513.0), "softcap"),
    (dict(softmax_scale=0.0), "softmax_scale"),
    (dict(softmax_scale=-0.1), "softmax_scale"),
    (dict(alibi_slopes=torch.zeros(8, dtype=BF16)), "alibi_slopes"),
    (dict(alibi_slopes=torch.zeros(3, 8)), "alibi_slopes"),
    (dict(out=torch.zeros(3, 8, 128)), "out must be"),
    (dict(out=torch.zeros(8, 3, 128, dtype=BF16).transpose(0, 1)), "out must be"),
])
def test_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _call(**change)


def test_options_with_a_plan_are_not_provided():
    q, k = torch.zeros(1, 1, 8, 128, dtype=BF16), _kv(1, 64)
    plan = torch.zeros(2, 1, 1, dtype=torch.int32)
    for more in (dict(softcap=1.0), dict(window_size=(3, -1)), dict(alibi_slopes=torch.zeros(8))):
        with pytest.raises(NotImplementedError, match="topk_idx"):
            infllmv2_attn_with_kvcache(q, k, k, cache_seqlens=_i32([3]), topk_idx=plan, **more)


def _entry(**kw):
    a = dict(q=16, q_rs=1024, cu=16, total=1, kp=None, vp=None, p_rs=0, p_len=0, k=16, v=16, c_bs=0, c_rs=256,
             capacity=8, lens=16, batch=1, H=8, G=2, D=128, dtype=_hip.LS_BF16, max_len=8, scale=0.1, causal=0,
             cap=0.0, slopes=None, s_bs=0, left=-1, right=-1, splits=0, out=16, lse=None, ws=None, nbytes=0,
             stream=None)
    a.update(kw)
    lib = _hip.lib()
    return lib.ls_cache_attn(*a.values()), lib.ls_last_error().decode()


@pytest.mark.parametrize("change,code,match", [
    (dict(batch=0), _hip.LS_ERR_INVALID, "bad sizes"),
    (dict(H=7), _hip.LS_ERR_INVALID, "bad sizes"),
    (dict(p_len=-1), _hip.LS_ERR_INVALID, "bad sizes"),
    (dict(D=64), _hip.LS_ERR_UNSUPPORTED, "head_dim"),
    (dict(H=34), _hip.LS_ERR_UNSUPPORTED, "16 query heads"),
    (dict(dtype=_hip.LS_F32), _hip.LS_ERR_UNSUPPORTED, "bf16 or fp16"),
    (dict(scale=0.0), _hip.LS_ERR_INVALID, "softmax_scale"),
    (dict(cap=-1.0), _hip.LS_ERR_INVALID, "softcap"),
    (dict(cap=1e-30), _hip.LS_ERR_UNSUPPORTED, "softcap"),
    (dict(cap=513.0), _hip.LS_ERR_UNSUPPORTED, "softcap"),
    (dict(splits=129), _hip.LS_ERR_INVALID, "n_splits"),
    (dict(capacity=1 << 30), _hip.LS_ERR_UNSUPPORTED, "2\\^30"),
    (dict(c_rs=1 << 24), _hip.LS_ERR_UNSUPPORTED, "2\\^24"),
    (dict(c_rs=130), _hip.LS_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(q=None), _hip.LS_ERR_INVALID, "null"),
    (dict(p_len=4), _hip.LS_ERR_INVALID, "null"),
    (dict(k=8), _hip.LS_ERR_UNSUPPORTED, "aligned"),
    (dict(splits=4), _hip.LS_ERR_WORKSPACE, "workspace"),
])
def test_entry_point_refusals(change, code, match):
    import re

    rc, message = _entry(**change)
    assert rc == code and re.search(match, message), (rc, message)


def test_no_rows_launch_nothing():
    assert _entry(total=0)[0] == _hip.LS_OK
    lib = _hip.lib()
    assert lib.ls_cache_attn_workspace_size(0, 1, 8, 2, 0, 8, -1, 0) == 0
    assert lib.ls_cache_attn_workspace_size(1, 1, 8, 2, 0, 100, -1, 1) == 0
    assert lib.ls_cache_attn_workspace_size(1, 1, 8, 2, 0, 100, -1, 4) >= 4 * 8 * 4 * 130


def test_refused_options_leave_the_cache():
    """A call with new keys that is refused for its options has not appended them."""
    q, kv, new = torch.zeros(1, 1, 8, 128, dtype=BF16), _kv(1, 64), _kv(1, 1)
    kept = kv.clone()
    for more in (dict(softcap=-1.0), dict(alibi_slopes=torch.zeros(3)), dict(window_size=(3, 0), softmax_scale=-1.0)):
        with pytest.raises(ValueError):
            infllmv2_attn_with_kvcache(q, kv, kv, new, new, cache_seqlens=3, **more)
    assert torch.equal(kv, kept)
