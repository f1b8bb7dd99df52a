"""Refusals of the 8-bit cache and the 4-bit products, before any GPU call, and what their
wrappers hand to the library (CPU only)."""
import contextlib
import ctypes

import pytest
import torch

from leanselect_amd import _hip, ops
from leanselect_amd.cache import LeanSelectKVCache
from leanselect_amd.minicpm import MiniCPMConfig, MiniCPMLeanSelect
from leanselect_amd.ops import (dense_attention_kvcache_q8, kvcache_append_q8, linear_mx4,
                                linear_mx4_silu_mul, new_kvcache_q8, quantize_mx4,
                                sparse_attention_kvcache_q8)

BF16 = torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _append(**kw):
    cache = list(new_kvcache_q8(2, 128, 2, device="cpu"))
    a = dict(cache=cache, lens=_i32([3, 0]), k=torch.zeros(4, 2, 128, dtype=BF16),
             v=torch.zeros(4, 2, 128, dtype=BF16), cu=_i32([0, 1, 4]))
    more = {k: v for k, v in kw.items() if k not in a}
    a.update({k: v for k, v in kw.items() if k in a})
    kvcache_append_q8(*a["cache"], a["lens"], a["k"], a["v"], a["cu"], **more)


def test_well_formed_cpu_arguments_reach_the_device_check():
    with pytest.raises(RuntimeError, match="GPU"):
        _append()
    with pytest.raises(RuntimeError, match="GPU"):
        _append(kc_cache=torch.zeros(2, 7, 2, 128, dtype=BF16))


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(4, 3, 128, dtype=BF16)), "k_new and v_new"),
    (dict(k=torch.zeros(4, 2, 64, dtype=BF16), v=torch.zeros(4, 2, 64, dtype=BF16)), "k_new and v_new"),
    (dict(k=torch.zeros(4, 2, 128), v=torch.zeros(4, 2, 128)), "bf16 or fp16"),
    (dict(v=torch.zeros(4, 2, 128, dtype=torch.float16)), "alike"),
    (dict(lens=torch.tensor([3, 0])), "int32"),
    (dict(lens=_i32([3])), "offsets"),
    (dict(cu=_i32([0, 1, 3])), "offsets"),
    (dict(cu=_i32([1, 1, 4])), "offsets"),
    (dict(cu=_i32([0, 4])), "offsets"),
    (dict(cu=_i32([0, 5, 4])), "capacity"),
    (dict(lens=_i32([3, 126])), "capacity"),
    (dict(lens=_i32([-1, 0])), "capacity"),
    (dict(cache_seqlens_host=[3, 0, 0]), "offsets"),
    (dict(cache=[t[:0] for t in new_kvcache_q8(1, 64, 2, device="cpu")], lens=_i32([]), cu=_i32([4])),
     "offsets"),
    (dict(cache=[t.expand(2, *t.shape[1:]) for t in new_kvcache_q8(1, 128, 2, device="cpu")]),
     "share pages"),
    (dict(kc_cache=torch.zeros(1, 7, 2, 128, dtype=BF16).expand(2, 7, 2, 128)), "share pages or windows"),
    (dict(kc_cache=torch.zeros(2, 7, 2, 128)), "kc_cache"),
    (dict(kc_cache=torch.zeros(2, 7, 2, 64, dtype=BF16)), "kc_cache"),
    (dict(lens=_i32([100, 0]), kc_cache=torch.zeros(2, 4, 2, 128, dtype=BF16)), "kc_capacity"),
    (dict(kc_cache=torch.zeros(2, 7, 2, 128, dtype=BF16), kernel_size=64), "windows of 32"),
])
def test_append_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _append(**change)


def _bad_caches():
    k8, v8, ks, vs = new_kvcache_q8(2, 128, 2, device="cpu")
    return [
        ((k8.view(torch.uint8), v8, ks, vs), "the cache must be"),
        ((k8[..., :64], v8, ks, vs), "the cache must be"),
        ((k8, k8, ks, vs), "the cache must be"),
        ((k8, v8, ks.int(), vs), "the cache must be"),
        ((k8, v8, ks[:, :1], vs), "the cache must be"),
        ((k8.transpose(1, 2), v8, ks, vs), "dense"),
        ((k8, v8, ks, vs.transpose(1, 2).contiguous().transpose(1, 2)), "dense"),
        ((torch.cat([k8, k8])[::2], v8, ks, vs), "batch strides"),
    ]


@pytest.mark.parametrize("i", range(8))
def test_malformed_caches(i):
    cache, match = _bad_caches()[i]
    with pytest.raises(ValueError, match=match):
        _append(cache=cache)
    q = torch.zeros(2, 32, 128, dtype=BF16)
    with pytest.raises(ValueError, match=match):
        dense_attention_kvcache_q8(q, *cache, _i32([3, 3]), _i32([0, 1, 2]), 3)


@pytest.mark.parametrize("q,match", [
    (torch.zeros(2, 32, 64, dtype=BF16), "q must"),
    (torch.zeros(2, 33, 128, dtype=BF16), "q must"),
    (torch.zeros(2, 34, 128, dtype=BF16), "16 times"),
    (torch.zeros(2, 32, 128), "q must"),
    (torch.zeros(32, 128, dtype=BF16), "q must"),
])
def test_attention_refuses_queries(q, match):
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    with pytest.raises(ValueError, match=match):
        dense_attention_kvcache_q8(q, *cache, _i32([3, 3]), _i32([0, 1, 2]), 3)


def test_attention_refuses_lengths_plans_and_outputs():
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    q = torch.zeros(2, 32, 128, dtype=BF16)
    n, cu = _i32([3, 3]), _i32([0, 1, 2])
    for lens, offsets in ((n.long(), cu), (n[:1], cu), (n, cu[:2]), (n, cu.long())):
        with pytest.raises(ValueError, match="cache_seqlens must be int32"):
            dense_attention_kvcache_q8(q, *cache, lens, offsets, 3)
    for ids in (None, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3, 4, dtype=torch.int32),
                torch.zeros(1, 2, 4, dtype=torch.int32), torch.zeros(2, 2, 0, dtype=torch.int32),
                torch.zeros(2, 2, 257, dtype=torch.int32)):
        with pytest.raises(ValueError, match="topk_idx must"):
            sparse_attention_kvcache_q8(q, *cache, n, ids, cu)
    with pytest.raises(ValueError, match="out must be"):
        dense_attention_kvcache_q8(q, *cache, n, cu, 3, out=torch.zeros(2, 32, 128))
    with pytest.raises(RuntimeError, match="GPU"):
        dense_attention_kvcache_q8(q, *cache, n, cu, 3)


def test_new_cache_refusals():
    for a in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError, match="positive"):
            new_kvcache_q8(*a, device="cpu")
    with pytest.raises(ValueError, match="128 channels"):
        new_kvcache_q8(1, 64, 1, 64, device="cpu")


def test_linear_refusals():
    x = torch.zeros(3, 136, dtype=BF16)
    codes = torch.zeros(2, 2, 64, 16, dtype=torch.uint8)
    scales = torch.zeros(2, 1, 64, 4, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_mx4(x, codes, scales, 20)
    for bad in (x.float(), x[0], x[None]):
        with pytest.raises(ValueError, match="x must"):
            linear_mx4(bad, codes, scales, 20)
    for n, k, c, s in ((33, 136, codes, scales), (16, 136, codes, scales), (20, 128, codes, scales),
                       (20, 136, codes.int(), scales), (20, 136, codes, scales[:1]),
                       (20, 136, codes.transpose(0, 1), scales), (20, 136, codes, scales.int())):
        with pytest.raises(ValueError, match="weight needs"):
            linear_mx4(x[:, :k], c, s, n)
    for n, k in ((0, 136), (20, 4), (20, 132)):
        with pytest.raises(ValueError, match="multiple of 8"):
            linear_mx4(torch.zeros(3, k, dtype=BF16), codes, scales, n)
    with pytest.raises(ValueError, match="multiple of 32"):
        linear_mx4_silu_mul(x, codes, scales, 20)
    with pytest.raises(ValueError, match="unit column stride"):
        quantize_mx4(torch.zeros(136, 20).t())
    with pytest.raises(ValueError, match="unsupported dtype"):
        quantize_mx4(torch.zeros(20, 136, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_mx4(torch.zeros(20, 136))


def test_c_entry_points_refuse_before_any_launch():
    L = _hip.lib()
    B = _hip.LS_BF16
    append = lambda **k: L.ls_kvcache_append_q8(*{**dict(  # noqa: E731
        k8=16, v8=16, cbs=16384, ks=1, vs=1, sbs=2, pages=1, lens=4, kn=16, vn=16, nrs=256, cu=4,
        total=1, batch=1, G=2, D=128, dt=B, kc=None, kbs=0, krs=0, kcr=0, stream=None), **k}.values())
    for change, rc, word in (
            (dict(D=64), _hip.LS_ERR_UNSUPPORTED, b"head_dim"), (dict(dt=_hip.LS_F32), _hip.LS_ERR_UNSUPPORTED, b"bf16"),
            (dict(total=-1), _hip.LS_ERR_INVALID, b"sizes"), (dict(nrs=257), _hip.LS_ERR_UNSUPPORTED, b"aligned"),
            (dict(k8=None), _hip.LS_ERR_INVALID, b"null"), (dict(kn=18), _hip.LS_ERR_UNSUPPORTED, b"aligned"),
            (dict(kc=18), _hip.LS_ERR_UNSUPPORTED, b"compressed"), (dict(G=70000), _hip.LS_ERR_INVALID, b"heads")):
        assert append(**change) == rc and word in L.ls_last_error(), change
    assert append(total=0, k8=None) == _hip.LS_OK
    attend = lambda **k: L.ls_attn_kvcache_q8(*{**dict(  # noqa: E731
        q=16, qrs=4096, cu=4, total=1, k8=16, v8=16, cbs=16384, ks=1, vs=1, sbs=2, pages=1, lens=4, batch=1,
        H=32, G=2, D=128, dt=B, ids=None, n_pages=1, scale=1.0, causal=0, splits=1, out=16, lse=None, ws=None,
        wsb=0, stream=None), **k}.values())
    for change, rc, word in (
            (dict(H=33), _hip.LS_ERR_INVALID, b"sizes"), (dict(H=34), _hip.LS_ERR_UNSUPPORTED, b"16 query"),
            (dict(D=64), _hip.LS_ERR_UNSUPPORTED, b"head_dim"), (dict(dt=_hip.LS_F32), _hip.LS_ERR_UNSUPPORTED, b"bf16"),
            (dict(splits=0), _hip.LS_ERR_INVALID, b"n_splits"), (dict(splits=257), _hip.LS_ERR_INVALID, b"n_splits"),
            (dict(n_pages=0), _hip.LS_ERR_INVALID, b"n_pages"), (dict(ids=4, n_pages=257), _hip.LS_ERR_UNSUPPORTED, b"plan ids"),
            (dict(splits=2, n_pages=9), _hip.LS_ERR_WORKSPACE, b"workspace"), (dict(splits=2, n_pages=9, ws=16, wsb=8), _hip.LS_ERR_WORKSPACE, b"workspace"),
            (dict(q=None), _hip.LS_ERR_INVALID, b"null"), (dict(q=18), _hip.LS_ERR_UNSUPPORTED, b"aligned"),
            (dict(qrs=4097), _hip.LS_ERR_UNSUPPORTED, b"aligned"), (dict(pages=1 << 25), _hip.LS_ERR_UNSUPPORTED, b"pages"),
            (dict(total=1 << 31), _hip.LS_ERR_UNSUPPORTED, b"rows"), (dict(batch=0), _hip.LS_ERR_INVALID, b"sizes")):
        assert attend(**change) == rc and word in L.ls_last_error(), change
    assert attend(total=0, q=None) == _hip.LS_OK
    assert L.ls_attn_kvcache_q8_workspace_size(4, 2, 1) == 0
    assert L.ls_attn_kvcache_q8_workspace_size(4, 32, 3) == 4 * 4 * 32 * 3 * 130
    linear = lambda **k: L.ls_linear_mx4(*{**dict(  # noqa: E731
        x=16, xrs=64, rows=1, K=64, codes=16, scales=4, N=32, silu=0, dt=B, out=2, ors=32, ws=None, wsb=0, stream=None), **k}.values())
    for change, rc, word in (
            (dict(K=63), _hip.LS_ERR_INVALID, b"multiple of 8"), (dict(N=0), _hip.LS_ERR_INVALID, b"out_features"),
            (dict(rows=-1), _hip.LS_ERR_INVALID, b"rows"), (dict(silu=1, N=48), _hip.LS_ERR_UNSUPPORTED, b"32"),
            (dict(dt=_hip.LS_F32), _hip.LS_ERR_UNSUPPORTED, b"bf16"), (dict(xrs=63), _hip.LS_ERR_UNSUPPORTED, b"aligned"),
            (dict(x=18), _hip.LS_ERR_UNSUPPORTED, b"aligned"), (dict(codes=None), _hip.LS_ERR_INVALID, b"null")):
        assert linear(**change) == rc and word in L.ls_last_error(), change
    assert linear(rows=0, x=None) == _hip.LS_OK
    assert L.ls_quantize_mx4(None, 32, 1, 32, B, 16, 4, None) == _hip.LS_ERR_INVALID
    assert L.ls_quantize_mx4(16, 32, 1, 31, B, 16, 4, None) == _hip.LS_ERR_INVALID
    assert L.ls_dequantize_mx4(16, 4, 1, 32, _hip.LS_F32, 16, 32, None) == _hip.LS_ERR_UNSUPPORTED
    assert L.ls_dequantize_mx4(16, 4, 1, 32, B, 18, 32, None) == _hip.LS_ERR_UNSUPPORTED


def test_cache_class_refusals():
    for bad in (dict(kv_format="int8"), dict(kv_format="q8", kernel_size=64),
                dict(kv_format="q8", kernel_stride=8), dict(kv_format="q8", dtype=torch.float32),
                dict(kv_format="q8", head_dim=64)):
        with pytest.raises(ValueError):
            LeanSelectKVCache(1, 1, 64, 1, device="cpu", **bad)
    c = LeanSelectKVCache(2, 3, 100, 4, device="cpu", kv_format="q8")
    assert c.capacity == 128 and [t.shape for t in c.layer(1)] == [
        (3, 2, 4, 64, 128), (3, 2, 4, 128, 64), (3, 2, 4), (3, 2, 4)]
    with pytest.raises(RuntimeError, match="no cache step"):
        c.attend(0, None, None, None)


def test_outputs_that_overlap_are_refused(monkeypatch):
    monkeypatch.setattr(_hip, "gpu_index", lambda *t: 0)
    codes = torch.zeros(8, 1, 64, 16, dtype=torch.uint8)
    scales = torch.zeros(8, 1, 64, 4, dtype=torch.uint8)
    x = torch.zeros(3, 128, dtype=BF16)
    for out in (x, torch.zeros(1, 128, dtype=BF16).expand(3, 128),
                torch.zeros(384, dtype=BF16).as_strided((3, 128), (64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            linear_mx4(x, codes, scales, 128, out=out)
    q = torch.zeros(2, 32, 128, dtype=BF16)
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    with pytest.raises(ValueError, match="overlap q"):
        dense_attention_kvcache_q8(q, *cache, _i32([3, 3]), _i32([0, 1, 2]), 3, out=q)


@pytest.fixture
def sent(monkeypatch):
    """What the wrappers hand to the library: (device, entry point, arguments), in turn, with
    the int32 arrays behind the pointers read at that moment."""
    calls = []

    def launch(index, name, *args):
        calls.append((index, name, args, [list((ctypes.c_int32 * n).from_address(args[at]))
                                          for at, n in INT_ARGS[name]]))

    monkeypatch.setattr(_hip, "gpu_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "launch", launch)
    return calls


# (argument, entries) of the int32 arrays, for two sequences.
INT_ARGS = {"ls_kvcache_append_q8": [(7, 2), (11, 3)], "ls_attn_kvcache_q8": [(2, 3), (11, 2)]}


def test_lengths_and_offsets_that_are_not_contiguous_stay_apart(sent):
    """Each is copied to rows of its own: neither copy may be given back before the call."""
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    lens, cu = _i32([[3, 9], [5, 9]])[:, 0], _i32([[0, 9], [1, 9], [2, 9]])[:, 0]
    x = torch.zeros(2, 2, 128, dtype=BF16)
    q = torch.zeros(2, 32, 128, dtype=BF16)
    ids = torch.zeros(2, 2, 1, dtype=torch.int32)
    kvcache_append_q8(*cache, lens, x, x, cu)
    dense_attention_kvcache_q8(q, *cache, lens, cu, 5)
    sparse_attention_kvcache_q8(q, *cache, lens, ids, cu)
    assert [c[3] for c in sent] == [[[3, 5], [0, 1, 2]], [[0, 1, 2], [3, 5]], [[0, 1, 2], [3, 5]]]


@pytest.mark.parametrize("max_len,pages", [(-5, 1), (0, 1), (64, 1), (65, 2), (1 << 45, 2)])
def test_the_longest_length_is_only_a_hint(sent, max_len, pages):
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    q = torch.zeros(2, 32, 128, dtype=BF16)
    dense_attention_kvcache_q8(q, *cache, _i32([3, 5]), _i32([0, 1, 2]), max_len)
    assert sent[0][2][18] == pages


@pytest.mark.parametrize("current", [0, 1])
def test_launches_are_made_on_the_tensors_device(monkeypatch, current):
    """With that device current while it launches, on that device's current stream."""
    now, seen = [current], []

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    class Library:
        @staticmethod
        def ls_linear_mx4(*args):
            seen.append((now[0], args))
            return _hip.LS_OK

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_hip, "lib", lambda: Library)
    _hip.launch(1, "ls_linear_mx4", 7, None)
    assert seen == [(1, (7, None, 101))] and now == [current]


@pytest.mark.parametrize("sizes", [dict(hidden_size=1028), dict(intermediate_size=2050)])
def test_a_model_whose_sizes_do_not_fit_keeps_its_weights(sizes):
    m = object.__new__(MiniCPMLeanSelect)
    m.cfg, m.lm_head = MiniCPMConfig(**sizes), object()
    m.layers, head = [], m.lm_head
    with pytest.raises(ValueError, match="multiples of 8"):
        m.quantize_weights()
    assert m.lm_head is head


def test_operators_are_public():
    for name in ("new_kvcache_q8", "kvcache_append_q8", "sparse_attention_kvcache_q8",
                 "dense_attention_kvcache_q8", "quantize_mx4", "lay_out_mx4", "dequantize_mx4",
                 "linear_mx4", "linear_mx4_silu_mul"):
        assert name in ops.__all__ and callable(getattr(ops, name))
