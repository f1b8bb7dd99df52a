"""Attention over a dense cache with capped, biased and windowed scores, with and without a shared
prefix, on the GPU against its 64-bit form (oracle/serving_oracle.py): within half a step of the
output's type and the bound that the oracle derives."""
import itertools
import math

import pytest
import torch

from leanselect_amd.infllm_v2 import infllmv2_attn_with_kvcache
from leanselect_amd.ops import dense_attention_kvcache, shared_prefix_attention
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
BF16, FP16 = torch.bfloat16, torch.float16


def _cu(counts):
    return [0, *itertools.accumulate(counts)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _slopes(H, batch=None):
    s = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])
    return s if batch is None else torch.stack([s * (0.5 + i) for i in range(batch)])


def _inputs(lens, new, H, G, dtype, seed, prefix=0, capacity=None, strong=3.0):
    g = torch.Generator().manual_seed(seed)
    capacity = capacity or max(1, max(lens))
    gain = torch.exp(0.5 * torch.randn(G, D, generator=g))
    gain[:, :4] *= strong
    q = torch.randn(sum(new), H, D, generator=g).to(dtype)
    k = (torch.randn(len(lens), capacity, G, D, generator=g) * gain).to(dtype)
    v = torch.randn(len(lens), capacity, G, D, generator=g).to(dtype)
    kp = (torch.randn(prefix, G, D, generator=g) * gain).to(dtype)
    vp = torch.randn(prefix, G, D, generator=g).to(dtype)
    return q, k, v, kp, vp


def _check(got, want, dtype):
    out, lse = got
    exact, exact_lse, bound, lse_bound = want
    out, lse = out.cpu().double(), lse.cpu().double()
    assert bool(torch.isfinite(out).all())
    tiny = 2.0 ** -25 if dtype == FP16 else 0.0
    allowed = torch.finfo(dtype).eps / 2 * (exact.abs() + bound) + bound + tiny
    worst = ((out - exact).abs() / allowed.clamp(min=1e-300)).max().item() if out.numel() else 0.0
    assert bool(((out - exact).abs() <= allowed).all()), worst
    empty = torch.isinf(exact_lse)
    assert torch.equal(torch.isinf(lse) & (lse > 0), empty)
    far = (lse - exact_lse).abs()[~empty]
    assert bool((far <= lse_bound[~empty]).all()), far.max().item()


def _run(lens, new, H, G, dtype, seed=0, prefix=0, capacity=None, n_splits=None, strong=3.0, **options):
    q, k, v, kp, vp = _inputs(lens, new, H, G, dtype, seed, prefix, capacity, strong)
    cu = _cu(new)
    slopes = options.pop("alibi_slopes", None)
    more = dict(options, alibi_slopes=None if slopes is None else slopes.to(DEV), n_splits=n_splits,
                return_lse=True)
    if prefix:
        got = shared_prefix_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), k.to(DEV), v.to(DEV), _i32(lens),
                                      _i32(cu), max(lens), **more)
        options.update(k_prefix=kp, v_prefix=vp)
    else:
        got = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32(lens), _i32(cu), max(lens), **more)
    _check(got, so.cache_attention(q, k, v, lens, cu, alibi_slopes=slopes, **options), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,G", [(32, 2), (4, 4), (5, 5), (6, 2), (16, 1)])
@pytest.mark.parametrize("options", [
    dict(softcap=5.0), dict(window=(37, -1)), dict(window=(0, 0)), dict(causal=True, window=(130, 5)),
    dict(softcap=30.0, window=(300, 20), causal=True), "alibi", "alibi of each sequence"], ids=str)
def test_options(dtype, H, G, options):
    lens, new = [1, 300, 33, 0, 129], [1, 3, 2, 1, 4]
    if isinstance(options, str):
        options = dict(alibi_slopes=_slopes(H, len(lens) if "each" in options else None), causal=True)
    _run(lens, new, H, G, dtype, seed=3, **options)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 127, 128, 129, 640, 1999])
@pytest.mark.parametrize("n_splits", [None, 1, 5, 128])
def test_lengths_and_slices(dtype, length, n_splits):
    _run([length, 1], [1, 1], 8, 2, dtype, seed=length, n_splits=n_splits, softcap=20.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("prefix", [1, 31, 64, 129, 1500])
@pytest.mark.parametrize("options", [
    dict(), dict(causal=True), dict(softcap=8.0, window=(100, -1), causal=True), dict(window=(3, 1)), "alibi"],
    ids=str)
def test_prefix(dtype, prefix, options):
    if isinstance(options, str):
        options = dict(alibi_slopes=_slopes(16, 4), causal=True)
    _run([1, 70, 0, 200], [1, 2, 1, 5], 16, 2, dtype, seed=prefix, prefix=prefix, **options)


@pytest.mark.parametrize("H,G,rows,batch", [
    (32, 2, 1, 1), (32, 2, 1, 2), (32, 2, 1, 3), (32, 2, 1, 5), (32, 2, 4, 9), (5, 5, 1, 70), (8, 8, 3, 30),
    (24, 4, 2, 11), (16, 1, 1, 17)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefix_batches(dtype, H, G, rows, batch):
    """Row tiles of every width, the last one partly filled."""
    lens = [rows + 7 * b % 40 for b in range(batch)]
    _run(lens, [rows] * batch, H, G, dtype, seed=batch, prefix=333, causal=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,lens", [([40, 1, 0, 23], [300, 129, 55, 23]), ([130], [130]), ([70, 64], [1000, 64])])
@pytest.mark.parametrize("H,G", [(8, 2), (3, 3), (16, 1)])
@pytest.mark.parametrize("window", [(-1, -1), (50, -1)])
def test_chunks(dtype, new, lens, H, G, window):
    _run(lens, new, H, G, dtype, seed=sum(new), causal=True, softcap=15.0, window=window)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,G,most", [(32, 2, 4), (32, 8, 16), (16, 1, 3), (10, 2, 12)])
@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("n_splits", [None, 3])
@pytest.mark.parametrize("options", [dict(causal=True), dict(causal=True, window=(300, -1), softcap=20.0)],
                         ids=["causal", "capped window"])
def test_a_few_rows_a_sequence(dtype, H, G, most, prefix, n_splits, options):
    """Guessed tokens: each sequence's rows in several narrow tiles or in one wide one."""
    new = [most, 1, 0, most, most - 1, most]
    lens = [1500, 700, 90, most, 257, 2049]
    _run(lens, new, H, G, dtype, prefix=prefix, n_splits=n_splits, **options)


@pytest.mark.parametrize("batch,length", [(24, 2000), (24, 900), (3, 2000), (70, 300)])
def test_a_few_rows_of_many_sequences(batch, length):
    _run([length - 37 * b % length for b in range(batch)], [4] * batch, 32, 2, BF16, causal=False)


@pytest.mark.parametrize("prefix", [0, 40])
def test_rows_that_see_nothing(prefix):
    """More rows than keys: with causal, the first rows stand in front of every own key (with a prefix
    they still see the part of it behind them)."""
    _run([2, 0, 5], [4, 3, 1], 4, 2, BF16, prefix=prefix, causal=True, softcap=9.0)
    _run([2, 0, 5], [4, 3, 1], 4, 2, BF16, prefix=prefix, causal=True, window=(1, -1))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), "lowest"])
@pytest.mark.parametrize("H,G", [(32, 2), (4, 4)])
def test_hidden_values_do_not_count(dtype, bad, H, G):
    """Anything may stand in keys and values that a row does not see: past the end, in front of the
    window, and ahead of the row in the same chunk (seen by the chunk's later rows)."""
    bad = torch.finfo(dtype).min if bad == "lowest" else bad
    lens, new, prefix = [90, 200], [3, 3], 70
    q, k, v, kp, vp = _inputs(lens, new, H, G, dtype, 5, prefix, capacity=260)
    options = dict(causal=True, window=(100, -1), softcap=12.0)
    cu = _cu(new)
    want = so.cache_attention(q, k, v, lens, cu, k_prefix=kp, v_prefix=vp, **options)
    for b, n in enumerate(lens):
        k[b, n:], v[b, n:] = bad, bad
        k[b, n - 1], v[b, n - 1] = bad, bad  # only the last row sees it
    k[1, :94], v[1, :94] = bad, bad          # 200 - 3 + i - 100 is the first seen
    kp[:40], vp[:40] = bad, bad
    out, lse = shared_prefix_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), k.to(DEV), v.to(DEV), _i32(lens),
                                       _i32(cu), max(lens), return_lse=True, **options)
    rows = [0, 1, 3, 4]  # not the last ones
    pick = [w[rows] if w.shape[0] == 6 else w[:, rows] for w in want]
    _check((out[rows], lse[:, rows]), pick, dtype)


def test_values_that_are_not_finite_and_seen():
    """A channel in which a row sees an infinity or NaN is not finite, and no other is touched."""
    lens, new = [100], [2]
    q, k, v, _, _ = _inputs(lens, new, 4, 2, BF16, 6)
    want = so.cache_attention(q, k, v, lens, [0, 2], causal=True, softcap=10.0)
    v[0, 99, 0, 7] = float("nan")  # seen by row 1 alone
    v[0, 50, 1, 9] = float("inf")  # seen by both
    out, lse = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32(lens), _i32([0, 2]), 100,
                                       causal=True, softcap=10.0, return_lse=True)
    odd = torch.zeros(2, 4, D, dtype=torch.bool)
    odd[1, :2, 7] = True
    odd[:, 2:, 9] = True
    assert torch.equal(~torch.isfinite(out.cpu()), odd)
    clean = torch.where(odd, 0.0, out.cpu().double())
    exact = torch.where(odd, 0.0, want[0])
    _check((clean.to(BF16), lse), (exact, *want[1:]), BF16)


def test_queries_and_keys_that_are_not_finite():
    """A NaN among a row's scores makes that row NaN (its heads alone); a score of -inf has no weight."""
    lens, new = [70], [3]
    q, k, v, _, _ = _inputs(lens, new, 4, 2, BF16, 7)
    q[1, 2, 5] = float("nan")
    out = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32(lens), _i32([0, 3]), 70, softcap=10.0).cpu()
    nan = torch.isnan(out).all(-1)
    assert nan[1, 2] and int(nan.sum()) == 1 and int(torch.isnan(out).any(-1).sum()) == 1
    q[1, 2, 5] = 0.5
    k[0, 10] = 0.0
    k[0, 10, :, 0] = float("-inf")
    q[:, :, 0] = q[:, :, 0].abs() + 0.1
    got = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32(lens), _i32([0, 3]), 70,
                                  window=(1000, -1), return_lse=True)
    keep = [j for j in range(70) if j != 10]
    want = so.cache_attention(q, k[:, keep], v[:, keep], [69], [0, 3])
    _check(got, want, BF16)


def test_strides():
    """Views: queries of a packed projection, a cache among others, keys and values of one buffer."""
    H, G, lens, new = 8, 2, [70, 33], [2, 1]
    q, k, v, kp, vp = _inputs(lens, new, H, G, BF16, 8, prefix=50, capacity=80)
    cu = _cu(new)
    want = so.cache_attention(q, k, v, lens, cu, k_prefix=kp, v_prefix=vp, causal=True, softcap=20.0)
    packed = torch.full((3, H * D + 24), float("nan"), dtype=BF16, device=DEV)
    packed[:, 8:8 + H * D] = q.view(3, -1).to(DEV)
    both = torch.full((3, 2, 100, 2, G, D), float("nan"), dtype=BF16, device=DEV)
    both[0, :, 10:90, 0], both[0, :, 10:90, 1] = k.to(DEV), v.to(DEV)
    pre = torch.full((50, 2 * G, D), float("nan"), dtype=BF16, device=DEV)
    pre[:, :G], pre[:, G:] = kp.to(DEV), vp.to(DEV)
    lens_2 = torch.stack((_i32(lens), _i32([999, 999])), 1)
    cu_2 = torch.stack((_i32(cu), _i32([9, 9, 9])), 1)
    for q_view in (packed[:, 8:8 + H * D].view(3, H, D), q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)):
        got = shared_prefix_attention(q_view, pre[:, :G], pre[:, G:], both[0, :, 10:90, 0], both[0, :, 10:90, 1],
                                      lens_2[:, 0], cu_2[:, 0], 70, causal=True, softcap=20.0, return_lse=True)
        _check(got, want, BF16)


def test_given_output_and_rows_behind_the_last_sequence():
    lens, new = [40, 50], [1, 2]
    q, k, v, _, _ = _inputs(lens, [1, 2, 3], 4, 2, BF16, 9, capacity=64)
    k, v = k[:2], v[:2]
    args = (k.to(DEV), v.to(DEV), _i32(lens), _i32([0, 1, 3]))
    want = so.cache_attention(q[:3], k, v, lens, [0, 1, 3])
    kp, vp = k[0, :20], v[0, :20]
    for n_splits in (None, 1, 3):
        out = torch.full((6, 4, D), 7.0, dtype=BF16, device=DEV)
        got = shared_prefix_attention(q.to(DEV), kp[:0].to(DEV), vp[:0].to(DEV), *args, 50, out=out,
                                      n_splits=n_splits, return_lse=True)
        assert got[0] is out and bool((out[3:] == 7.0).all())
        _check((out[:3], got[1][:, :3]), want, BF16)
    buffer = torch.zeros(6, 8, D, dtype=BF16, device=DEV)
    qv = buffer[:, :4]
    qv.copy_(q.to(DEV))
    with pytest.raises(ValueError, match="overlap"):
        shared_prefix_attention(qv, kp[:0].to(DEV), vp[:0].to(DEV), *args, 50, out=buffer.view(-1)[:6 * 4 * D].view(6, 4, D))
    with pytest.raises(ValueError, match="overlap"):
        shared_prefix_attention(q.to(DEV), kp[:0].to(DEV), vp[:0].to(DEV), *args, 50, out=args[0].view(-1)[:6 * 4 * D].view(6, 4, D))


def test_no_rows_and_lengths_past_the_capacity():
    q, k, v, _, _ = _inputs([10], [1], 4, 2, BF16, 10)
    none = dense_attention_kvcache(q[:0].to(DEV), k.to(DEV), v.to(DEV), _i32([10]), _i32([0, 0]), 10, softcap=3.0)
    assert none.shape == (0, 4, D)
    a = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32([10]), _i32([0, 1]), 10, softcap=3.0)
    b = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32([500]), _i32([0, 1]), 500, softcap=3.0)
    assert torch.equal(a, b)
    c = dense_attention_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), _i32([-3]), _i32([0, 1]), 10, softcap=3.0)
    assert bool((c == 0).all())


def test_a_cache_past_32_bits():
    """Byte offsets of the visible keys lie above 2^32."""
    cap, n = (1 << 23) + 300, 300
    k = torch.empty(1, cap, 2, D, dtype=BF16, device=DEV)
    v = torch.empty(1, cap, 2, D, dtype=BF16, device=DEV)
    q, ks, vs, _, _ = _inputs([n], [1], 8, 2, BF16, 11)
    k[0, cap - n:], v[0, cap - n:] = ks[0].to(DEV), vs[0].to(DEV)
    got = dense_attention_kvcache(q.to(DEV), k, v, _i32([cap]), _i32([0, 1]), cap, window=(n - 1, -1), return_lse=True)
    _check(got, so.cache_attention(q, ks, vs, [n], [0, 1]), BF16)


def test_large_magnitudes():
    """Scores of hundreds, of both signs: the running maximum moves often."""
    _run([700], [2], 4, 2, BF16, seed=12, strong=60.0, window=(600, -1))
    _run([700], [2], 4, 2, FP16, seed=12, strong=60.0, window=(600, -1))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("softcap", [1e-20, 0.01, 512.0])
def test_the_least_and_largest_caps(dtype, rows, softcap):
    _run([400, 90], [rows, 3], 32, 2, dtype, causal=True, softcap=softcap)


def test_rows_in_front_of_the_first_sequence():
    """They belong to none, and are left as they are where the output is given."""
    q, k, v, kp, vp = _inputs([300], [6], 32, 2, BF16, 3, prefix=900)
    out = torch.full((6, 32, D), 7.0, dtype=BF16, device=DEV)
    shared_prefix_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), k.to(DEV), v.to(DEV), _i32([300]), _i32([2, 5]), 300, out=out)
    want = so.cache_attention(q[2:5], k, v, [300], [0, 3], k_prefix=kp, v_prefix=vp)
    assert bool((out[:2] == 7).all()) and bool((out[5:] == 7).all())
    exact, _, bound, _ = want
    allowed = torch.finfo(BF16).eps / 2 * (exact.abs() + bound) + bound
    assert bool(((out[2:5].cpu().double() - exact).abs() <= allowed).all())


@pytest.mark.parametrize("options", [dict(softcap=20.0), dict(window_size=(40, 0)), dict(window_size=(30, -1), causal=True),
                                     dict(alibi_slopes=_slopes(8, 2), causal=True)], ids=str)
def test_with_kvcache_options(options):
    """The drop-in appends the new keys and attends with the options."""
    B, Sq, H, G, cap = 2, 3, 8, 2, 128
    lens = [70, 20]
    q, k, v, _, _ = _inputs([x + Sq for x in lens], [Sq] * B, H, G, BF16, 13, capacity=cap)
    kc, vc = k.clone().to(DEV), v.clone().to(DEV)
    new = [torch.stack([t[b, n:n + Sq] for b, n in enumerate(lens)]).to(DEV) for t in (k, v)]
    for t in (kc, vc):
        for b, n in enumerate(lens):
            t[b, n:] = float("nan")
    more = {n: o.to(DEV) if torch.is_tensor(o) else o for n, o in options.items()}
    out, lse = infllmv2_attn_with_kvcache(q.view(B, Sq, H, D).to(DEV), kc, vc, *new, cache_seqlens=_i32(lens),
                                          return_softmax_lse=True, **more)
    options = {("window" if n == "window_size" else n): o for n, o in options.items()}
    want = so.cache_attention(q, k, v, [x + Sq for x in lens], _cu([Sq] * B), **options)
    _check((out.view(B * Sq, H, D), lse.permute(1, 0, 2).reshape(H, B * Sq)), want, BF16)


def test_a_row_does_not_depend_on_the_batch():
    """Rows of other sequences do not change a row's value beyond the order of its sums, and two calls agree."""
    q, k, v, kp, vp = _inputs([60, 90, 33], [1, 1, 1], 8, 2, BF16, 14, prefix=500)
    args = [t.to(DEV) for t in (q, kp, vp, k, v)]
    a = shared_prefix_attention(*args, _i32([60, 90, 33]), _i32([0, 1, 2, 3]), 90)
    b = shared_prefix_attention(*args, _i32([60, 90, 33]), _i32([0, 1, 2, 3]), 90)
    assert torch.equal(a, b)
    args[0] = args[0].clone()
    args[0][1:] = float("nan")
    c = shared_prefix_attention(*args, _i32([60, 90, 33]), _i32([0, 1, 2, 3]), 90)
    assert torch.equal(a[0], c[0])
