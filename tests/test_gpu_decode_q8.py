"""The 8-bit KV cache on the GPU against its 64-bit forms (oracle/lowbit_oracle.py): the append
byte for byte, attention within what its roundings can move (a half step of the output's type,
and the bound the oracle derives from fp16 weights and float32 scores)."""
import math

import pytest
import torch

from leanselect_amd import minicpm
from leanselect_amd.cache import LeanSelectKVCache
from leanselect_amd.ops import (decode_topk_idx, dense_attention_kvcache_q8, kvcache_append_q8,
                                new_kvcache_q8, sparse_attention_kvcache_q8)
from leanselect_amd.ops.decode import n_windows
from oracle import lowbit_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _cu(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _garbage(batch, capacity, G, seed=0):
    """A cache whose bytes and codes are anything, NaN patterns and code 255 among them."""
    g = torch.Generator().manual_seed(seed)
    cache = new_kvcache_q8(batch, capacity, G)
    for t in cache:
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    cache[2].fill_(255)
    cache[3].fill_(255)
    return cache


def _rows(n, G, dtype, g, spread=1.0):
    x = torch.randn(n, G, D, generator=g) * torch.exp(spread * torch.randn(n, G, 1, generator=g))
    return x.to(dtype)


def _same_bytes(cache, want, lens):
    """Every visible byte and code equals the oracle's; returns nothing else's state."""
    got = lo.Q8Cache(*cache)
    for b, n in enumerate(lens):
        pages = -(-n // 64)
        for a, c in ((got.kcode, want.kcode), (got.vcode, want.vcode)):
            assert torch.equal(a[b, :pages], c[b, :pages]), b
        for name in ("k", "v"):
            a = getattr(got, name)[b].transpose(1, 2).reshape(-1, got.k.shape[2], D)[:n]
            c = getattr(want, name)[b].transpose(1, 2).reshape(-1, got.k.shape[2], D)[:n]
            assert torch.equal(torch.isnan(a), torch.isnan(c)), (name, b)
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(c)), (name, b)


def _filled(lens, G, dtype, seed, capacity=None, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    cache = _garbage(len(lens), capacity or max(64, max(lens)), G, seed)
    k, v = _rows(sum(lens), G, dtype, g, spread), _rows(sum(lens), G, dtype, g, spread)
    kvcache_append_q8(*cache, _i32([0] * len(lens)), k.to(DEV), v.to(DEV), _i32(_cu(lens)))
    return cache


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,steps", [
    (2, [[37, 64, 0, 1], [1, 1, 1, 1], [26, 0, 63, 64], [1, 1, 1, 1], [130, 5, 2, 0]]),
    (1, [[65], [1], [62], [1], [1], [200]]),
    (5, [[0, 3, 300], [0, 0, 0], [1, 1, 1], [64, 61, 20]]),
])
def test_append_equals_the_definition_byte_for_byte(dtype, G, steps):
    g = torch.Generator().manual_seed(11)
    B, cap = len(steps[0]), 512
    cache = _garbage(B, cap, G, 3)
    kc = torch.full((B, n_windows(cap), G, D), 7.0, dtype=dtype, device=DEV)
    want = lo.Q8Cache(*cache)
    lens = [0] * B
    for new in steps:
        k, v = _rows(sum(new), G, dtype, g), _rows(sum(new), G, dtype, g)
        want.append(lens, k, v, _cu(new))
        before = [n_windows(n) for n in lens]
        kc_before = kc.clone()
        kvcache_append_q8(*cache, _i32(lens), k.to(DEV), v.to(DEV), _i32(_cu(new)), kc_cache=kc)
        lens = [a + b for a, b in zip(lens, new)]
        _same_bytes(cache, want, lens)
        eps = torch.finfo(dtype).eps / 2
        for b in range(B):
            after = n_windows(lens[b])
            assert torch.equal(kc[b, :before[b]], kc_before[b, :before[b]])
            assert torch.equal(kc[b, after:], kc_before[b, after:])
            for w in range(before[b], after):
                for h in range(G):
                    ref = want.window(b, h, w)
                    # 32 terms in float32, then one rounding (a subnormal fp16 step is 2^-24).
                    size = want.keys(b, h)[16 * w:16 * w + 32].abs().mean(0)
                    tol = eps * ref.abs() + 2.0 ** -19 * size + 2.0 ** -25
                    assert bool(((kc[b, w, h].cpu().double() - ref).abs() <= tol).all()), (b, w, h)


def test_append_leaves_what_it_does_not_write():
    """Rows after the new ones, pages not touched and other sequences keep their bytes."""
    G = 2
    cache = _garbage(3, 256, G, 5)
    before = [t.clone() for t in cache]
    g = torch.Generator().manual_seed(1)
    k, v = _rows(70, G, torch.bfloat16, g).to(DEV), _rows(70, G, torch.bfloat16, g).to(DEV)
    kvcache_append_q8(*cache, _i32([0, 0, 0]), k, v, _i32([0, 0, 70, 70]))
    for t, o in zip(cache, before):
        assert torch.equal(t[0].view(torch.uint8), o[0].view(torch.uint8))
        assert torch.equal(t[2].view(torch.uint8), o[2].view(torch.uint8))
        assert torch.equal(t[1, 2:].view(torch.uint8), o[1, 2:].view(torch.uint8))
    got, old = lo.Q8Cache(*cache), lo.Q8Cache(*before)
    for a, c in ((got.k, old.k), (got.v, old.v)):
        a, c = a[1, 1, :, 6:], c[1, 1, :, 6:]
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_of_extreme_rows(dtype):
    """Zeros, the smallest and largest finite magnitudes, infinities and NaN, a maximum at a
    code's border, and a page raised by 2^100 whose older rows become zeros."""
    G, top = 1, torch.finfo(dtype).max
    rows = torch.zeros(9, G, D)
    rows[1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    rows[2, 0, 0] = 448.0 * 2.0 ** -7
    rows[3, 0, 0] = 450.0 * 2.0 ** -7
    rows[4, 0, 0] = torch.finfo(dtype).tiny
    rows[5, 0, :] = -0.0
    rows[6, 0, 0] = 2.0 ** -20
    rows[7, 0, 0] = top
    rows[8, 0, 1] = -top
    rows = rows.to(dtype)
    cache = _garbage(9, 64, G, 2)
    want = lo.Q8Cache(*cache)
    for order in (list(range(9)), [6, 5, 4, 3, 2, 1, 0, 8, 7], [7, 6, 0, 1, 2, 8, 3, 4, 5]):
        for pos, i in enumerate(order):  # the same rows one by one into sequence i, in this order
            n = [pos] * 9
            x = torch.stack([rows[order[(s + pos) % 9]] for s in range(9)])
            want.append(n, x, x, list(range(10)))
            kvcache_append_q8(*cache, _i32(n), x.to(DEV), x.to(DEV), _i32(list(range(10))))
            _same_bytes(cache, want, [pos + 1] * 9)


def test_append_reads_strided_and_unaligned_rows():
    G, n = 2, 100
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(n, 3 * G * D + 8, generator=g).to(torch.bfloat16).to(DEV)
    views = [(wide[:, :G * D].view(n, G, D), wide[:, G * D:2 * G * D].view(n, G, D)),
             (wide[:, 4:G * D + 4].view(n, G, D), wide[:, G * D:2 * G * D].view(n, G, D)),
             (wide[:, :G * D].view(n, G, D).clone(), wide[:, G * D:2 * G * D].view(n, G, D)),
             (wide[:, :G * D].view(n, D, G).transpose(1, 2), wide[:, 8:G * D + 8].view(n, G, D))]
    for k, v in views:
        cache = _garbage(1, 128, G, 1)
        want = lo.Q8Cache(*cache)
        want.append([0], k.cpu(), v.cpu(), [0, n])
        kvcache_append_q8(*cache, _i32([0]), k, v, _i32([0, n]))
        _same_bytes(cache, want, [n])


def test_append_to_many_sequences():
    """More sequences than a wave scans at once, some idle."""
    G, B = 1, 150
    lens = [(7 * b) % 70 for b in range(B)]
    cache = _garbage(B, 192, G, 4)
    want = lo.Q8Cache(*cache)
    g = torch.Generator().manual_seed(6)
    x = _rows(sum(lens), G, torch.bfloat16, g)
    want.append([0] * B, x, x, _cu(lens))
    kvcache_append_q8(*cache, _i32([0] * B), x.to(DEV), x.to(DEV), _i32(_cu(lens)))
    new = [(b % 3) * (b % 5) for b in range(B)]
    y = _rows(sum(new), G, torch.bfloat16, g)
    want.append(lens, y, y, _cu(new))
    kc = torch.zeros(B, n_windows(192), G, D, dtype=torch.bfloat16, device=DEV)
    kvcache_append_q8(*cache, _i32(lens), y.to(DEV), y.to(DEV), _i32(_cu(new)), kc_cache=kc)
    after = [a + b for a, b in zip(lens, new)]
    _same_bytes(cache, want, after)
    for b in range(B):
        for w in range(n_windows(lens[b]), n_windows(after[b])):
            ref = want.window(b, 0, w)
            size = want.keys(b, 0)[16 * w:16 * w + 32].abs().mean(0)
            assert bool(((kc[b, w, 0].cpu().double() - ref).abs()
                         <= 2.0 ** -8 * ref.abs() + 2.0 ** -19 * size).all()), (b, w)


def test_offsets_past_the_new_rows_write_nothing():
    """Offsets on the device that pass the rows there are (the host's lists say otherwise):
    the rows there are get written, and no page or code behind them."""
    cache = _garbage(2, 256, 1, 5)
    x = _rows(2, 1, torch.bfloat16, torch.Generator().manual_seed(30)).to(DEV)
    before = [t.view(torch.uint8).clone() for t in cache]
    kvcache_append_q8(*cache, _i32([0, 0]), x, x, _i32([0, 200, 200]), cache_seqlens_host=[0, 0],
                      cu_seqlens_new_host=[0, 1, 2])
    for t, old in zip(cache, before):
        new = t.view(torch.uint8)
        assert torch.equal(new[0, 1:], old[0, 1:]) and torch.equal(new[1], old[1])


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _check(out, lse, want, want_lse, bound, dtype, rows=None):
    got = out.cpu().double()
    rows = slice(None) if rows is None else rows
    eps = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err = (got - want).abs()[rows]
    tol = (eps * want.abs() + bound * (1 + eps) + tiny)[rows]
    assert bool((err <= tol).all()), f"largest excess {(err - tol).max().item():.3e}"
    if lse is not None:
        a, b = lse.cpu().double()[:, rows], want_lse[:, rows]
        assert torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(b)
        # The weights' fp16 rounding moves the sum by 2^-12 at most; scores in float32.
        assert bool(((a - b).abs()[ok] <= 2.0 ** -11 + 2.0 ** -16 * (1 + b.abs()[ok])).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G", [(32, 2), (16, 1), (24, 4), (5, 5), (3, 1)])
def test_dense_attention_at_the_lengths_where_pages_end(dtype, H, G):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 0]
    cache = _filled(lens, G, dtype, 7)
    ref = lo.Q8Cache(*cache)
    g = torch.Generator().manual_seed(8)
    cu = list(range(len(lens) + 1))
    q = torch.randn(len(lens), H, D, generator=g).to(dtype)
    want, want_lse, bound = lo.attend(ref, q, lens, cu)
    for n_splits in (None, 1, 3, 200):
        out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), _i32(cu), max(lens),
                                              n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)
        assert bool((out[-1] == 0).all()) and bool(torch.isinf(lse[:, -1]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sparse_attention_of_messy_plans(dtype):
    """-1, repeated, unsorted, out-of-range ids, an empty plan, and a sequence of no tokens."""
    lens, H, G = [700, 65, 1500, 1, 0], 32, 2
    cache = _filled(lens, G, dtype, 9)
    ref = lo.Q8Cache(*cache)
    g = torch.Generator().manual_seed(10)
    q = torch.randn(5, H, D, generator=g).to(dtype)
    cu = list(range(6))
    ids = torch.randint(-2, 30, (G, 5, 19), generator=g, dtype=torch.int32)
    ids[:, :, 5] = ids[:, :, 2]
    ids[0, 2] = -1
    ids[1, 0, 3] = 2 ** 31 - 1
    ids[1, 0, 4] = -2 ** 31
    ids[0, 3, 0] = 0
    want, want_lse, bound = lo.attend(ref, q, lens, cu, ids)
    for n_splits in (None, 1, 2, 19):
        out, lse = sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), ids.to(DEV), _i32(cu),
                                               n_splits=n_splits, return_lse=True)
        _check(out, lse, want, want_lse, bound, dtype)


@pytest.mark.parametrize("take", [1, 64, 65, 200, 256])
def test_sparse_attention_of_long_plans_with_repeats(take):
    lens, H, G = [4000, 777], 16, 1
    cache = _filled(lens, G, torch.bfloat16, 12)
    g = torch.Generator().manual_seed(13)
    q = torch.randn(2, H, D, generator=g).to(torch.bfloat16)
    ids = torch.randint(0, 63, (G, 2, take), generator=g, dtype=torch.int32)
    want, want_lse, bound = lo.attend(lo.Q8Cache(*cache), q, lens, [0, 1, 2], ids)
    out, lse = sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), ids.to(DEV),
                                           _i32([0, 1, 2]), return_lse=True)
    _check(out, lse, want, want_lse, bound, torch.bfloat16)


@pytest.mark.parametrize("sparse", [True, False])
def test_several_rows_a_sequence(sparse):
    """Causal rows of a multi-token step, a sequence with more rows than keys among them, rows
    behind the last sequence left as they were, and a caller's scale."""
    lens, lq, H, G = [300, 3, 64], [3, 5, 1], 24, 4
    cache = _filled(lens, G, torch.bfloat16, 14)
    ref = lo.Q8Cache(*cache)
    cu = _cu(lq)
    g = torch.Generator().manual_seed(15)
    q = torch.randn(cu[-1] + 2, H, D, generator=g).to(torch.bfloat16)
    ids = torch.tensor([0, 4, 1, -1], dtype=torch.int32).expand(G, cu[-1] + 2, 4).contiguous()
    for causal in (True, False):
        for n_splits in (None, 1, 2):
            out = torch.full((cu[-1] + 2, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
            args = dict(causal=causal, softmax_scale=0.2, n_splits=n_splits, out=out)
            if sparse:
                sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), ids.to(DEV), _i32(cu), **args)
            else:
                dense_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), _i32(cu), 300, **args)
            want, _, bound = lo.attend(ref, q, lens, cu, ids if sparse else None, causal, 0.2)
            _check(out, None, want, None, bound, torch.bfloat16, slice(0, cu[-1]))
            assert bool((out[cu[-1]:] == 3.0).all())


@pytest.mark.parametrize("max_len", [0, 1, 65, 1 << 40])
@pytest.mark.parametrize("n_splits", [None, 1, 2, 7])
def test_the_longest_length_only_cuts_the_work(max_len, n_splits):
    lens, H, G = [1300, 1, 640], 16, 2
    cache = _filled(lens, G, torch.bfloat16, 33)
    q = torch.randn(3, H, D, generator=torch.Generator().manual_seed(34)).to(torch.bfloat16)
    want, want_lse, bound = lo.attend(lo.Q8Cache(*cache), q, lens, [0, 1, 2, 3])
    out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), _i32([0, 1, 2, 3]), max_len,
                                          n_splits=n_splits, return_lse=True)
    _check(out, lse, want, want_lse, bound, torch.bfloat16)


@pytest.mark.parametrize("sparse", [True, False])
def test_more_sequences_than_a_wave(sparse):
    """Rows are found by search then; sequences without a row and rows behind the last one."""
    B, H, G = 70, 8, 2
    lens = [(37 * b) % 200 for b in range(B)]
    lq = [(b % 5) // 2 for b in range(B)]
    cache = _filled(lens, G, torch.bfloat16, 31)
    ref = lo.Q8Cache(*cache)
    cu, total = _cu(lq), sum(lq) + 3
    g = torch.Generator().manual_seed(32)
    q = torch.randn(total, H, D, generator=g).to(torch.bfloat16)
    ids = torch.randint(-1, 5, (G, total, 6), generator=g, dtype=torch.int32)
    want, want_lse, bound = lo.attend(ref, q, lens, cu, ids if sparse else None, True)
    for n_splits in (None, 1, 2):
        out = torch.full((total, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
        args = dict(causal=True, n_splits=n_splits, out=out, return_lse=True)
        if sparse:
            _, lse = sparse_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), ids.to(DEV), _i32(cu), **args)
        else:
            _, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32(lens), _i32(cu), max(lens), **args)
        _check(out, lse, want, want_lse, bound, torch.bfloat16, slice(0, cu[-1]))
        assert bool((out[cu[-1]:] == 3.0).all())


def test_values_that_are_not_seen_do_not_matter():
    """The cache past a sequence's end, pages outside the plan and a later key under the causal
    limit hold NaN (and code 255): outputs are the same bits as over zeros there."""
    lens, H, G = [70, 200], 32, 2
    cache = _filled(lens, G, torch.bfloat16, 16, capacity=320)
    clean = [t.clone() for t in cache]
    ref = lo.Q8Cache(*clean)  # places of tokens
    for b, n in enumerate(lens):
        for tok in range(n, 320):
            p, s = divmod(tok, 64)
            cache[0][b, p, :, s] = math.nan
            cache[1][b, p, :, :, lo.place(s)] = math.nan
            clean[0].view(torch.uint8)[b, p, :, s] = 0
            clean[1].view(torch.uint8)[b, p, :, :, lo.place(s)] = 0
    g = torch.Generator().manual_seed(17)
    q = torch.randn(2, H, D, generator=g).to(torch.bfloat16).to(DEV)
    cu = _i32([0, 1, 2])
    a = dense_attention_kvcache_q8(q, *cache, _i32(lens), cu, 200)
    b = dense_attention_kvcache_q8(q, *clean, _i32(lens), cu, 200)
    assert torch.equal(a, b) and bool(torch.isfinite(a).all())
    want, _, bound = lo.attend(ref, q.cpu(), lens, [0, 1, 2])
    _check(a, None, want, None, bound, torch.bfloat16)
    # One row of two does not see the last key, which is NaN; the other does.
    k = torch.zeros(1, G, D, dtype=torch.bfloat16, device=DEV)
    k[0, 1] = math.nan
    kvcache_append_q8(*cache, _i32(lens), k, k, _i32([0, 0, 1]))
    q2 = q[:1].expand(2, H, D).contiguous()
    out = dense_attention_kvcache_q8(q2, *cache, _i32([70, 201]), _i32([0, 0, 2]), 201, causal=True)
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(out[1, :H // 2]).all())
    assert bool(torch.isnan(out[1, H // 2:]).all())


def test_scores_far_apart():
    """A key that takes all the weight, in the first and in the last page; equal keys."""
    H, G, n = 16, 1, 1000
    g = torch.Generator().manual_seed(18)
    for at in (0, 500, n - 1):
        k = torch.randn(n, G, D, generator=g) * 0.1
        k[at] = 30.0
        v = torch.randn(n, G, D, generator=g)
        cache = _garbage(1, n, G)
        kvcache_append_q8(*cache, _i32([0]), k.bfloat16().to(DEV), v.bfloat16().to(DEV), _i32([0, n]))
        q = torch.cat([torch.full((1, H, D), 3.0), torch.full((1, H, D), -3.0), torch.zeros(1, H, D)])
        q = q.bfloat16()
        want, want_lse, bound = lo.attend(lo.Q8Cache(*cache), q, [n], [0, 3])
        out, lse = dense_attention_kvcache_q8(q.to(DEV), *cache, _i32([n]), _i32([0, 3]), n,
                                              return_lse=True)
        _check(out, lse, want, want_lse, bound, torch.bfloat16)


def test_queries_in_a_packed_projection():
    lens, H, G = [130, 64], 32, 2
    cache = _filled(lens, G, torch.bfloat16, 19)
    g = torch.Generator().manual_seed(20)
    qkv = torch.randn(2, (H + 2 * G) * D + 8, generator=g).bfloat16().to(DEV)
    cu = _i32([0, 1, 2])
    for q in (qkv[:, :H * D].view(2, H, D), qkv[:, 3:H * D + 3].view(2, H, D),
              qkv[:, :H * D].view(2, D, H).transpose(1, 2)):
        out = dense_attention_kvcache_q8(q, *cache, _i32(lens), cu, 130)
        again = dense_attention_kvcache_q8(q.contiguous().clone(), *cache, _i32(lens), cu, 130)
        assert torch.equal(out, again)


def test_a_cache_past_four_gigabytes():
    """Pages whose byte offsets pass 2^32, in the last of two sequences."""
    G, pages, H = 2, 1 << 17, 32
    cache = new_kvcache_q8(2, pages * 64, G)
    n = pages * 64 - 30
    g = torch.Generator().manual_seed(21)
    k, v = _rows(200, G, torch.bfloat16, g), _rows(200, G, torch.bfloat16, g)
    for t in (cache[2], cache[3]):
        t.fill_(120)
    first = (n - 200) // 64 * 64  # the pages before are never read
    kvcache_append_q8(*cache, _i32([0, first]), k.to(DEV), v.to(DEV), _i32([0, 0, 200]),
                      cache_seqlens_host=[0, first], cu_seqlens_new_host=[0, 0, 200])
    small = new_kvcache_q8(1, 256, G)
    kvcache_append_q8(*small, _i32([0]), k.to(DEV), v.to(DEV), _i32([0, 200]))
    q = torch.randn(1, H, D, generator=g).bfloat16().to(DEV)
    p = first // 64
    ids = torch.arange(4, dtype=torch.int32, device=DEV).expand(G, 1, 4).contiguous()
    a = sparse_attention_kvcache_q8(q, *cache, _i32([0, first + 200]), ids + p, _i32([0, 0, 1]))
    b = sparse_attention_kvcache_q8(q, *small, _i32([200]), ids, _i32([0, 1]))
    assert torch.equal(a, b)


def test_a_step_captured_and_replayed():
    """Append and attention in one graph: three replays, each against the eager calls on a copy,
    with eager work between them; lengths on the device move between replays."""
    lens, H, G = [100, 63, 640], 32, 2
    cache = _filled(lens, G, torch.bfloat16, 22, capacity=704)
    twin = [t.clone() for t in cache]
    g = torch.Generator().manual_seed(23)
    B = len(lens)
    q = torch.empty(B, H, D, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.empty(B, G, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    before, after, cu = _i32(lens), _i32([n + 1 for n in lens]), _i32(list(range(B + 1)))
    host = dict(cache_seqlens_host=lens, cu_seqlens_new_host=list(range(B + 1)))

    def step(c):
        kvcache_append_q8(*c, before, k, v, cu, **host)
        return dense_attention_kvcache_q8(q, *c, after, cu, 704)

    def fill():
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))

    fill()
    warm = [t.clone() for t in cache]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(warm)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for _ in range(3):
        fill()
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, c in zip(cache, twin):
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
        before += 1
        after += 1


def test_two_streams_at_once():
    lens, H, G = [3000], 32, 2
    sides = []
    for seed in (24, 25):
        cache = _filled(lens, G, torch.bfloat16, seed)
        q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)
        sides.append((cache, q, dense_attention_kvcache_q8(q, *cache, _i32(lens), _i32([0, 1]), 3000)))
    n, cu = _i32(lens), _i32([0, 1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(5):
        for i, (cache, q, _) in enumerate(sides):
            with torch.cuda.stream(streams[i]):
                got[i].append(dense_attention_kvcache_q8(q, *cache, n, cu, 3000))
    torch.cuda.synchronize()
    for i, (_, _, want) in enumerate(sides):
        assert all(torch.equal(x, want) for x in got[i])


def test_nothing_to_do():
    cache = _filled([5], 2, torch.bfloat16, 26)
    q = torch.empty(0, 32, D, dtype=torch.bfloat16, device=DEV)
    assert dense_attention_kvcache_q8(q, *cache, _i32([5]), _i32([0, 0]), 5).shape == (0, 32, D)
    ids = torch.empty(2, 0, 3, dtype=torch.int32, device=DEV)
    assert sparse_attention_kvcache_q8(q, *cache, _i32([5]), ids, _i32([0, 0])).shape == (0, 32, D)
    none = torch.empty(0, 2, D, dtype=torch.bfloat16, device=DEV)
    kvcache_append_q8(*cache, _i32([5]), none, none, _i32([0, 0]))


# ---------------------------------------------------------------------------
# In the cache class and the model
# ---------------------------------------------------------------------------
def test_cache_class_runs_the_operators_together():
    """Prompt, then ragged steps through ``LeanSelectKVCache(kv_format="q8")``: its tensors equal
    the definition's bytes, the plans come from its compressed keys, attention reads them."""
    G, H, layers = 2, 32, 2
    cache = LeanSelectKVCache(layers, 3, 600, G, kv_format="q8")
    plain = LeanSelectKVCache(layers, 3, 600, G)
    assert cache.k8.shape == (layers, 3, 10, G, 64, 128)
    want = [lo.Q8Cache(*cache.layer(i)) for i in range(layers)]
    g = torch.Generator().manual_seed(30)
    lens = [0, 0, 0]
    for new in ([500, 65, 31], [1, 1, 1], [1, 0, 1], [1, 1, 1]):
        for c in (cache, plain):
            c.begin(new)
        rows = [b for b in range(3) for _ in range(new[b])]
        cu = _cu(new)
        after = [a + b for a, b in zip(lens, new)]
        for i in range(layers):
            k, v = _rows(cu[-1], G, torch.bfloat16, g, 0.3), _rows(cu[-1], G, torch.bfloat16, g, 0.3)
            want[i].append(lens, k, v, cu)
            for c in (cache, plain):
                c.update(i, k.to(DEV), v.to(DEV))
            _same_bytes(cache.layer(i), want[i], after)
            if max(new) == 1:
                q = torch.randn(len(rows), H, D, generator=g).bfloat16()
                ids = decode_topk_idx(q.to(DEV), cache.kc[i], cache.seqlens_after, _i32(cu), topk=4,
                                      local_blocks=1, cache_seqlens_host=after, cu_seqlens_q_host=cu)
                out, lse = cache.attend(i, q.to(DEV), ids, _i32(cu), return_lse=True)
                ref, ref_lse, bound = lo.attend(want[i], q, after, cu, ids.cpu())
                _check(out, lse, ref, ref_lse, bound, torch.bfloat16)
                assert plain.attend(i, q.to(DEV), ids, _i32(cu)).shape == out.shape
        for c in (cache, plain):
            c.end()
        lens = after
        # Each key within e4m3's half step (relative, or half a subnormal step of the page's scale),
        # so the compressed keys within the mean of that, and a rounding on either side.
        for i in range(layers):
            for b in range(3):
                n = n_windows(lens[b])
                if not n:
                    continue
                x = plain.k[i, b, :lens[b]].double().cpu()
                pages = torch.arange(lens[b]) // 64
                step = 2.0 ** (want[i].kcode[b][pages].double() - 127 - 10)[..., None]
                # Twice: a row may have been brought under a raised code.
                off = 2 * (2.0 ** -4 * x.abs()).maximum(step) * (1 + 2.0 ** -4)
                tol = off.unfold(0, 32, 16).mean(-1) + 2.0 ** -7 * (x.abs() + off).unfold(0, 32, 16).mean(-1)
                d = (cache.kc[i, b, :n].double() - plain.kc[i, b, :n].double()).abs().cpu()
                assert bool((d <= tol).all()), (i, b, (d - tol).max().item())


def test_model_decodes_over_an_8_bit_cache():
    """Logits of decode steps over both caches: close, as 8 bits of keys and values allow, and
    the step's attention equal to the operators' on the cache."""
    cfg = minicpm.MiniCPMConfig(hidden_size=1024, num_hidden_layers=2, num_attention_heads=8,
                                num_key_value_heads=2, intermediate_size=2048, vocab_size=4096,
                                topk=64, local_blocks=4)
    model = minicpm.MiniCPMLeanSelect(cfg, device=DEV, seed=3)
    g = torch.Generator(device=DEV).manual_seed(11)
    ids = torch.randint(0, 4096, (817,), generator=g, device=DEV, dtype=torch.int32)
    caches = [model.new_cache(2, 1024, kv_format=f) for f in ("native", "q8")]
    first = [model.prefill(ids, [0, 300, 817], cache=c) for c in caches]
    assert torch.equal(first[0], first[1])  # a prefill does not read the cache
    for _ in range(6):
        tok = torch.randint(0, 4096, (2,), generator=g, device=DEV, dtype=torch.int32)
        a, b = (model.decode_step(tok, c) for c in caches)
        assert bool(torch.isfinite(b).all())
        rel = ((a - b).norm() / a.norm()).item()
        # Keys and values off by 2^-4 at most each, in two of the residual stream's layers.
        assert rel < 2 * 2 * 2.0 ** -4, rel
    assert caches[1].lengths == [306, 523]
