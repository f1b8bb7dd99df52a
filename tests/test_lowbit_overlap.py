"""Memory that a call both reads and writes, or writes twice, is refused wherever it overlaps
(CPU only: nothing is launched)."""
import random

import pytest
import torch

from leanselect_amd import _hip
from leanselect_amd.ops import (dense_attention_kvcache_q8, kvcache_append_q8, linear_mx4,
                                linear_mx4_silu_mul, new_kvcache_q8, sparse_attention_kvcache_q8)

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(_hip, "gpu_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "launch", lambda index, name, *args: calls.append(name))
    return calls


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_rows_overlap_is_the_bytes_that_are_shared():
    rng = random.Random(1)
    for _ in range(6000):
        sides = []
        for _ in range(2):
            width, rows = rng.randint(1, 6), rng.randint(0, 5)
            stride = rng.choice((width, width + rng.randint(0, 12), rng.randint(1, 20)))
            sides.append((rng.randint(0, 50), max(1, stride), rows, width))
        if rng.random() < 0.5:  # rows of one buffer
            sides[1] = (sides[1][0], sides[0][1], *sides[1][2:])
        at = [{start + i * stride + c for i in range(rows) for c in range(width)}
              for start, stride, rows, width in sides]
        assert _hip.rows_overlap(*sides[0], *sides[1]) == bool(at[0] & at[1]), sides


@pytest.mark.parametrize("product,n_out", [(linear_mx4, 128), (linear_mx4_silu_mul, 64)])
def test_an_output_among_the_rows_it_is_formed_of(launched, product, n_out):
    codes = torch.zeros(8, 1, 64, 16, dtype=torch.uint8)
    scales = torch.zeros(8, 1, 64, 4, dtype=torch.uint8)
    buf = torch.zeros(8, 512, dtype=BF16)
    flat = torch.zeros(4096, dtype=BF16)
    bad = [(buf[1:, :128], buf[:-1, :n_out]), (buf[:, 128:256], buf[:, 200:200 + n_out]),
           (flat[:1024].view(8, 128), flat[1016:1016 + 8 * n_out].view(8, n_out)),
           (buf[0, :128].expand(3, 128), buf[:3, 120:120 + n_out]),
           (buf[::2, :128], buf[2:6, 64:64 + n_out])]
    for x, out in bad:
        with pytest.raises(ValueError, match="overlap"):
            product(x, codes, scales, 128, out=out)
    assert not launched
    fine = [(buf[:, :128], buf[:, 128:128 + n_out]), (buf[::2, :128], buf[1::2, :n_out]),
            (buf[1:, :128], buf[:-1, 128:128 + n_out]), (buf[0, :128].expand(3, 128), buf[1:4, :n_out]),
            (flat[:1024].view(8, 128), flat[1024:1024 + 8 * n_out].view(8, n_out)),
            (buf[:1, :128], buf[:1, 256:256 + n_out]), (buf[:0, :128], buf[:0, :n_out])]
    for x, out in fine:
        assert product(x, codes, scales, 128, out=out) is out
    assert len(launched) == len(fine)


def test_an_output_among_the_queries(launched):
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    flat = torch.zeros(10, 16, 128, dtype=BF16)
    wide = torch.zeros(2, 24, 128, dtype=BF16)
    n, cu, ids = _i32([3, 3]), _i32([0, 2, 4]), torch.zeros(2, 4, 1, dtype=torch.int32)
    for q, out in ((flat[:4], flat[1:5]), (flat[3:7], flat[:4]), (flat[:1].expand(4, 16, 128), flat[:4]),
                   (flat[::2][:4], flat[3:7])):
        with pytest.raises(ValueError, match="overlap q"):
            dense_attention_kvcache_q8(q, *cache, n, cu, 3, out=out)
        with pytest.raises(ValueError, match="overlap q"):
            sparse_attention_kvcache_q8(q, *cache, n, ids, cu, out=out)
    assert not launched
    dense_attention_kvcache_q8(flat[:4], *cache, n, cu, 3, out=flat[4:8])
    dense_attention_kvcache_q8(wide[:, :16], *cache, n, _i32([0, 1, 2]), 3, out=flat[:2])
    assert len(launched) == 2


def _append(cache, kc=None, total=4):
    x = torch.zeros(total, 2, 128, dtype=BF16)
    kvcache_append_q8(*cache, _i32([3, 0]), x, x, _i32([0, 1, total]), kc_cache=kc)


def test_a_cache_whose_keys_and_values_share_memory(launched):
    k8, v8, ks, vs = new_kvcache_q8(2, 128, 2, device="cpu")
    as_values = k8.view(2, 2, 2, 128, 64)
    pages = torch.zeros(5, *k8.shape[1:], dtype=torch.uint8).view(torch.float8_e4m3fn)
    codes = torch.zeros(5, 2, 2, dtype=torch.uint8)
    for cache in ((k8, as_values, ks, vs), (k8, v8, ks, ks),
                  (pages[:2], pages[1:3].view(2, 2, 2, 128, 64), ks, vs),
                  (pages[:4:2], pages[2:5:2].view(2, 2, 2, 128, 64), codes[:4:2], codes[1:5:2]),
                  (k8, v8, codes[:2], codes[1:3])):
        with pytest.raises(ValueError, match="share pages or scales"):
            _append(cache)
    assert not launched
    # Keys and values of a sequence side by side.
    _append((pages[:4:2], pages[1:5:2].view(2, 2, 2, 128, 64), codes[:4:2], codes[1:5:2]))
    assert len(launched) == 1


def test_compressed_windows_that_overlap(launched):
    cache = new_kvcache_q8(2, 128, 2, device="cpu")
    flat = torch.zeros(8192, dtype=BF16)

    def at(batch, row, capacity=7):
        return flat.as_strided((2, capacity, 2, 128), (batch, row, 128, 1))

    for kc in (at(7 * 256, 0), at(7 * 256, 128), at(6 * 256, 256), at(128, 512), at(256, 256), at(1, 256)):
        with pytest.raises(ValueError, match="windows must not overlap"):
            _append(cache, kc)
    assert not launched
    for kc in (at(7 * 256, 256), at(256, 512), at(6 * 256 + 256, 256), at(4096, 264), at(256, 0, 1)):
        _append(cache, kc)
    assert len(launched) == 5
