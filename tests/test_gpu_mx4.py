"""4-bit weights on the GPU: laying out byte for byte, products against 64-bit ones within the
roundings of float32 sums and of the output's type."""
import math

import pytest
import torch

from leanselect_amd import minicpm
from leanselect_amd.ops import (dequantize_mx4, lay_out_mx4, linear_mx4, linear_mx4_silu_mul,
                                quantize_mx4)
from oracle import lowbit_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weight(n, k, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(n, k, generator=g) * 0.02
    return w * torch.exp(spread * torch.randn(n, 1, generator=g))


def _values(n, k, seed, low=110, high=130):
    """Random 4-bit values and codes, the kernel's tensors and the float64 weight."""
    g = torch.Generator().manual_seed(seed)
    values = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    codes = torch.randint(low, high + 1, (n, -(-k // 32)), generator=g, dtype=torch.uint8)
    laid = lay_out_mx4(values.to(DEV), codes.to(DEV))
    return laid, lo.e2m1_weight(values, codes)


def _check(got, x, w, silu=False):
    """|error| <= half a step of the output's type, plus float32 sums: at most K / 32 matrix
    instructions in a chain, 32 products in each, and the waves' sums (2^-24 of the sum of
    magnitudes for each addition on the longest path)."""
    x = x.double().cpu()
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    d = size * (x.shape[1] / 32 + 64) * 2.0 ** -24
    eps = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    if silu:
        gate, up = y.chunk(2, -1)
        dg, du = d.chunk(2, -1)
        s = gate * torch.sigmoid(gate)
        # |silu'| <= 1.1; the exponential and the quotient in float32.
        d = 1.1 * dg * (up.abs() + du) + s.abs() * du + (s * up).abs() * (gate.abs() + 8) * 2.0 ** -22
        y = s * up
    err = (got.cpu().double() - y).abs()
    tol = eps * y.abs() + d * (1 + eps) + tiny
    assert got.shape == y.shape
    assert bool((err <= tol).all()), f"largest excess {(err - tol).max().item():.3e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (17, 136), (40, 520), (33, 1048)])
def test_quantize_is_the_definition_byte_for_byte(dtype, n, k):
    w = _weight(n, k, n * k).to(dtype)
    w[0, :32] = 0.0
    if k > 32:
        w[0, 32:64] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 4)
        w[n - 1, -8:] = -torch.finfo(dtype).max
    values, codes = lo.e2m1_codes(w)
    want = lo.tile_bytes(values, codes)
    got = quantize_mx4(w.to(DEV))
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    wide = torch.zeros(n, k + 24, dtype=dtype, device=DEV)
    wide[:, 8:k + 8] = w
    again = quantize_mx4(wide[:, 8:k + 8])
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(1, 8), (19, 136), (33, 1048)])
def test_quantize_reads_rows_of_any_place_and_stride(dtype, n, k):
    w = _weight(n, k, n + k).to(dtype).to(DEV)
    want = quantize_mx4(w)
    for at, cols in ((0, k), (1, k + 1), (3, k + 8), (8, k + 8), (4, k + 4), (0, k + 5)):
        wide = torch.full((n, at + cols), math.nan, dtype=dtype, device=DEV)
        wide[:, at:at + k] = w
        got = quantize_mx4(wide[:, at:at + k])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (at, cols)


@pytest.mark.parametrize("n,k", [(1, 8), (17, 136), (40, 520)])
def test_dequantize_gives_the_values(n, k):
    (codes, scales), w = _values(n, k, n + k, 8, 252)
    assert torch.equal(dequantize_mx4(codes, scales, n, k).cpu().double(), w)
    assert torch.equal(dequantize_mx4(codes, scales, n, k, torch.float16).cpu(), w.half())
    (codes, scales), w = _values(n, k, n + k, 104, 140)
    assert torch.equal(dequantize_mx4(codes, scales, n, k, torch.float16).cpu().double(), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 2, 7, 15, 16, 17, 31, 33, 64, 65, 200])
def test_linear_at_every_row_count(dtype, m):
    n, k = 40, 1096
    (codes, scales), w = _values(n, k, m)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype)
    _check(linear_mx4(x.to(DEV), codes, scales, n), x, w)


@pytest.mark.parametrize("n,k", [(1, 8), (3, 32), (16, 120), (17, 128), (31, 136), (48, 504), (100, 512),
                                 (129, 520), (64, 2056), (30, 5000), (21, 16384)])
@pytest.mark.parametrize("m", [1, 5, 40])
def test_linear_at_odd_sizes(n, k, m):
    (codes, scales), w = _values(n, k, n * k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)).bfloat16()
    _check(linear_mx4(x.to(DEV), codes, scales, n), x, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inter,k", [(16, 8), (48, 520), (512, 4096)])
@pytest.mark.parametrize("m", [1, 16, 19, 70])
def test_silu_mul(dtype, inter, k, m):
    w32 = _weight(2 * inter, k, inter, 0.3)
    codes, scales = quantize_mx4(w32.to(DEV))
    w = lo.e2m1_weight(*lo.e2m1_codes(w32))
    x = (2 * torch.randn(m, k, generator=torch.Generator().manual_seed(m))).to(dtype)
    _check(linear_mx4_silu_mul(x.to(DEV), codes, scales, 2 * inter), x, w, silu=True)


@pytest.mark.parametrize("n,k,m", [
    (4608, 264, 1), (4624, 264, 9),        # two tiles a workgroup of eight waves
    (16400, 136, 1), (16400, 136, 16),     # four tiles a workgroup of four
    (16400, 128, 17), (16390, 120, 70),    # the same, 32 rows a workgroup
    (16640, 512, 1), (32768, 264, 5),      # shared rows, one slice
    (48, 8200, 3), (2048, 8192, 40),       # shared rows, slices and their join
    (2048, 2056, 130), (48, 16400, 3), (100, 12296, 15),
    (4096, 2056, 33), (16384, 1032, 40), (40, 4104, 20)])
def test_linear_in_each_form(n, k, m):
    (codes, scales), w = _values(n, k, n + 2 * k + m)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    _check(linear_mx4(x.to(DEV), codes, scales, n), x, w)


@pytest.mark.parametrize("n,k,m", [(16896, 128, 2), (16896, 120, 40), (32800, 72, 16), (20480, 512, 1),
                                   (2048, 8200, 5), (2048, 2056, 33), (2048, 16392, 5),
                                   (512, 4104, 17)])
def test_silu_mul_in_each_form(n, k, m):
    (codes, scales), w = _values(n, k, n + 3 * k + m, 112, 122)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    _check(linear_mx4_silu_mul(x.to(DEV), codes, scales, n), x, w, silu=True)


def test_scales_at_the_ends_of_their_range():
    for code in (8, 60, 200, 250):
        (codes, scales), w = _values(24, 264, code, code, code)
        x = torch.randn(3, 264, generator=torch.Generator().manual_seed(1)) * 2.0 ** (127 - code)
        x = x.bfloat16()
        if bool(torch.isfinite(x).all()):
            _check(linear_mx4(x.to(DEV), codes, scales, 24), x, w)


def test_rows_do_not_depend_on_each_other():
    """A row's result is the same bits whatever shares the call, NaN and infinities included."""
    n, k = 72, 1024
    (codes, scales), _ = _values(n, k, 5)
    x = torch.randn(64, k, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    alone = torch.cat([linear_mx4(x[i:i + 1], codes, scales, n) for i in range(64)])
    bad = x.clone()
    bad[1] = math.nan
    bad[40] = math.inf
    out = linear_mx4(bad, codes, scales, n)
    keep = [i for i in range(64) if i not in (1, 40)]
    assert torch.equal(out[keep], alone[keep])
    assert bool(torch.isnan(out[1]).all()) and not bool(torch.isfinite(out[40]).any())
    assert torch.equal(linear_mx4(x, codes, scales, n), alone)


@pytest.mark.parametrize("n,k,m", [(40, 136, 3), (40, 1032, 20), (48, 8200, 3), (16384, 264, 18), (48, 16392, 3)])
def test_an_infinity_among_the_last_inputs(n, k, m):
    """The padding past the last input is no zero times infinity: an output is NaN only where the
    infinite input meets a weight of zero."""
    (codes, scales), w = _values(n, k, n + k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    x[1, k - 1], x[m - 1, k - 3] = math.inf, -math.inf
    got, want = linear_mx4(x.to(DEV), codes, scales, n).cpu().double(), x.double() @ w.t()
    for row in (1, m - 1):
        assert torch.equal(torch.isnan(got[row]), torch.isnan(want[row]))
        finite = ~torch.isnan(want[row])
        assert torch.equal(got[row][finite], want[row][finite])  # infinities of the same sign
    keep = [i for i in range(m) if i not in (1, m - 1)]
    _check(linear_mx4(x.to(DEV), codes, scales, n)[keep], x[keep], w)


def test_strided_rows_and_outputs():
    n, k, m = 50, 264, 6
    (codes, scales), _ = _values(n, k, 8)
    wide = torch.randn(m, 2 * k + 8, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV)
    for x in (wide[:, :k], wide[:, 8:k + 8], wide[:, 3:k + 3], wide[:, ::2][:, :k], wide[::2, :k],
              wide[:, :k].t().contiguous().t()):
        want = linear_mx4(x.contiguous().clone(), codes, scales, n)
        assert torch.equal(linear_mx4(x, codes, scales, n), want)
        for cols, at in ((n, 0), (n + 6, 0), (n + 9, 1), (n + 9, 5)):
            out = torch.full((x.shape[0], cols), 5.0, dtype=torch.bfloat16, device=DEV)
            got = linear_mx4(x, codes, scales, n, out=out[:, at:at + n])
            assert got.data_ptr() == out[:, at:].data_ptr()
            assert torch.equal(out[:, at:at + n], want)
            assert bool((out[:, :at] == 5.0).all()) and bool((out[:, at + n:] == 5.0).all())


def test_no_rows():
    (codes, scales), _ = _values(16, 32, 1)
    x = torch.empty(0, 32, dtype=torch.bfloat16, device=DEV)
    assert linear_mx4(x, codes, scales, 16).shape == (0, 16)


def test_captured_and_replayed():
    n, k = 96, 1024
    (codes, scales), _ = _values(n, k, 10)
    g = torch.Generator().manual_seed(11)
    x = torch.randn(4, k, generator=g).bfloat16().to(DEV)
    linear_mx4(x, codes, scales, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_mx4(x, codes, scales, n)
        act = linear_mx4_silu_mul(x, codes, scales, n)
    for _ in range(3):
        x.copy_(torch.randn(4, k, generator=g))
        graph.replay()
        assert torch.equal(out, linear_mx4(x, codes, scales, n))
        assert torch.equal(act, linear_mx4_silu_mul(x, codes, scales, n))
        torch.cuda.synchronize()


def test_weights_that_are_not_finite_are_refused():
    for bad in (math.inf, math.nan):
        w = torch.zeros(16, 32, device=DEV)
        w[3, 3] = bad
        with pytest.raises(ValueError, match="finite"):
            quantize_mx4(w)


def _small_model(seed):
    cfg = minicpm.MiniCPMConfig(hidden_size=1024, num_hidden_layers=2, num_attention_heads=8,
                                num_key_value_heads=2, intermediate_size=2048, vocab_size=4100,
                                topk=64, local_blocks=4)
    return minicpm.MiniCPMLeanSelect(cfg, device=DEV, seed=seed)


def test_model_with_4_bit_weights_is_the_model_of_their_values():
    """A quantised model's prefill (library products of the values) and decode steps (4-bit
    products) against the same model whose 16-bit weights are those values."""
    a, b = _small_model(5).quantize_weights(), _small_model(5)
    for L in b.layers:
        for name in ("w_qkv", "w_o", "w_gate_up", "w_down"):
            w = getattr(L, name)
            setattr(L, name, dequantize_mx4(*quantize_mx4(w), *w.shape))
    b.lm_head = dequantize_mx4(*quantize_mx4(b.lm_head), *b.lm_head.shape)
    assert a.quantize_weights() is a  # again: nothing left to do
    g = torch.Generator(device=DEV).manual_seed(12)
    lens = [300, 600]
    ids = torch.randint(0, 4100, (sum(lens),), generator=g, device=DEV, dtype=torch.int32)
    for kv in ("native", "q8"):
        caches = [m.new_cache(2, 1024, kv_format=kv) for m in (a, b)]
        got, want = (m.prefill(ids, [0, 300, 900], cache=c) for m, c in zip((a, b), caches))
        # Prefill of 900 rows: the same library products, so the same bits.
        assert torch.equal(got, want)
        for _ in range(3):
            tok = torch.randint(0, 4100, (2,), generator=g, device=DEV, dtype=torch.int32)
            got, want = (m.decode_step(tok, c) for m, c in zip((a, b), caches))
            rel = ((got - want).norm() / want.norm()).item()
            # Two layers whose 16-bit roundings (2^-9 each, some ten a layer) may differ.
            assert rel < 20 * 2.0 ** -9, (kv, rel)
