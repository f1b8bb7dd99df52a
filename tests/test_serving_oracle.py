"""The 64-bit forms of attention over a cache and of sampling against plain loops and torch's attention."""
import math

import pytest
import torch

from oracle import serving_oracle as so


def _inputs(seed=0, lens=(9, 5), new=(3, 2), H=4, G=2, prefix=0):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return (f(cu[-1], H, 128), f(len(lens), max(lens), G, 128), f(len(lens), max(lens), G, 128), list(lens), cu,
            f(prefix, G, 128), f(prefix, G, 128))


@pytest.mark.parametrize("prefix", [0, 6])
@pytest.mark.parametrize("options", [
    dict(), dict(causal=True), dict(softcap=2.0), dict(alibi=True), dict(window=(2, -1)), dict(window=(1, 1)),
    dict(causal=True, window=(3, 0), softcap=1.5, alibi=True, softmax_scale=0.3)], ids=str)
def test_attention_against_a_loop_over_keys(prefix, options):
    q, k, v, lens, cu, kp, vp = _inputs(prefix=prefix)
    options = dict(options)
    slopes = torch.tensor([0.5, 0.25, 0.125, 1.0]) if options.pop("alibi", False) else None
    more = dict(k_prefix=kp, v_prefix=vp) if prefix else {}
    out, lse, _, _ = so.cache_attention(q, k, v, lens, cu, alibi_slopes=slopes, **more, **options)
    scale, cap = options.get("softmax_scale", 128 ** -0.5), options.get("softcap", 0.0)
    left, right = options.get("window", (-1, -1))
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            p = prefix + length - n + i
            for h in range(4):
                total, acc = 0.0, torch.zeros(128, dtype=torch.float64)
                for j in range(prefix + length):
                    if options.get("causal") and j > p or left >= 0 and j < p - left or right >= 0 and j > p + right:
                        continue
                    key, value = (kp[j, h // 2], vp[j, h // 2]) if j < prefix else \
                        (k[b, j - prefix, h // 2], v[b, j - prefix, h // 2])
                    x = scale * float(key @ q[cu[b] + i, h])
                    if cap:
                        x = cap * math.tanh(x / cap)
                    if slopes is not None:
                        x -= float(slopes[h]) * abs(p - j)
                    total += math.exp(x)
                    acc += math.exp(x) * value
                assert math.isclose(lse[h, cu[b] + i], math.log(total), rel_tol=1e-12, abs_tol=1e-12)
                assert torch.allclose(out[cu[b] + i, h], acc / total, rtol=1e-11, atol=1e-13)


def test_attention_against_torch():
    q, k, v, lens, cu, _, _ = _inputs(3, lens=(40,), new=(40,), H=2, G=2)
    out, _, bound, _ = so.cache_attention(q, k, v, lens, cu, causal=True)
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), is_causal=True).transpose(0, 1)
    assert torch.allclose(out, want, rtol=1e-10, atol=1e-12)
    assert bool((bound > 0).all())


def test_a_row_without_keys():
    q, k, v, _, cu, _, _ = _inputs()
    out, lse, _, _ = so.cache_attention(q, k, v, [0, 5], cu)
    assert bool((out[:3] == 0).all()) and bool((lse[:, :3] == math.inf).all()) and bool(torch.isfinite(lse[:, 3:]).all())


def test_a_missing_cap_is_seen():
    q, k, v, lens, cu, _, _ = _inputs()
    plain, _, bound, _ = so.cache_attention(q, k, v, lens, cu)
    capped = so.cache_attention(q, k, v, lens, cu, softcap=1.0)[0]
    assert bool(((plain - capped).abs() > bound).any())


@pytest.mark.parametrize("settings", [
    (1.0, 0, 1.0, 0.0), (0.7, 3, 1.0, 0.0), (1.3, 0, 0.6, 0.0), (1.0, 0, 1.0, 0.2), (0.9, 5, 0.8, 0.1), (2.0, 4, 0.3, 0.0)],
    ids=str)
def test_sampling_against_a_loop(settings):
    t, top_k, top_p, min_p = settings
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, generator=g).double().tolist()
    x[7] = x[2]
    w = [math.exp((a - max(x)) / t) for a in x]
    order = sorted(range(12), key=lambda i: (-x[i], i))
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        run, total, kept = 0.0, sum(w[i] for i in order), []
        for i in order:
            kept.append(i)
            run += w[i]
            if run >= top_p * total:
                break
        order = kept
    order = sorted(i for i in order if w[i] >= min_p)
    for u in (0.0, 0.1, 0.35, 0.6, 0.85, 0.999):
        total, run = sum(w[i] for i in order), 0.0
        for i in order:
            run += w[i]
            if run > u * total:
                break
        token, logprob, sure, _ = so.sample_row(x, u, t, top_k, top_p, min_p)
        assert sure and token == i
        assert math.isclose(logprob, math.log(w[i] / total), rel_tol=1e-12, abs_tol=1e-12)


def test_sampling_edges():
    inf = math.inf
    assert so.sample_row([math.nan, -inf], 0.5, 1.0, 0, 1.0, 0.0)[:2] == (-1, -inf)
    assert so.sample_row([1.0, 3.0, 3.0, math.nan], 0.9, 0.0, 0, 1.0, 0.0)[:2] == (1, 0.0)
    assert so.sample_row([1.0, inf, 3.0, inf], 0.6, 1.0, 0, 1.0, 0.0)[:2] == (3, math.log(0.5))
    # a draw on the very edge between two tokens is not sure
    assert not so.sample_row([0.0, math.log(3.0)], 0.25, 1.0, 0, 1.0, 0.0)[2]
