"""Sampling on the GPU against its definition in 64 bits (oracle/serving_oracle.py): the same tokens
wherever no border lies within the errors that the oracle derives, and their log-probabilities."""
import itertools
import math

import pytest
import torch

from leanselect_amd.ops import sample_logits
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _of_row(value, r):
    return value[r].item() if torch.is_tensor(value) else value


def _check(logits, u, **settings):
    """Every row's token and log-probability; returns how many were sure."""
    kw = {n: v.to(DEV) if torch.is_tensor(v) else v for n, v in settings.items()}
    tokens, logprobs = sample_logits(logits.to(DEV), u.to(DEV), return_logprob=True, **kw)
    assert tokens.dtype == torch.int32 and logprobs.dtype == torch.float32
    tokens, logprobs = tokens.tolist(), logprobs.tolist()
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    sure = 0
    x = logits.float().numpy()
    for r in range(logits.shape[0]):
        want, lp, ok, off = so.sample_row(x[r], u[r].item(), *(_of_row(full[n], r) for n in
                                                               ("temperature", "top_k", "top_p", "min_p")))
        if not ok:
            continue
        sure += 1
        assert tokens[r] == want, (r, tokens[r], want)
        if math.isinf(lp):
            assert logprobs[r] == lp
        else:  # float32's rounding, and the sum's error
            allowed = 2.0 ** -24 * abs(lp) + 2 * off + 1e-12
            assert abs(logprobs[r] - lp) <= allowed, (r, logprobs[r], lp)
    return sure


def _logits(rows, vocab, dtype, seed, spread=2.0, likely=6.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    n = min(vocab, 30)
    at = torch.randint(0, vocab, (rows, n), generator=g)
    x.scatter_add_(1, at, likely + 2.0 * torch.randn(rows, n, generator=g))
    return x.to(dtype), torch.rand(rows, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 300, 1023, 1025, 4097, 12345])
@pytest.mark.parametrize("settings", [
    dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=4.0), dict(top_k=1), dict(top_k=50),
    dict(top_p=0.9), dict(min_p=0.05), dict(top_k=40, top_p=0.8, temperature=0.7),
    dict(top_p=0.95, min_p=0.1, temperature=1.3), dict(top_k=200, min_p=0.02), dict(top_k=1500, top_p=0.7),
    dict(top_k=30, top_p=0.6, min_p=0.3), dict(top_p=1e-6), dict(min_p=1.0), dict(top_k=3000)], ids=str)
def test_settings(dtype, vocab, settings):
    x, u = _logits(6, vocab, dtype, vocab)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    assert _check(x, u, **settings) >= 4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("settings", [
    dict(), dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_p=0.95, temperature=0.7), dict(top_p=0.999),
    dict(min_p=1e-4), dict(top_k=20000, top_p=0.9)], ids=str)
@pytest.mark.parametrize("spread", [0.01, 1.0, 3.0])
def test_a_whole_vocabulary(dtype, settings, spread):
    """Flat rows among them, whose kept set does not fit in LDS."""
    x, u = _logits(3, 73448, dtype, 5, spread, 0.0 if spread < 1 else 6.0)
    assert _check(x, u, **settings) >= 2


def test_the_longest_vocabulary():
    x, u = _logits(2, 1 << 19, torch.bfloat16, 6)
    assert _check(x, u, top_p=0.9) + _check(x, u) + _check(x, u, top_k=7) >= 5
    x, u = _logits(2, (1 << 19) - 3, torch.float32, 6)
    assert _check(x, u) >= 1


@pytest.mark.parametrize("vocab,top_p,count", [(10, 0.5, 5), (1000, 0.25, 250), (20000, 0.5, 10000), (4000, 0.75, 3000)])
def test_equal_logits(vocab, top_p, count):
    """Cuts go by the lowest index: a share of equal weights is exact."""
    x = torch.full((5, vocab), 1.5)
    u = torch.tensor([0.0, 0.2, 0.5, 0.8, 1.0 - 2.0 ** -24])
    assert _check(x, u, top_p=top_p) == 5
    tokens = sample_logits(x.to(DEV), u.to(DEV), top_p=top_p).cpu()
    assert int(tokens[-1]) == count - 1 and int(tokens[0]) == 0
    assert _check(x, u, top_k=count) == 5
    assert _check(x, u, top_k=count, top_p=0.5) == 5


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_at_the_borders(dtype):
    """Logits of few values: every border falls among equal ones."""
    g = torch.Generator().manual_seed(7)
    x = torch.randint(0, 6, (8, 5000), generator=g).to(dtype)
    u = torch.rand(8, generator=g)
    for settings in (dict(top_k=1000), dict(top_k=37), dict(top_p=0.5), dict(top_p=0.9), dict(min_p=math.exp(-1.5)),
                     dict(top_k=2000, top_p=0.5), dict(top_p=0.3, temperature=0.2), dict(top_k=4999)):
        assert _check(x, u, **settings) >= 7


def test_signed_zeros_are_equal():
    x = torch.tensor([[-0.0, 0.0, -1.0, 0.0, -0.0]])
    for u in (0.0, 0.3, 0.6, 0.9):
        assert _check(x, torch.tensor([u]), top_k=2) == 1
    assert _check(x, torch.tensor([0.5]), temperature=0.0) == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("settings", [dict(), dict(top_k=20), dict(top_p=0.9), dict(temperature=0.0), dict(min_p=0.1),
                                      dict(top_k=5000, top_p=0.8)], ids=str)
def test_infinities_and_nan(dtype, settings):
    inf, nan = float("inf"), float("nan")
    x, u = _logits(8, 6000, dtype, 8)
    x[0, ::2] = -inf
    x[1, 1:] = -inf                      # one token left
    x[2] = -inf                          # none
    x[3] = nan
    x[4, 100:] = nan
    x[5, [7, 70, 5000]] = inf            # only these
    x[6, :5990] = torch.finfo(dtype).min
    x[7, 3], x[7, 4] = -inf, nan
    u[0] = 0.0
    assert _check(x, u, **settings) >= 7
    got = sample_logits(x.to(DEV), u.to(DEV), **settings).tolist()
    assert got[1] == 0 and got[2] == got[3] == -1 and got[5] in (7, 70, 5000) and got[6] >= 5990


@pytest.mark.parametrize("settings", [
    dict(temperature=1e-30), dict(temperature=1e-6), dict(temperature=1e20), dict(temperature=1e35), dict(temperature=0.05), dict(top_p=0.5),
    dict(top_p=1.0 - 2.0 ** -24)], ids=str)
@pytest.mark.parametrize("scale,shift", [(1.0, 0.0), (1e-30, 0.0), (1e3, 0.0), (1.0, 1e6), (0.0, -3e38), (1e37, 0.0)])
def test_top_p_at_odd_scales(settings, scale, shift):
    """Where top_p's border falls far from, at or just below the maximum, or the distances overflow."""
    g = torch.Generator().manual_seed(11)
    x = scale * torch.randn(5, 10007, generator=g).clamp(-4, 4) + shift
    x[1, 17], x[2, ::2], x[3, 9000] = float("inf"), -float("inf"), 3e38
    _check(x, torch.rand(5, generator=g), **dict(dict(top_p=0.9), **settings))


def test_masked_tokens_are_never_drawn():
    """A mask of the lowest value leaves no weight, for any number and temperature."""
    x = torch.full((64, 3000), torch.finfo(torch.float32).min)
    x[:, 1234] = 0.0
    u = torch.linspace(0, 1 - 2.0 ** -24, 64)
    for t in (0.01, 1.0, 100.0):
        for more in (dict(), dict(top_p=0.99), dict(top_k=10)):
            tokens = sample_logits(x.to(DEV), u.to(DEV), temperature=t, **more)
            assert bool((tokens == 1234).all())


def test_settings_of_each_row():
    rows = 40
    x, u = _logits(rows, 9000, torch.float32, 9)
    g = torch.Generator().manual_seed(9)

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,), generator=g)]

    settings = dict(temperature=pick([0.0, 0.5, 1.0, 2.0]), top_k=pick([-1, 0, 1, 5, 500, 3000, 100000], torch.int32),
                    top_p=pick([0.2, 0.9, 1.0, 2.0]), min_p=pick([0.0, 0.01, 0.3, 1.0]))
    assert _check(x, u, **settings) >= rows - 2
    assert _check(x, u, **dict(settings, top_k=50, min_p=0.0)) >= rows - 2


def test_numbers_out_of_range_on_the_device():
    """A row's own settings are not checked; they end the search all the same."""
    nan, inf = float("nan"), float("inf")
    x, _ = _logits(6, 2000, torch.float32, 10)
    odd = torch.tensor([nan, -1.0, inf, 0.0, 5.0, -inf])
    for name in ("temperature", "top_p", "min_p"):
        tokens = sample_logits(x.to(DEV), torch.full((6,), 0.5, device=DEV), **{name: odd.to(DEV)}).cpu()
        assert bool(((tokens >= 0) & (tokens < 2000)).all())
    tokens = sample_logits(x.to(DEV), odd.to(DEV)).cpu()
    assert bool(((tokens >= 0) & (tokens < 2000)).all())


def test_strides_and_rows():
    x, u = _logits(5, 777, torch.bfloat16, 11)
    wide = torch.full((5, 1000), float("nan"), dtype=torch.bfloat16)
    wide[:, 5:782] = x
    want = sample_logits(x.to(DEV), u.to(DEV), top_p=0.8)
    assert torch.equal(want, sample_logits(wide.to(DEV)[:, 5:782], u.to(DEV), top_p=0.8))
    assert torch.equal(want, sample_logits(x.t().contiguous().to(DEV).t(), u.to(DEV), top_p=0.8))
    both = torch.stack((u, u), 1).to(DEV)
    assert torch.equal(want, sample_logits(x.to(DEV), both[:, 0], top_p=0.8))
    one = torch.cat([sample_logits(x[r:r + 1].to(DEV), u[r:r + 1].to(DEV), top_p=0.8) for r in range(5)])
    assert torch.equal(want, one)
    assert torch.equal(want[:1].expand(5), sample_logits(x[:1].to(DEV).expand(5, 777), u[:1].to(DEV).expand(5), top_p=0.8))
    assert sample_logits(x[:0].to(DEV), u[:0].to(DEV)).shape == (0,)


def test_the_distribution_is_followed():
    """Evenly spaced numbers meet each token as often as its share, to one draw."""
    x = torch.tensor([[0.0, 2.0, 1.0, -1.0, 0.5, 1.5]])
    n = 4000
    u = (torch.arange(n) + 0.5) / n
    for settings, kept in ((dict(), [0, 1, 2, 3, 4, 5]), (dict(top_k=3), [1, 2, 5]), (dict(min_p=0.2), [1, 2, 4, 5])):
        tokens = sample_logits(x.expand(n, 6).to(DEV), u.to(DEV), **settings).cpu()
        w = torch.zeros(6, dtype=torch.float64)
        w[kept] = torch.exp(x[0, kept].double())
        counts = torch.bincount(tokens, minlength=6).double()
        assert bool(((counts - n * w / w.sum()).abs() <= 1.0).all()), counts


def test_every_combination_agrees_with_itself():
    """A call with several cuts draws from the run that the tightest leaves."""
    x, u = _logits(4, 5000, torch.float32, 12)
    for k, p, m in itertools.product((0, 25), (1.0, 0.7), (0.0, 0.1)):
        assert _check(x, u, top_k=k, top_p=p, min_p=m, temperature=0.9) >= 3
