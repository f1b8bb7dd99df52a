"""The bounds under which sampling looks for what is kept, where they fall on zero, on logits that lie
close together or on the smallest numbers: the same tokens as the definition's (oracle/serving_oracle.py)."""
import math

import pytest
import torch

from leanselect_amd.ops import sample_logits
from test_gpu_sampling import DEV, DTYPES, _check

pytestmark = pytest.mark.gpu

_U = torch.tensor([0.0, 0.1, 0.37, 0.52, 0.7, 0.83, 0.96, 1.0 - 2.0 ** -24])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5000, 73448])
@pytest.mark.parametrize("settings", [dict(top_k=50), dict(top_k=1500), dict(top_k=50, top_p=0.9), dict(top_k=50, min_p=0.01),
                                      dict(top_k=1500, top_p=0.99, temperature=2.0)], ids=str)
def test_a_few_logits_above_zeros(dtype, vocab, settings):
    """The border falls among logits of 0 and -0, with none below and with some."""
    x = torch.zeros(8, vocab, dtype=dtype)
    x[:, ::7] = -0.0
    x[:, [10, 300, 4000]] = torch.tensor([1.0, 3.0, 2.0], dtype=dtype)
    x[4:, 1::2] = -1.0
    assert _check(x, _U, **settings) >= 7


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 100, 5000, 73448])
@pytest.mark.parametrize("more", [dict(), dict(top_k=50), dict(top_k=50, top_p=0.9), dict(top_p=0.9), dict(temperature=0.3)], ids=str)
def test_a_largest_logit_of_zero_alone(dtype, vocab, more):
    """min_p of 1 keeps the largest logits, also where they are 0 and -0."""
    g = torch.Generator().manual_seed(vocab)
    x = (-0.5 - torch.rand(8, vocab, generator=g)).to(dtype)
    x[:, vocab // 2] = 0.0
    x[4:, vocab // 3] = -0.0
    assert _check(x, _U, min_p=1.0, **more) >= 7
    assert _check(x, _U, min_p=torch.ones(8), **more) >= 7
    above = sample_logits(x.to(DEV), _U.to(DEV), min_p=torch.full((8,), 1.5, device=DEV), **more).cpu()
    assert torch.equal(above, sample_logits(x.to(DEV), _U.to(DEV), min_p=1.0, **more).cpu())


@pytest.mark.parametrize("offset,eps", [(100.0, 1e-3), (1e6, 1.0), (20.0, 1e-4), (1000.0, 1e-2), (20.0, 1e-3), (-1e6, 1.0), (3e30, 1e24)])
@pytest.mark.parametrize("settings", [dict(top_k=1), dict(top_k=50), dict(top_k=200, top_p=0.8), dict(top_k=1500),
                                      dict(top_k=50, min_p=0.9)], ids=str)
def test_logits_within_a_few_steps_of_each_other(offset, eps, settings):
    g = torch.Generator().manual_seed(3)
    x = offset + eps * torch.randn(8, 73448, generator=g)
    temperature = max(1.0, eps)
    assert _check(x, _U, temperature=temperature, **settings) >= 7


@pytest.mark.parametrize("settings", [dict(top_k=2), dict(top_k=50), dict(top_k=1500, top_p=0.5)], ids=str)
@pytest.mark.parametrize("value", [1.0, -1.0, 20.0])
def test_two_neighbouring_values(value, settings):
    """One logit a step above all others, which are equal."""
    x = torch.full((8, 9000), value)
    x[:, 4321] = torch.nextafter(x[0, 0], torch.tensor(math.inf))
    assert _check(x, _U, **settings) >= 7


@pytest.mark.parametrize("settings", [dict(top_k=50), dict(top_k=1500), dict(top_k=50, top_p=0.5)], ids=str)
@pytest.mark.parametrize("scale", [1e-36, 1e-37, 1e-40, 1e-44])
def test_the_smallest_logits(scale, settings):
    """Logits whose range's reciprocal float32 does not hold, a single one above zeros among them."""
    g = torch.Generator().manual_seed(4)
    x = scale * torch.randn(8, 9000, generator=g)
    x[4:] = 0.0
    x[4:, 777] = scale
    assert _check(x, _U, **settings) >= 7


@pytest.mark.parametrize("settings", [dict(top_k=2), dict(top_k=50), dict(top_k=1500, top_p=0.5)], ids=str)
def test_two_neighbouring_small_values(settings):
    test_two_neighbouring_values(1e-30, settings)


@pytest.mark.parametrize("scale,temperature", [(1e-38, 1e-38), (1e-37, 1e-37), (1e-40, 3e-40), (1e-38, 1e-30), (1.0, 1e-40)])
@pytest.mark.parametrize("settings", [dict(top_p=0.5), dict(top_p=0.9, min_p=0.02), dict(top_k=5000, top_p=0.5)], ids=str)
def test_the_smallest_temperatures(scale, temperature, settings):
    """Temperatures whose reciprocal float32 does not hold, with weights that matter."""
    g = torch.Generator().manual_seed(5)
    x = scale * torch.randn(8, 10007, generator=g)
    assert _check(x, _U, temperature=temperature, **settings) >= 7


@pytest.mark.parametrize("offset", [0.0, 1e6, -3e7, 1e9])
def test_a_draw_next_to_an_edge_far_from_zero(offset):
    """A weight goes by the distance from the largest logit, which a common offset does not change: numbers
    2^-38 to 2^-29 from the edge between two tokens, on both sides of it."""
    t = torch.linspace(0.5, 3.0, 60001)
    step = 2.0 ** max(1, math.frexp(offset)[1] - 23)  # (representable apart)
    t = t * step
    edge = 1.0 / (1.0 + torch.exp(-step / t.double()))
    u = edge.float()
    gap = (u.double() - edge).abs()
    near = (gap > 2.0 ** -38) & (gap < 2.0 ** -29)
    t, u = t[near], u[near]
    x = torch.tensor([[offset, offset - step]]).expand(len(t), 2).contiguous()
    assert len(t) > 500
    assert _check(x, u, temperature=t) == len(t)
