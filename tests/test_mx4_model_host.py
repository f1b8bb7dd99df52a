"""Replacing a model's weights by 4-bit ones, without the kernels (CPU)."""
import math

import pytest
import torch

from leanselect_amd import minicpm
from leanselect_amd.minicpm import MiniCPMConfig, MiniCPMLeanSelect, Mx4Weight

NAMES = ("w_qkv", "w_o", "w_gate_up", "w_down")


def _model():
    m = object.__new__(MiniCPMLeanSelect)
    m.cfg, m.layers = MiniCPMConfig(), [minicpm._Layer() for _ in range(2)]
    for layer in m.layers:
        for name in NAMES:
            setattr(layer, name, torch.ones(16, 8))
    m.lm_head = torch.ones(16, 8)
    return m


def _weights(m):
    return [getattr(layer, name) for layer in m.layers for name in NAMES] + [m.lm_head]


@pytest.fixture(autouse=True)
def laid(monkeypatch):
    """Laying out as the kernels do it, as far as refusing goes."""
    def lay(w):
        if not bool(torch.isfinite(w).all()):
            raise ValueError("weight must be finite")
        return Mx4Weight(w, w, *w.shape)

    monkeypatch.setattr(minicpm, "_mx4", lay)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [0, 5, 7, 8])
def test_a_weight_that_is_not_finite_leaves_the_model_as_it_was(at, bad):
    m = _model()
    before = _weights(m)
    before[at][3, 5] = bad
    with pytest.raises(ValueError, match="finite"):
        m.quantize_weights()
    assert all(a is b for a, b in zip(_weights(m), before))


def test_every_weight_is_replaced_once():
    m = _model()
    assert m.quantize_weights() is m
    first = _weights(m)
    assert all(isinstance(w, Mx4Weight) for w in first)
    m.quantize_weights()
    assert all(a is b for a, b in zip(_weights(m), first))
