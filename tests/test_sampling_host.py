"""Refusals of sampling, before any GPU call (CPU only)."""
import math

import pytest
import torch

from leanselect_amd import _hip
from leanselect_amd.ops import sample_logits


def _call(logits=None, u=None, **kw):
    sample_logits(torch.zeros(3, 10) if logits is None else logits, torch.zeros(3) if u is None else u, **kw)


def test_well_formed_cpu_arguments_reach_the_device_check():
    for kw in (dict(), dict(temperature=0.0, top_k=-1, top_p=2.0, min_p=1.0), dict(top_k=torch.zeros(3, dtype=torch.int32)),
               dict(temperature=torch.ones(3), top_p=torch.ones(3), min_p=torch.ones(3))):
        with pytest.raises(RuntimeError, match="GPU"):
            _call(**kw)


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(3, 10, dtype=torch.float64)), "logits"),
    (dict(logits=torch.zeros(30)), "logits"),
    (dict(logits=torch.zeros(3, 0)), "vocabulary"),
    (dict(logits=torch.zeros(1, 1).expand(3, (1 << 19) + 1)), "vocabulary"),
    (dict(u=torch.zeros(4)), "u must"),
    (dict(u=torch.zeros(3, dtype=torch.float64)), "u must"),
    (dict(temperature=-0.1), "temperature"),
    (dict(temperature=math.nan), "temperature"),
    (dict(temperature=math.inf), "temperature"),
    (dict(top_k=math.inf), "top_k"),
    (dict(top_k=math.nan), "top_k"),
    (dict(temperature=torch.ones(2)), "temperature"),
    (dict(temperature=torch.ones(3, dtype=torch.bfloat16)), "temperature"),
    (dict(top_k=1.5), "top_k"),
    (dict(top_k=torch.ones(3)), "top_k"),
    (dict(top_k=torch.ones(3, dtype=torch.int64)), "top_k"),
    (dict(top_p=0.0), "top_p"),
    (dict(top_p=-1.0), "top_p"),
    (dict(top_p=math.nan), "top_p"),
    (dict(min_p=-0.1), "min_p"),
    (dict(min_p=1.1), "min_p"),
    (dict(min_p=math.nan), "min_p"),
])
def test_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _call(**change)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), _hip.LS_ERR_INVALID), (dict(vocab=0), _hip.LS_ERR_INVALID),
    (dict(vocab=(1 << 19) + 1), _hip.LS_ERR_UNSUPPORTED), (dict(rows=1 << 22), _hip.LS_ERR_UNSUPPORTED),
    (dict(dtype=7), _hip.LS_ERR_UNSUPPORTED), (dict(t=-1.0), _hip.LS_ERR_INVALID), (dict(t=math.nan), _hip.LS_ERR_INVALID),
    (dict(p=0.0), _hip.LS_ERR_INVALID), (dict(m=2.0), _hip.LS_ERR_INVALID), (dict(logits=None), _hip.LS_ERR_INVALID),
    (dict(u=None), _hip.LS_ERR_INVALID), (dict(tokens=None), _hip.LS_ERR_INVALID), (dict(rows=0, logits=None), _hip.LS_OK),
])
def test_entry_point_refusals(change, code):
    a = dict(logits=16, rs=10, rows=1, vocab=10, dtype=_hip.LS_F32, u=16, t=1.0, k=0, p=1.0, m=0.0, ts=None, ks=None,
             ps=None, ms=None, tokens=16, logprobs=None, stream=None)
    a.update(change)
    assert _hip.lib().ls_sample_logits(*a.values()) == code
