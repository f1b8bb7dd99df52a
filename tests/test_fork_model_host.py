"""What the model refuses of a forked cache, before any GPU call (CPU only)."""
from types import SimpleNamespace

import pytest
import torch

from leanselect_amd.cache import LeanSelectKVCache
from leanselect_amd.minicpm import MiniCPMLeanSelect


def _prompt(length=70):
    cache = LeanSelectKVCache(2, 1, 128, 2, device="cpu")
    if length:
        cache.begin([length])
        cache.end()
    return cache


@pytest.mark.parametrize("batch", [1, 3])
def test_a_fork_is_not_prefilled(batch):
    """Its sequences hold the prompt already: their next tokens do not stand at position 0."""
    fork = _prompt().fork(batch, 10)
    ids = torch.zeros(2 * batch, dtype=torch.int32)
    cu = list(range(0, 2 * batch + 1, 2))
    with pytest.raises(ValueError, match="empty cache"):
        MiniCPMLeanSelect.prefill(SimpleNamespace(cfg=None), ids, cu, cache=fork)
    assert fork.positions == [70] * batch
    fork.begin([1] * batch)  # no step was left open
    with pytest.raises(ValueError, match="empty cache"):
        MiniCPMLeanSelect.prefill(SimpleNamespace(cfg=None), ids, cu, cache=_prompt())
    with pytest.raises(RuntimeError, match="GPU"):  # an empty one is taken
        MiniCPMLeanSelect.prefill(SimpleNamespace(cfg=None), ids[:2], cache=_prompt(0))


@pytest.mark.parametrize("sampling,error", [
    (dict(return_logprob=True), TypeError), (dict(temperature=-1.0), ValueError), (dict(top_p=0.0), ValueError),
    (dict(top_k=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(), RuntimeError)], ids=str)
def test_settings_are_checked_before_the_prompts_pass(sampling, error):
    model = SimpleNamespace(new_cache=lambda *a: pytest.fail("a cache was made"))
    with pytest.raises(error):
        MiniCPMLeanSelect.generate(model, torch.zeros(5, dtype=torch.int32), torch.zeros(4, 3), **sampling)
