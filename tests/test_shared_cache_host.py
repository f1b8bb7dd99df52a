"""The forked cache's protocol and refusals (CPU only)."""
import pytest
import torch

from leanselect_amd.cache import LeanSelectKVCache, SharedPrefixKVCache


def _prompt(length=70, **kw):
    cache = LeanSelectKVCache(2, kw.pop("batch", 1), 128, 2, device="cpu", **kw)
    cache.begin([length] * cache.batch)
    cache.end()
    return cache


def test_a_fork_counts_on_from_the_prompt():
    prompt = _prompt()
    cache = prompt.fork(3, 10)
    assert isinstance(cache, SharedPrefixKVCache) and cache.batch == 3 and cache.capacity == 64
    assert cache.positions == [70] * 3 and cache.lengths == [0] * 3 and prompt.positions == [70]
    assert cache.k_prefix.shape == (2, 70, 2, 128) and cache.k_prefix.data_ptr() == prompt.k.data_ptr()
    cache.begin([1, 2, 0])
    assert cache.lengths_after == [1, 2, 0]
    cache.end()
    assert cache.positions == [71, 72, 70]
    with pytest.raises(ValueError, match="capacity"):
        cache.begin([64, 0, 0])
    with pytest.raises(RuntimeError, match="no cache step"):
        cache.attend(0, torch.zeros(3, 4, 128), torch.zeros(4, dtype=torch.int32))


def test_what_cannot_be_shared():
    with pytest.raises(ValueError, match="prefilled"):
        LeanSelectKVCache(1, 1, 64, 2, device="cpu").fork(2, 10)
    with pytest.raises(ValueError, match="one sequence"):
        _prompt(batch=2).fork(2, 10)
    with pytest.raises(ValueError, match="16-bit"):
        _prompt(kv_format="q8").fork(2, 10)
    with pytest.raises(ValueError, match="16-bit"):
        _prompt().fork(2, 10).fork(2, 10)
    prompt = _prompt()
    prompt.begin([1])
    with pytest.raises(ValueError, match="no step open"):
        prompt.fork(2, 10)
    with pytest.raises(ValueError, match="positive"):
        _prompt().fork(0, 10)
