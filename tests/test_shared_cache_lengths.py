"""What a forked cache reports and holds (CPU only)."""
from leanselect_amd.cache import LeanSelectKVCache


def _fork(batch=3, capacity=10, **kw):
    cache = LeanSelectKVCache(2, 1, 128, 2, device="cpu", **kw)
    cache.begin([70])
    cache.end()
    return cache.fork(batch, capacity)


def test_a_sequence_is_as_long_as_its_prefix_and_own_tokens():
    fork = _fork()
    assert fork.get_seq_length() == 70
    fork.begin([1, 4, 0])
    fork.end()
    assert fork.get_seq_length() == 74 and fork.lengths == [1, 4, 0]


def test_no_compressed_keys_are_allocated(monkeypatch):
    """Its attention is dense: none are formed."""
    import torch

    prompt = LeanSelectKVCache(2, 1, 128, 2, device="cpu")
    prompt.begin([70])
    prompt.end()
    shapes, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda shape, **kw: shapes.append(tuple(shape)) or empty(shape, **kw))
    fork = prompt.fork(3, 100)
    assert fork.kc is None and shapes == [(2, 3, 128, 2, 128)] * 2
    assert LeanSelectKVCache(2, 1, 128, 2, device="cpu").kc.shape == (2, 1, 7, 2, 128)
