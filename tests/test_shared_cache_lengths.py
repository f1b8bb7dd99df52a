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
