"""Calls that a launch of 2^32 - 1 threads along a dimension does not hold are refused by name
before any launch (CPU: the C entry points, with addresses that nothing reads)."""
from leanselect_amd import _hip

B = _hip.LS_BF16


def _refused(rc, word):
    return rc == _hip.LS_ERR_UNSUPPORTED and word in _hip.lib().ls_last_error()


def _attend(total, splits, q=16):
    return _hip.lib().ls_attn_kvcache_q8(
        q, 128, 4, total, 16, 16, 16384, 1, 1, 2, 1 << 12, 4, 1, 1, 1, 128, B, None, 1 << 12, 1.0, 0,
        splits, 16, None, 16, 1 << 60, None)


def test_attention_rows():
    most = (2 ** 32 - 1) // 512
    for splits in (1, 2, 256):
        assert _refused(_attend(most // splits + 1, splits), b"too many rows")
        # One fewer is looked at further.
        assert _attend(most // splits, splits, q=None) == _hip.LS_ERR_INVALID
        assert b"null" in _hip.lib().ls_last_error()


def test_append_tokens():
    append = lambda total, k=16: _hip.lib().ls_kvcache_append_q8(  # noqa: E731
        16, 16, 16384, 1, 1, 2, 1 << 24, 4, k, k, 128, 4, total, 1, 1, 128, B, None, 0, 0, 0, None)
    assert _refused(append(2 ** 32 // 256 * 64), b"too many new tokens")
    assert _refused(append(2 ** 40), b"too many new tokens")


def test_weights():
    linear = lambda n: _hip.lib().ls_linear_mx4(  # noqa: E731
        16, 8, 1, 8, 16, 4, n, 0, B, 16, n, None, 0, None)
    quantize = lambda n, k: _hip.lib().ls_quantize_mx4(16, k, n, k, B, 16, 4, None)  # noqa: E731
    assert _refused(linear(2 ** 30), b"too many outputs")
    assert _refused(quantize(2 ** 28, 8), b"too large")
    assert _refused(quantize(2 ** 21, 2 ** 17), b"too large")
