"""Plans of wider integers reach the decode kernels as the pages they name (CPU: the launch is
replaced)."""
import ctypes

import pytest
import torch

from leanselect_amd import _hip
from leanselect_amd.ops import decode, decode_q8

IDS = [0, 5, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 32, -2 ** 63, 2 ** 63 - 1]
WANT = [0, 5, -1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -1, -1, 2 ** 31 - 1]


def _read(pointer, n):
    return list((ctypes.c_int32 * n).from_address(pointer))


def _plan(layout):
    ids = torch.tensor(IDS, dtype=torch.int64)
    if layout == "strided":
        ids = torch.stack((ids, ids), -1)[:, 0]
    return ids.expand(2, 1, len(IDS)) if layout == "expanded" else ids.repeat(2, 1, 1) \
        if layout == "dense" else torch.stack((ids, ids))[:, None]


@pytest.mark.parametrize("layout", ["dense", "strided", "expanded"])
def test_ids_that_int32_does_not_hold_stay_out_of_range(monkeypatch, layout):
    seen = []
    q = torch.zeros(1, 32, 128, dtype=torch.bfloat16)
    n, cu = torch.tensor([300], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    monkeypatch.setattr(_hip, "gpu_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "launch", lambda index, name, *a: seen.append(_read(a[17], 2 * len(IDS))))
    cache = decode_q8.new_kvcache_q8(1, 320, 2, device="cpu")
    decode_q8.sparse_attention_kvcache_q8(q, *cache, n, _plan(layout), cu)

    class Library:
        @staticmethod
        def ls_sparse_attn_kvcache_workspace_size(*a):
            return 16

        @staticmethod
        def ls_sparse_attn_kvcache(*a):
            seen.append(_read(a[14], 2 * len(IDS)))
            return _hip.LS_OK

    monkeypatch.setattr(_hip, "require_gpu", lambda *t: q.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: 0)
    monkeypatch.setattr(_hip, "lib", lambda: Library)
    k = torch.zeros(1, 320, 2, 128, dtype=torch.bfloat16)
    decode.sparse_attention_kvcache(q, k, k, n, _plan(layout), cu)
    assert seen == [WANT * 2] * 2
