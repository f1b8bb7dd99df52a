"""How many slices the 8-bit cache's attention cuts a row into (CPU: the launch is replaced)."""
import pytest
import torch

from leanselect_amd import _hip
from leanselect_amd.ops import dense_attention_kvcache_q8, new_kvcache_q8


@pytest.mark.parametrize("rows,pages,slices", [
    (1, 1, 1), (1, 24, 1), (1, 25, 7), (1, 64, 16), (1, 2048, 128), (2, 2048, 64),
    (48, 24, 1), (17, 32, 7), (24, 32, 1), (24, 33, 5), (32, 32, 1), (48, 32, 1), (48, 63, 2), (56, 63, 2), (64, 63, 1),
    (64, 125, 2), (65, 469, 1), (300, 2048, 1)])
def test_slices_of_rows_of_two_heads(monkeypatch, rows, pages, slices):
    sent = []
    monkeypatch.setattr(_hip, "gpu_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "launch", lambda index, name, *args: sent.append(args))
    cache = [t.expand(rows, *t.shape[1:]) for t in new_kvcache_q8(1, 64 * pages, 2, device="cpu")]
    q = torch.zeros(rows, 2, 128, dtype=torch.bfloat16)
    lens = torch.full((rows,), 64 * pages, dtype=torch.int32)
    cu = torch.arange(rows + 1, dtype=torch.int32)
    dense_attention_kvcache_q8(q, *cache, lens, cu, 64 * pages)
    assert sent[0][18] == pages and sent[0][21] == slices
