"""A tensor that a wrapper copies for the kernels is held until the call has been made: memory given
back before is handed to the next copy (CPU: the library is replaced)."""
import ast
import ctypes
from pathlib import Path

import pytest
import torch

import leanselect_amd
from leanselect_amd import _hip
from leanselect_amd.ops import attention, decode

BF16 = torch.bfloat16
# Entry point: (argument, entries) of its int32 arrays.
ARRAYS = {"ls_kvcache_append": [(4, 2), (8, 3)], "ls_decode_select": [(2, 3), (7, 2)],
          "ls_sparse_attn_kvcache": [(2, 3), (8, 2)], "ls_dense_attn_kvcache": [(2, 3), (8, 2)],
          "ls_stage1_scores": [(2, 3), (6, 3)], "ls_sparse_attn_varlen": [(6, 3), (7, 3)]}


@pytest.fixture
def sent(monkeypatch):
    calls = []

    class Library:
        def __getattr__(self, name):
            def call(*args):
                if name in ARRAYS:
                    calls.append((name, [list((ctypes.c_int32 * n).from_address(args[at]))
                                         for at, n in ARRAYS[name]]))
                    return _hip.LS_OK
                return 16  # a workspace's size
            return call

    monkeypatch.setattr(_hip, "lib", lambda: Library())
    monkeypatch.setattr(_hip, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_hip, "stream_of", lambda device: 0)
    monkeypatch.setattr(_hip, "check_attn_status", lambda *a, **kw: None)
    return calls


def _strided(x):
    return torch.tensor([[v, -7] for v in x], dtype=torch.int32)[:, 0]


def test_strided_lengths_and_offsets_arrive(sent):
    k = torch.zeros(2, 128, 2, 128, dtype=BF16)
    kc = torch.zeros(2, 7, 2, 128, dtype=BF16)
    x, q = torch.zeros(2, 2, 128, dtype=BF16), torch.zeros(2, 32, 128, dtype=BF16)
    ids = torch.zeros(2, 2, 1, dtype=torch.int32)
    lens, cu = _strided([3, 65]), _strided([0, 1, 2])
    decode.kvcache_append(k, k, lens, x, x, cu)
    decode.decode_topk_idx(q, kc, lens, cu, topk=4)
    decode.sparse_attention_kvcache(q, k, k, lens, ids, cu)
    decode.dense_attention_kvcache(q, k, k, lens, cu, 65)
    decode.stage1_scores(q, kc[0], cu, _strided([0, 3, 7]), 4)
    attention.sparse_attention(q, x, x, cu, _strided([0, 0, 2]), 1, 2, ids)
    want = {"ls_kvcache_append": [[3, 65], [0, 1, 2]], "ls_decode_select": [[0, 1, 2], [3, 65]],
            "ls_sparse_attn_kvcache": [[0, 1, 2], [3, 65]], "ls_dense_attn_kvcache": [[0, 1, 2], [3, 65]],
            "ls_stage1_scores": [[0, 1, 2], [0, 3, 7]], "ls_sparse_attn_varlen": [[0, 1, 2], [0, 0, 2]]}
    assert dict(sent) == want


def _copies(call: ast.Call) -> int:
    """``x.contiguous().data_ptr()`` among a call's own arguments."""
    def is_copy(node):
        return (isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute)
                and node.func.attr == "data_ptr" and isinstance(node.func.value, ast.Call)
                and isinstance(node.func.value.func, ast.Attribute)
                and node.func.value.func.attr in ("contiguous", "clone", "to", "float", "int"))
    return sum(map(is_copy, call.args))


@pytest.mark.parametrize("path", sorted(Path(leanselect_amd.__file__).parent.rglob("*.py")),
                         ids=lambda p: p.name)
def test_no_call_is_given_two_copies_that_nothing_holds(path):
    for node in ast.walk(ast.parse(path.read_text())):
        if isinstance(node, ast.Call):
            assert _copies(node) <= 1, f"{path.name}:{node.lineno}"
