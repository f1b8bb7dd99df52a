"""How far a capped score, and with it the float32 lse, is from cap tanh(x / cap): rows that see one key."""
import pytest
import torch

from leanselect_amd.ops import dense_attention_kvcache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("cap", [0.5, 30.0, 50.0, 128.0, 512.0])
def test_within_cap_2_21(dtype, rows, cap):
    """z = 1 / (1 + 2^y): y is off by 2^-23 of itself (a factor's and a product's rounding), which moves z by 0.23 2^-23 at
    most; the exponential's unit moves it by 2^-25, the sum's rounding and the reciprocal's unit by 2^-24 and 2^-23 of z.
    The score is 2 cap z away from cap: cap 2^-21 in all, and a few roundings of itself.  The weight's two parts hold
    2^-17 of it in bf16, 2^-21 in fp16; its exponent, formed of two roundings, is below 8 in bf16, 16 in fp16, whose lse
    takes 10 off the maximum and adds a logarithm of 10 to 15: ln 2 (2 2^-22) and ln 2 (4 2^-21)."""
    n = 300
    g = torch.Generator().manual_seed(int(cap))
    a = (cap * torch.randn(n, generator=g) * torch.logspace(-3, 1, n)).to(dtype)
    q, k = torch.zeros(n, 1, 128, dtype=dtype), torch.zeros(1, 1, 1, 128, dtype=dtype)
    q[:, 0, 5], k[..., 5] = a, 1.0  # one exact product
    for i in range(0, n, rows):
        _, lse = dense_attention_kvcache(q[i:i + rows].to(DEV), k.to(DEV), k.to(DEV), torch.tensor([1], dtype=torch.int32, device=DEV),
                                         torch.tensor([0, rows], dtype=torch.int32, device=DEV), 1, softmax_scale=1.0, softcap=cap,
                                         return_lse=True)
        want = cap * torch.tanh(a[i:i + rows].double() / cap)
        off = (lse[0].cpu().double() - want).abs()
        weight = 2.0 ** -17 + 1.4 * 2.0 ** -22 if dtype == torch.bfloat16 else 2.0 ** -21 + 2.8 * 2.0 ** -21
        assert bool((off <= cap * 2.0 ** -21 + 2.0 ** -21 * want.abs() + weight).all())
