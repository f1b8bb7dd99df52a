"""The 64-bit forms of the 8-bit cache and the 4-bit weights against other ways of saying the
same, and the layout helper that needs no GPU."""
import math

import pytest
import torch

from leanselect_amd.ops import lay_out_mx4
from oracle import lowbit_oracle as lo


def test_e4m3_rounding_is_torchs():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(4000, generator=g) * 100, torch.linspace(-448, 448, 3001),
                   torch.randn(4000, generator=g) * 0.01, lo.e4m3_values().float(),
                   (lo.e4m3_values()[1:] + lo.e4m3_values()[:-1]).float() / 2]).clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).double()
    assert torch.equal(lo.e4m3_round(x.double()), want)
    bad = lo.e4m3_round(torch.tensor([math.inf, -math.inf, math.nan], dtype=torch.float64))
    assert bool(bad.isnan().all())


def test_scale_codes_at_the_borders():
    assert lo.scale_code(448.0, 448.0, 1) == 127 and lo.scale_code(448.0001, 448.0, 1) == 128
    assert lo.scale_code(6.0, 6.0, 8) == 127 and lo.scale_code(6.1, 6.0, 8) == 128
    assert lo.scale_code(0.0, 448.0, 1) == 1


def test_place_is_its_own_inverse():
    assert [lo.place(lo.place(t)) for t in range(64)] == list(range(64))
    assert sorted(lo.place(t) for t in range(64)) == list(range(64))


def test_e2m1_ties_go_to_the_even_code():
    w = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0] + [0.0] * 22])
    values, codes = lo.e2m1_codes(w)
    assert codes.tolist() == [[127]]
    assert values[0, :10].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 8, 14]


@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (17, 136), (40, 520), (33, 1048)])
def test_lay_out_places_every_value(n, k):
    g = torch.Generator().manual_seed(n + k)
    values = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    codes = torch.randint(100, 140, (n, -(-k // 32)), generator=g, dtype=torch.uint8)
    got = lay_out_mx4(values, codes)
    want = lo.tile_bytes(values, codes)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lay_out_refuses_what_the_kernel_does_not_read():
    v = torch.zeros(4, 32, dtype=torch.uint8)
    s = torch.full((4, 1), 127, dtype=torch.uint8)
    for bad in (0, 7, 253, 255):
        with pytest.raises(ValueError, match="8..252"):
            lay_out_mx4(v, torch.full_like(s, bad))
    with pytest.raises(ValueError, match="0..15"):
        lay_out_mx4(v + 16, s)
    with pytest.raises(ValueError, match="scale_codes"):
        lay_out_mx4(v, s.expand(4, 2))
    with pytest.raises(ValueError, match="multiple of 8"):
        lay_out_mx4(v[:, :31], s)


def test_append_raises_a_page_and_keeps_the_older_rows():
    """A later, larger row raises the page's code; the older rows still stand for their values
    to e4m3's half step, and a sequence's untouched pages stay."""
    g = torch.Generator().manual_seed(5)
    z = torch.zeros(1, 2, 1, 64, 128).to(torch.float8_e4m3fn)
    code = torch.full((1, 2, 1), 99, dtype=torch.uint8)
    c = lo.Q8Cache(z, z.transpose(-1, -2), code, code)
    a = torch.randn(10, 1, 128, generator=g).double()
    c.append([0], a, a, [0, 10])
    c.append([10], 50 * a[:1], 50 * a[:1], [0, 1])
    got = c.keys(0, 0)[:11]
    want = torch.cat([a, 50 * a[:1]])[:, 0]
    step = 2.0 ** (float(c.kcode[0, 0, 0]) - 127 - 9)
    # Two roundings: 2^-4 relative each, or half a subnormal step.
    assert bool(((got - want).abs() <= 2 * (2.0 ** -4 * want.abs() * (1 + 2.0 ** -4)).clamp(min=step)).all())
    assert int(c.kcode[0, 1, 0]) == 99


def test_e2m1_codes_end_where_bf16_does():
    top = torch.finfo(torch.float32).max
    values, codes = lo.e2m1_codes(torch.tensor([[top, -top, 1e38] + [0.0] * 29]))
    assert codes.tolist() == [[252]] and values[0, :3].tolist() == [7, 15, 4]
    w = lo.e2m1_weight(values, codes)[0, :3]
    assert torch.equal(w.bfloat16().double(), w) and bool(torch.isfinite(w.float()).all())
