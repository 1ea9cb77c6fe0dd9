"""What the sums of the experts in 8-bit floating point hold: their hidden activations, seen through a second matrix that is the identity, and the second product of these."""
import pytest
import torch

from tests import fp8_oracle as orc
from tests.fp8_plans import limit_32
from tests.gpu_util import sync
from tests.test_gpu_fp8_ops import F8, TYPES, experts, expert_case, gen

pytestmark = pytest.mark.gpu


def identity_case(rows, width, ff, E, seed):
    """one expert a row, weight 1, its second matrix the identity: y is the quantised activation times its scale, in one product each"""
    a, sa, gu, sgu, _, _, idx, _ = expert_case(rows, width, ff, E, 1, seed)
    one = torch.eye(ff, device="cuda").to(F8).expand(E, ff, ff).contiguous()
    return a, sa, gu, sgu, one, torch.ones(E, orc.blocks(ff), orc.blocks(ff), device="cuda"), idx, torch.ones(rows, 1, device="cuda")


# one and four choices as pairs, lists, tiles of 128 places and (the last) of 192
IDENTITY = [(1, 2048, 2048, 2), (4, 1024, 1024, 3), (40, 1040, 1040, 3), (200, 512, 512, 8), (700, 640, 640, 2), (1300, 384, 384, 1), (2600, 1152, 1152, 16)]


@pytest.mark.parametrize("rows,width,ff,E", IDENTITY)
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_hidden_activations_are_the_same_whatever_the_output_type(rows, width, ff, E, kind):
    """A product of the second matrix has one term that is not 0, so 8-bit instructions give it exactly: a 16-bit output is the 32-bit one rounded, if the activations behind both are the same."""
    a, sa, gu, sgu, down, sdown, idx, wgt = identity_case(rows, width, ff, E, rows + kind)
    y = {}
    for dtype in (0, 1, 2):
        y[dtype] = torch.full((rows, width), 3.0, device="cuda").to(TYPES[dtype])
        experts(kind, a, sa, width, gu, sgu, down, sdown, idx, wgt, dtype, y[dtype], 0)
    sync()
    assert torch.equal(y[1], y[0].to(torch.float16)) and torch.equal(y[2], y[0].to(torch.bfloat16))


@pytest.mark.parametrize("rows,width,ff,E", IDENTITY)
def test_hidden_activations_have_sums_of_32_bits(rows, width, ff, E):
    """A block's largest activation is 448 times its scale, which no rounding to e4m3 touches; the test above says that the other types have the same.  Against 64 bits, all blocks together: a gate or up is a
    sum of at most 17 blocks' sums, 8 waves' among them, the activation a dozen roundings behind it, each off by 2^-24 of what it rounds at most and no two alike: sqrt(2 * 17 + 12) 2^-24 < 2^-21 of terms that
    do not cancel; 2^-20 with as much again for those that do.  Sums without what lies below 2^-13 of the largest of eight terms are 2^-16 off."""
    a, sa, gu, sgu, down, sdown, idx, wgt = identity_case(rows, width, ff, E, rows)
    y = torch.zeros(rows, width, device="cuda")
    experts(0, a, sa, width, gu, sgu, down, sdown, idx, wgt, 0, y, 0); sync()
    v = torch.empty(rows, ff, dtype=torch.float64, device="cuda")
    for e in range(E):
        t = (idx[:, 0] == e).nonzero()[:, 0]
        at = orc.values(a.float()[t], sa[t])
        g, u = (at @ orc.matrix_values(gu[e, i], sgu[e, i]).t() for i in (0, 1))
        v[t] = orc.gated(0, g, u)
    want = 448 * orc.scales(v)
    got = torch.stack([p.abs().amax(-1) for p in y.double().split(128, -1)], -1)
    assert float((got - want).norm()) <= 2.0 ** -20 * float(want.norm())


@pytest.mark.parametrize("rows,width,ff,E", IDENTITY)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_the_second_product_has_sums_of_32_bits_for_32_bit_outputs(rows, width, ff, E, accumulate):
    """The hidden activations as the identity shows them (each one rounding, 2^-24, off) times another second matrix, in 64 bits; then a weight's product and an addition: three roundings beside a product's."""
    a, sa, gu, sgu, one, sone, idx, wgt = identity_case(rows, width, ff, E, rows + 5)
    hidden = torch.zeros(rows, width, device="cuda")
    experts(0, a, sa, width, gu, sgu, one, sone, idx, wgt, 0, hidden, 0)
    down, sdown = orc.matrix(width, ff, 9, count=E, std=ff ** -0.5)
    wgt = torch.randn(rows, 1, generator=gen(2), device="cuda")
    y0 = torch.randn(rows, width, generator=gen(3), device="cuda")
    y = y0.clone()
    experts(0, a, sa, width, gu, sgu, down, sdown, idx, wgt, 0, y, accumulate); sync()
    want = torch.empty(rows, width, dtype=torch.float64, device="cuda")
    for e in range(E):
        t = (idx[:, 0] == e).nonzero()[:, 0]
        want[t] = hidden[t].double() @ orc.matrix_values(down[e], sdown[e]).t() * wgt[t].double()
    full = want + (y0.double() if accumulate else 0.0)
    assert float((y.double() - full).norm()) <= (limit_32(orc.blocks(ff)) + 2 * 2.0 ** -24) * float(want.norm()) + 2.0 ** -24 * float(full.norm())
