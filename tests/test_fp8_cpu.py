"""What the operators of a feed-forward in 8-bit floating point refuse: before anything is launched, so without a GPU too."""
import ctypes as C
import math

import pytest
import torch

import inferflow_amd as ia
from tests import fp8_oracle as orc

ARG, DTYPE = -1, -2
P = 1 << 20          # an address on 16 bytes that nothing reads
F32, F16, BF16 = 0, 1, 2


def call(name, good, **changed):
    args = dict(good, **changed)
    assert list(args) == list(good)
    return getattr(ia.lib(), name)(*args.values())


NORM = dict(dtype=F32, x=P, ldx=64, rows=2, cols=64, m=P + 4096, ldm=64, w=P, w_offset=0.0, eps=1e-6, h=P + 8192, ldh=64, q=P, ldq=64, scale=P, lds=1, stream=None)
GLU = dict(kind=0, limit=7.0, dtype=F16, gu=P, ld=128, rows=2, cols=64, q=P, ldq=64, scale=P, lds=1, stream=None)
LINEAR = dict(w=P, sw=P, rows=32, cols=144, a=P, lda=144, sa=P, lds=2, tokens=3, bias=P, accumulate=0, dtype=BF16, c=P, ldc=32, ws=P, ws_bytes=0, stream=None)
ROUTE = dict(score=1, groups=4, kept=2, best=2, renorm=1, eps=0.0, scale=1.0, logits=P, ld=32, rows=3, n_all=32, top=6, corr=None, idx=P, wgt=P, stream=None)
EXPERTS = dict(kind=0, limit=7.0, a=P, lda=64, sa=P, lds=1, rows=3, width=64, ff=48, experts=4, top=2, gu=P, sgu=P, down=P, sdown=P, idx=P, wgt=P, ws=P, ws_bytes=1 << 30, dtype=F32, y=P, ldy=64,
               accumulate=0, stream=None)


@pytest.mark.parametrize("changed", [dict(x=None), dict(q=None), dict(scale=None), dict(rows=0), dict(cols=0), dict(cols=40), dict(cols=32768 + 16, ldx=40000, ldm=40000, ldh=40000, ldq=40000, lds=300),
                                     dict(ldx=48), dict(ldx=66), dict(ldm=48), dict(ldh=48), dict(ldq=56), dict(ldq=72), dict(lds=0), dict(x=P + 4), dict(m=P + 8), dict(h=P + 4), dict(q=P + 8),
                                     dict(w=P + 1), dict(scale=P + 2), dict(h=P), dict(m=P), dict(rows=1 << 22)])
def test_norm_refuses(changed):
    assert call("ifa_norm_add_fp8", NORM, **changed) == ARG and b"ifa_norm_add_fp8" in ia.lib().ifa_last_error()


@pytest.mark.parametrize("changed", [dict(gu=None), dict(q=None), dict(scale=None), dict(kind=-1), dict(kind=5), dict(rows=0), dict(cols=8), dict(ld=64), dict(ld=132), dict(ldq=48), dict(lds=0),
                                     dict(gu=P + 2), dict(q=P + 4), dict(rows=1 << 30)])
def test_activation_refuses(changed):
    assert call("ifa_glu_fp8", GLU, **changed) == ARG and b"ifa_glu_fp8" in ia.lib().ifa_last_error()


@pytest.mark.parametrize("changed", [dict(w=None), dict(sw=None), dict(a=None), dict(sa=None), dict(c=None), dict(rows=0), dict(tokens=0), dict(cols=0), dict(cols=136), dict(lda=128), dict(lda=152),
                                     dict(lds=1), dict(ldc=31), dict(w=P + 8), dict(a=P + 4), dict(c=P + 1), dict(bias=P + 1), dict(sa=P + 2), dict(tokens=1000001), dict(rows=1 << 26, ldc=1 << 26)])
def test_product_refuses(changed):
    assert call("ifa_linear_fp8", LINEAR, **changed) == ARG and b"ifa_linear_fp8" in ia.lib().ifa_last_error()


@pytest.mark.parametrize("changed", [dict(logits=None), dict(idx=None), dict(wgt=None), dict(score=2), dict(groups=0), dict(groups=5), dict(groups=65, n_all=130, ld=130), dict(kept=0), dict(kept=5),
                                     dict(best=0), dict(best=3), dict(top=0), dict(top=17), dict(kept=4, groups=4, n_all=512, ld=512, top=65), dict(n_all=1028, ld=1028), dict(ld=31), dict(rows=0), dict(rows=1 << 25)])
def test_router_refuses(changed):
    assert call("ifa_moe_route_groups_f32", ROUTE, **changed) == ARG and b"ifa_moe_route_groups_f32" in ia.lib().ifa_last_error()


@pytest.mark.parametrize("changed", [dict(a=None), dict(sa=None), dict(gu=None), dict(sgu=None), dict(down=None), dict(sdown=None), dict(idx=None), dict(wgt=None), dict(ws=None), dict(y=None),
                                     dict(kind=4), dict(kind=-1), dict(rows=0), dict(width=72), dict(ff=40), dict(experts=0), dict(experts=1025), dict(top=0), dict(top=65), dict(lda=48), dict(lda=72),
                                     dict(lds=0), dict(ldy=63), dict(ws_bytes=100), dict(ws=P + 8), dict(gu=P + 8), dict(down=P + 1), dict(y=P + 2), dict(rows=600000), dict(width=65536, ff=32768, lda=65536, lds=512, ldy=65536), dict(width=65536, ff=16, lda=65536, lds=512, ldy=65536, rows=300000)])
def test_experts_refuse(changed):
    assert call("ifa_moe_experts_fp8", EXPERTS, **changed) == ARG and b"ifa_moe_experts_fp8" in ia.lib().ifa_last_error()


@pytest.mark.parametrize("name,good", [("ifa_norm_add_fp8", NORM), ("ifa_glu_fp8", GLU), ("ifa_linear_fp8", LINEAR), ("ifa_moe_experts_fp8", EXPERTS)])
@pytest.mark.parametrize("dtype", [-1, 3, 8, 99])
def test_unknown_types_are_refused(name, good, dtype):
    assert call(name, good, dtype=dtype) == DTYPE


def test_workspaces_grow_with_the_work():
    f = ia.lib().ifa_moe_experts_fp8_workspace_bytes
    assert 0 < f(1, 2, 64, 48, 4) <= f(16, 2, 64, 48, 4) <= f(4096, 8, 2048, 1408, 64)
    assert f(0, 2, 64, 48, 4) == f(1, 0, 64, 48, 4) == f(1, 2, -64, 48, 4) == 0


@pytest.mark.parametrize("sizes", [(1000001, 1, 64, 48, 4), (600000, 2, 64, 48, 4), (1 << 62, 4, 64, 48, 4), (1, 65, 64, 48, 4), (1, 2, 72, 48, 4), (1, 2, 64, 40, 4), (1, 2, 65552, 48, 4),
                                   (1, 2, 64, 65552, 4), (1, 2, 64, 48, 1025), (1, 2, 65536, 32768, 4), (300000, 2, 65536, 16, 4)])
def test_sizes_that_are_refused_have_no_workspace(sizes):
    rows, top, width, ff, E = sizes
    assert ia.lib().ifa_moe_experts_fp8_workspace_bytes(*sizes) == 0
    assert call("ifa_moe_experts_fp8", EXPERTS, rows=rows, top=top, width=width, ff=ff, experts=E, lda=width, lds=orc.blocks(width), ldy=width, ws_bytes=1 << 60) == ARG


def test_oracle_rounds_to_e4m3_like_torch():
    v = torch.cat([torch.linspace(-460, 460, 20001, dtype=torch.float64), torch.linspace(-0.07, 0.07, 20001, dtype=torch.float64)])
    every = torch.arange(256, dtype=torch.uint8).view(orc.F8).double()
    every = every[~every.isnan()].unique()
    ties = torch.cat([every, (every[1:] + every[:-1]) / 2])
    for x in (v, ties):
        assert torch.equal(orc.e4m3(x), x.float().to(orc.F8).double())


def test_oracle_route_takes_what_plain_sorting_takes():
    g = torch.Generator().manual_seed(3)
    z, corr = torch.randn(40, 32, generator=g), 0.1 * torch.randn(32, generator=g)
    idx, wgt = orc.route(1, 1, 1, 2, True, 0.0, 1.0, z, corr, 5)
    want = (torch.sigmoid(z.double()) + corr.double()).topk(5, -1).indices
    assert torch.equal(idx.long(), want) and torch.allclose(wgt.sum(-1), torch.ones(40, dtype=torch.float64))
    idx, _ = orc.route(0, 4, 2, 1, False, 0.0, 1.0, z, None, 16)
    best = torch.softmax(z.double(), -1).view(40, 4, 8).amax(-1).topk(2, -1).indices
    assert all(set((idx[t] // 8).tolist()) == set(best[t].tolist()) for t in range(40))
    z[7, :] = -math.inf
    idx, wgt = orc.route(0, 4, 2, 2, True, 0.0, 1.0, z, corr, 5)
    assert idx[7].tolist() == [-1] * 5 and wgt[7].tolist() == [0.0] * 5
