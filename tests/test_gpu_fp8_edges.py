"""The operators in 8-bit floating point at the ends of what they take: one column block's sixteenth, one matrix row, the most rows, the most columns, the most experts."""
import pytest
import torch

from tests import fp8_oracle as orc
from tests.gpu_util import sync
from tests.test_gpu_fp8_ops import FLIPS, NORM_ERR, TYPES, check_product, check_quantised, codes, expert_case, experts, gen, glu, linear, norm, room, route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,rows,cols", [(1, 1, 16), (17, 1, 16), (5000, 1, 16), (1000000, 1, 16), (1000000, 17, 32), (40, 70000, 16), (33, 1, 65536), (2, 16, 1 << 20), (70, 16, (1 << 22) + 16)])
def test_products(tokens, rows, cols):
    a, sa = orc.quantised(tokens, cols, tokens)
    w, sw = orc.matrix(rows, cols, rows)
    for dtype in (0, 2):
        c = torch.full((tokens + 1, rows), 6.0, device="cuda").to(TYPES[dtype])
        linear(w, sw, a, sa, tokens, cols, None, 0, dtype, c, room(rows, cols, tokens)); sync()
        want, bound = orc.product(a, sa, w, sw, dtype == 0)
        check_product(c[:tokens], want, bound, dtype)
        assert (c[tokens] == 6.0).all()


@pytest.mark.parametrize("rows,cols", [((1 << 22) - 1, 16), (100001, 32)])
@pytest.mark.parametrize("dtype", [0, 2])
def test_many_short_rows_of_a_norm(rows, cols, dtype):
    g = gen(rows)
    x0, m = (torch.randn(rows, cols, generator=g, device="cuda").to(TYPES[dtype]) for _ in range(2))
    x, q, scale = x0.clone(), codes(rows + 1, cols), torch.full((rows + 1, 1), 3.0, device="cuda")
    norm(dtype, x, m, None, 1.0, 1e-5, cols, None, q, scale); sync()
    want = (x0.float() + m.float()).to(TYPES[dtype])
    assert torch.equal(x, want) and (q[rows] == 0x55).all() and (scale[rows] == 3.0).all()
    v = want.double()
    check_quantised(q[:rows], scale[:rows], v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5), NORM_ERR)


@pytest.mark.parametrize("rows,cols", [(1 << 22, 16), (3, 1 << 22)])
def test_activations(rows, cols):
    gu = torch.randn(rows, 2 * cols, generator=gen(1), device="cuda").to(torch.bfloat16)
    q, scale = codes(rows + 1, cols), torch.full((rows + 1, orc.blocks(cols)), 3.0, device="cuda")
    glu(2, 2, gu, cols, q[:rows], scale[:rows]); sync()
    v = gu[:, :cols].double().clamp_min(0) * gu[:, cols:].double()
    check_quantised(q[:rows], scale[:rows], v, 2.0 ** -24)
    assert (q[rows] == 0x55).all() and (scale[rows] == 3.0).all()


@pytest.mark.parametrize("rows,n,groups,top", [((1 << 25) - 1, 2, 1, 1), (300001, 64, 8, 6), (7, 1024, 16, 64), (5, 1024, 1, 64), (3, 1, 1, 1)])
def test_router(rows, n, groups, top):
    z = torch.randn(rows, n, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda")
    idx, wgt = route(1, groups, max(1, groups // 2), 2, True, 1e-20, 1.0, z, None, top); sync()
    pick = torch.arange(rows)[-40:]
    want_i, want_w = orc.route(1, groups, max(1, groups // 2), 2, True, 1e-20, 1.0, z[pick.cuda()].cpu(), None, top)
    assert torch.equal(idx[pick.cuda()].cpu(), want_i) and ((wgt[pick.cuda()].cpu().double() - want_w).abs() <= 2.0 ** -24 * (1 + 1e-6) * want_w).all()
    assert (idx >= 0).all() and (idx < n).all() and ((wgt.sum(-1) - 1).abs() < 1e-5).all()


@pytest.mark.parametrize("rows,width,ff,E,top", [(1, 16, 16, 1, 1), (3, 16, 16, 2, 2), (40, 16, 16, 4, 1), (700, 16, 16, 3, 2), (100000, 16, 16, 5, 3), (2, 48, 16, 1024, 64), (30, 48, 16, 1024, 64), (100, 32, 48, 1024, 64), (70, 65536, 16, 4, 1),
                                                 (700, 65536, 16, 2, 1), (1, 16, 65536, 4, 1), (9, 16, 65536, 4, 2), (2, 256, 4112, 8, 2), (40, 256, 4096, 8, 2)])
def test_experts(rows, width, ff, E, top):
    a, sa, gu, sgu, down, sdown, idx, wgt = expert_case(rows, width, ff, E, top, rows + width)
    bounds = {wide: orc.experts(0, a, sa, gu, sgu, down, sdown, idx, wgt, wide) for wide in (True, False)}
    for dtype in (0, 2):
        y = torch.full((rows + 1, width), 4.0, device="cuda").to(TYPES[dtype])
        ws_rows = y[:rows]
        experts(0, a, sa, width, gu, sgu, down, sdown, idx, wgt, dtype, ws_rows, 0); sync()
        want, bound = bounds[dtype == 0]
        check_product(y[:rows], want, bound, dtype, extra=2.0 ** -24 * (want.abs() + 8), loose=FLIPS)
        assert (y[rows] == 4.0).all()


@pytest.mark.parametrize("bad", [-float("inf"), float("nan")])
def test_experts_whose_correction_takes_them_out(bad):
    """as if their logits were -inf: not taken, nothing added to their group (sigmoid scores, so that the others' stay)"""
    z, out = torch.randn(50, 32, generator=torch.Generator().manual_seed(1)), [0, 5, 8, 9, 10, 11, 12, 13, 14, 15, 31]
    corr = 0.1 * torch.randn(32, generator=torch.Generator().manual_seed(2))
    masked, taken_out = z.clone(), corr.clone()
    masked[:, out], taken_out[out] = -float("inf"), bad
    a, b = (route(1, 4, 3, 2, True, 1e-20, 1.0, *args, 12) for args in ((z, taken_out), (masked, corr)))
    sync()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not set(a[0].flatten().tolist()) & set(out)
