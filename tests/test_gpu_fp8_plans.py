"""Products in 8-bit floating point by every kernel there is for them (tests/fp8_plans.py holds the sizes, tests/test_fp8_plans_cpu.py that they bring each), against the formula in 64 bits: whole and other rows of
output, biases, sums into what is there, neighbours, workspaces, far offsets; and a feed-forward whose products are tiles, captured and on two streams."""
import math

import pytest
import torch

import inferflow_amd as ia
from tests import fp8_oracle as orc
from tests.fp8_plans import PLANS, limit_32, plan
from tests.gpu_util import capi, p, sync
from tests.test_gpu_fp8_ops import Block, HALF_STEP, TYPES, check_product, gen, here, linear, room

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", PLANS, ids=str)
def test_product_by_its_plan(sizes):
    tokens, rows, cols = sizes
    a, sa = orc.quantised(tokens, cols, tokens + cols)
    w, sw = orc.matrix(rows, cols, rows)
    g, nb = gen(tokens * rows), orc.blocks(cols)
    bias = torch.randn(rows, generator=g, device="cuda").to(torch.bfloat16)
    bounds = {wide: orc.product(a, sa, w, sw, wide) for wide in (True, False)}
    for dtype in (0, 1, 2):
        want, bound = bounds[dtype == 0]
        # rows of the matrix's own length (whole 16 bytes, where that is a multiple of 8) with a bias, added to what is there; longer rows without either; and each by itself
        for ldc, biased, accumulate in ((rows, True, 1), (rows + 5, False, 0), (rows + 8, False, 1), (rows + 1, True, 0)):
            c0 = torch.randn(tokens + 1, ldc, generator=g, device="cuda").to(TYPES[dtype])
            c = c0.clone()
            ws = room(rows, cols, tokens)
            ia.check(capi().ifa_linear_fp8(p(w), p(sw), rows, cols, p(a), cols, p(sa), sa.shape[1], tokens, p(bias if biased else None), accumulate, dtype, p(c), ldc, p(ws), ws.numel(), here())); sync()
            full = want + (bias.double() if biased else 0.0) + (c0[:tokens, :rows].double() if accumulate else 0.0)
            check_product(c[:tokens, :rows], full, bound + 2 * 2.0 ** -24 * (want.abs() + 8), dtype)
            if dtype == 0:          # (the bias's and the old value's additions: two roundings more, of values that are no larger than these norms)
                assert float((c[:tokens, :rows].double() - full).norm()) <= limit_32(nb) * float(want.norm()) + 2 * 2.0 ** -24 * float(full.norm())
            assert torch.equal(c[tokens], c0[tokens]) and torch.equal(c[:, rows:], c0[:, rows:])


# 32-bit outputs: a stream, tiles of one part and of several
SOME = [(30, 700, 1040), (128, 4096, 4096), (40, 4096, 4096), (520, 4096, 256), (1030, 4000, 2064), (4097, 137, 8080)]


@pytest.mark.parametrize("sizes", SOME, ids=str)
@pytest.mark.parametrize("dtype", [0, 2])
def test_a_row_is_the_same_every_time_and_whatever_is_beside_it(sizes, dtype):
    tokens, rows, cols = sizes
    a, sa = orc.quantised(tokens, cols, 1)
    w, sw = orc.matrix(rows, cols, 2)
    out = []
    for _ in range(3):
        c = torch.full((tokens, rows), math.nan, device="cuda").to(TYPES[dtype])
        linear(w, sw, a, sa, tokens, cols, None, 0, dtype, c, room(rows, cols, tokens)); sync()
        out.append(c)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    keep = tokens // 2 + 1
    for bad_values, bad_scales in ((True, False), (False, True)):
        a2, sa2 = a.clone(), sa.clone()
        if bad_values:
            a2.view(torch.uint8)[keep:] = 0x7F
        if bad_scales:
            sa2[keep:] = math.nan
        c = torch.zeros(tokens, rows, device="cuda").to(TYPES[dtype])
        linear(w, sw, a2, sa2, tokens, cols, None, 0, dtype, c, room(rows, cols, tokens)); sync()
        assert torch.equal(c[:keep], out[0][:keep]) and c[keep:].isnan().all()
    # and a matrix row that is none touches its column alone
    w2 = w.clone()
    w2.view(torch.uint8)[rows - 3] = 0x7F
    c = torch.zeros(tokens, rows, device="cuda").to(TYPES[dtype])
    linear(w2, sw, a, sa, tokens, cols, None, 0, dtype, c, room(rows, cols, tokens)); sync()
    assert c[:, rows - 3].isnan().all() and torch.equal(c[:, :rows - 3], out[0][:, :rows - 3]) and torch.equal(c[:, rows - 2:], out[0][:, rows - 2:])


@pytest.mark.parametrize("tokens,rows,cols", [(128, 4096, 4096), (40, 4096, 4096), (4097, 137, 8080)])
def test_with_less_or_no_workspace_the_sums_are_the_same_but_for_their_order(tokens, rows, cols):
    a, sa = orc.quantised(tokens, cols, 1)
    w, sw = orc.matrix(rows, cols, 2)
    full = capi().ifa_linear_fp8_workspace_bytes(rows, cols, tokens)
    parts = plan(tokens, rows, cols, 0)[2]
    assert parts > 1 and plan(tokens, rows, cols, 0, 0)[2] == 1
    got, plans = {}, set()
    for n in (full, 2 * tokens * rows * 4, 2 * tokens * rows * 4 - 1, 0):
        ws = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device="cuda")
        c = torch.zeros(tokens, rows, device="cuda")
        ia.check(capi().ifa_linear_fp8(p(w), p(sw), rows, cols, p(a), cols, p(sa), sa.shape[1], tokens, None, 0, 0, p(c), rows, p(ws), n, here())); sync()
        assert (ws[n:] == 0x5A).all()
        got[n] = c
        plans.add(plan(tokens, rows, cols, 0, n))
    assert len(plans) > 1
    for c in got.values():
        assert float((c - got[full]).norm()) <= 2 * limit_32(orc.blocks(cols)) * float(got[full].norm())


@pytest.mark.parametrize("tokens,rows,cols,dtype,ldc", [(520, 4096, 128, 2, (1 << 23) + 8), (520, 4096, 128, 0, (1 << 23) + 4), (40, 4096, 4096, 2, (1 << 27) + 8), (40, 4099, 4112, 1, (1 << 27) + 3)])
def test_tiles_with_offsets_past_32_bits(tokens, rows, cols, dtype, ldc):
    """the last rows of output lie 2^32 values on"""
    form = plan(tokens, rows, cols, dtype)
    assert form[0] > 0 and (form[2] > 1) == (tokens == 40) and tokens * ldc > 1 << 32
    a, sa = orc.quantised(tokens, cols, 1)
    w, sw = orc.matrix(rows, cols, 2)
    c = torch.full((tokens, ldc), 1.0, dtype=TYPES[dtype], device="cuda")
    linear(w, sw, a, sa, tokens, cols, None, 0, dtype, c, room(rows, cols, tokens)); sync()
    want, bound = orc.product(a, sa, w, sw, dtype == 0)
    check_product(c[:, :rows], want, bound, dtype)
    assert (c[:, rows:rows + 64] == 1).all() and (c[:, -64:] == 1).all()


def large(rows, seed):
    """a feed-forward whose two plain products are tiles, the columns of at least one shared out"""
    b = Block(rows, width=4096, ff=4096, E=8, top=2, seed=seed)
    b.router *= 0.25          # (logits of order 1 at this width too)
    forms = [plan(rows, 2 * b.ff, b.width, 0, b.ws.numel()), plan(rows, b.width, b.ff, 0, b.ws.numel())]
    assert all(f[0] > 0 for f in forms)
    return b, forms


@pytest.mark.parametrize("rows", [40, 128, 300])
def test_a_feed_forward_of_tiles(rows):
    b, forms = large(rows, 3)
    assert rows > 128 or any(f[2] > 1 for f in forms)
    b.step(); sync()
    b.check()


@pytest.mark.parametrize("rows", [40, 128])
def test_tiles_captured_and_replayed_beside_eager_work(rows):
    """two captured steps that share a workspace, the planes of the products' parts in it, replayed in turn with eager work and synchronisations between, on new inputs"""
    (b, _), (other, _) = large(rows, 3), large(rows, 8)
    other.ws = b.ws
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(); other.step()
    torch.cuda.current_stream().wait_stream(side)
    sync()
    graphs = []
    for block in (b, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block.step()
        graphs.append(graph)
    for turn in range(4):
        for block, graph in zip((b, other), graphs):
            block.x0.copy_(torch.randn(block.x0.shape, generator=gen(turn), device="cuda"))
            block.x.fill_(math.nan); block.act.fill_(math.nan)
            graph.replay()
            if turn % 2:
                sync()
        sync()
        got = [t.clone() for t in (b.x, other.x, b.act, other.act, b.idx, other.idx)]
        b.step(); sync(); other.step(); sync()
        assert all(torch.equal(u, v) for u, v in zip(got, (b.x, other.x, b.act, other.act, b.idx, other.idx)))
    b.check()


def test_tiles_on_two_streams_at_once():
    blocks, streams = [large(128, s)[0] for s in (1, 2)], [torch.cuda.Stream() for _ in range(2)]
    sync()
    for _ in range(3):
        for block, stream in zip(blocks, streams):
            with torch.cuda.stream(stream):
                block.step()
    sync()
    for block in blocks:
        block.check()
