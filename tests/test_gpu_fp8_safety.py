"""Calls of the operators in 8-bit floating point whose operands move while they run."""
import ctypes as C

import pytest
import torch

import inferflow_amd as ia
from tests.gpu_util import capi, sync
from tests.test_gpu_fp8_ops import expert_case, gen

pytestmark = pytest.mark.gpu


class Graph:
    """a captured call with a copy put behind its first kernel"""

    def __init__(self, call, dst, src):
        self.hip = hip = capi()          # (the HIP runtime that the library is linked to)
        self.stream, self.graph, self.run = torch.cuda.Stream(), C.c_void_p(), C.c_void_p()
        s = C.c_void_p(self.stream.cuda_stream)
        self.ok(hip.hipStreamBeginCapture(s, 2))          # (relaxed)
        call(self.stream.cuda_stream)
        self.ok(hip.hipStreamEndCapture(s, C.byref(self.graph)))
        n = C.c_size_t(0)
        self.ok(hip.hipGraphGetEdges(self.graph, None, None, C.byref(n)))
        frm, to = (C.c_void_p * n.value)(), (C.c_void_p * n.value)()
        self.ok(hip.hipGraphGetEdges(self.graph, frm, to, C.byref(n)))
        self.launches = n.value + 1
        first = [k for k in range(n.value) if frm[k] not in list(to)]
        assert len(first) == 1          # (a chain)
        first, second = C.c_void_p(frm[first[0]]), C.c_void_p(to[first[0]])
        node = C.c_void_p()
        self.ok(hip.hipGraphAddMemcpyNode1D(C.byref(node), self.graph, C.byref(first), C.c_size_t(1), C.c_void_p(dst.data_ptr()), C.c_void_p(src.data_ptr()), C.c_size_t(dst.numel() * dst.element_size()), 3))
        self.ok(hip.hipGraphAddDependencies(self.graph, C.byref(node), C.byref(second), C.c_size_t(1)))
        self.ok(hip.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, C.c_size_t(0)))

    @staticmethod
    def ok(rc):
        assert rc == 0, rc

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.run, C.c_void_p(self.stream.cuda_stream)))
        sync()

    def close(self):
        self.ok(self.hip.hipGraphExecDestroy(self.run)); self.ok(self.hip.hipGraphDestroy(self.graph))


def test_places_are_given_out_as_they_were_counted():
    """Tiles of experts, five launches.  Choices that change behind the first one (it counts the rows of each expert) do not move the places that the second one gives out: the call is as with the choices that
    were counted, and neither lists nor rows are written past their ends."""
    rows, width, ff, E, top = 600, 256, 192, 6, 3
    a, sa, gu, sgu, down, sdown, idx, wgt = expert_case(rows, width, ff, E, top, 11)
    n = capi().ifa_moe_experts_fp8_workspace_bytes(rows, top, width, ff, E)
    ws = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")

    def call(y, idx, stream):
        ia.check(capi().ifa_moe_experts_fp8(0, 7.0, a.data_ptr(), width, sa.data_ptr(), sa.shape[1], rows, width, ff, E, top, gu.data_ptr(), sgu.data_ptr(), down.data_ptr(), sdown.data_ptr(), idx.data_ptr(),
                                            wgt.data_ptr(), ws.data_ptr(), n, 0, y.data_ptr(), width, 0, stream))
    others = [torch.full_like(idx, 2), torch.full_like(idx, -1), torch.where(torch.rand(idx.shape, generator=gen(4), device="cuda") < 0.5, idx, (idx + 1) % E), torch.full_like(idx, 1 << 30)]
    want = torch.empty(rows, width, device="cuda")
    call(want, idx, torch.cuda.current_stream().cuda_stream); sync()
    for other in others:
        moving, y = idx.clone(), torch.empty(rows, width, device="cuda")
        sync()
        graph = Graph(lambda stream: call(y, moving, stream), moving, other)
        assert graph.launches == 5
        for _ in range(3):
            moving.copy_(idx); y.fill_(7.0); sync()
            graph.replay()
            assert torch.equal(moving, other) and torch.equal(y, want) and (ws[n:] == 0x5A).all()
        graph.close()
