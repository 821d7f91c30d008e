"""Options that the products on operands held in few bits follow, on a B200: how many CTAs their kernels are launched with."""
import ctypes

import pytest
import torch

from test_gpu_codes import BF16, F32, check, gradient_case, product_case
from wmma_extension_b200 import tcec

pytestmark = pytest.mark.gpu


def grids(call):
    """CTAs of each kernel that `call` launches, from a captured graph of it."""
    cuda, p = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    count = ctypes.c_size_t(0)
    raw = p(graph.raw_cuda_graph())
    assert cuda.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (p * count.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    found = []
    for node in nodes:
        kind, params = ctypes.c_int(-1), (ctypes.c_uint32 * 64)()  # function (64 bits), then grid and block
        assert cuda.cuGraphNodeGetType(p(node), ctypes.byref(kind)) == 0 and kind.value == 0
        assert cuda.cuGraphKernelNodeGetParams_v2(p(node), params) == 0
        found.append(params[2] * params[3] * params[4])
    graph.reset()
    return found


# tokens, outputs, inputs: the staging has few CTAs, the products without the option more than there are SMs to take
@pytest.mark.parametrize("m,n,k,dtype", [(1000, 4, 8192, BF16), (1000, 16, 2300, BF16), (1000, 16, 8200, BF16), (900, 10, 16500, F32), (1000, 40, 30000, BF16)])
def test_gradients_leave_sms_to_others(m, n, k, dtype):
    dy, packed, exact, tol = gradient_case(m, n, k, dtype, n, F32)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    check(tcec.wgrad_q8(dy, packed, k, dtype=F32), exact, tol)
    for reserve in (20, 64):
        tcec.set_option("reserve_sms", reserve)
        try:
            got = tcec.wgrad_q8(dy, packed, k, dtype=F32)
            seen = grids(lambda: tcec.wgrad_q8(dy, packed, k, dtype=F32))
        finally:
            tcec.set_option("reserve_sms", 0)
        check(got, exact, tol)
        assert len(seen) >= 2 and max(seen) <= sms - reserve, seen
    tcec.device_status()


def test_prompts_leave_sms_to_others():
    x, packed, exact, tol = product_case(40, 30000, 1024, 128, BF16, 53)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tcec.set_option("reserve_sms", 20)
    try:
        check(tcec.gemm_q4(x, packed, 30000), exact, tol)
        seen = grids(lambda: tcec.gemm_q4(x, packed, 30000))
    finally:
        tcec.set_option("reserve_sms", 0)
    assert len(seen) == 2 and max(seen) <= sms - 20, seen


def test_gradients_in_several_launches_are_captured_and_replayed():
    dy, packed, exact, tol = gradient_case(1000, 16, 16500, BF16, 83, F32)
    c = torch.zeros(16, 16500, device=dy.device)
    tcec.wgrad_q8(dy, packed, 16500, c)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    tcec.set_option("reserve_sms", 20)
    try:
        tcec.wgrad_q8(dy, packed, 16500, c.zero_())
        once = c.clone()
        with torch.cuda.graph(graph):
            tcec.wgrad_q8(dy, packed, 16500, c)
            tcec.wgrad_q8(dy, packed, 16500, c, beta=1.0)
    finally:
        tcec.set_option("reserve_sms", 0)
    check(once, exact, tol)
    for _ in range(3):
        c.zero_()
        graph.replay()
        assert torch.equal(c, once + once)
    tcec.device_status()
