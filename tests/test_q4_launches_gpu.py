"""Products with weights of 4 bits: the launches that a call counts are those that it makes."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def nodes_of(graph) -> int:
    n = ctypes.c_size_t(0)
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("T,n,k", [(1, 256, 256), (64, 3584, 1024), (200, 640, 512), (700, 3584, 4096), (2048, 3584, 18944)])
def test_every_launch_is_counted(T, n, k):
    from tensorline_b200 import ops, ops_q4
    w = ops_q4.quantize(torch.ones(n, k, dtype=torch.bfloat16, device="cuda")).settle()
    x = torch.ones(T, k, dtype=torch.bfloat16, device="cuda")
    ops_q4.gemm_q4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = ops.launch_count()
    with torch.cuda.graph(graph):
        ops_q4.gemm_q4(x, w)
    counted = ops.launch_count() - before
    assert counted == nodes_of(graph)
    assert counted > 1 or T != 700
