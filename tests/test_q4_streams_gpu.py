"""Products with 4-bit weights whose clusters share SMs with products that take all of their tensor memory, on two streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,n,k", [(20, 640, 256), (32, 1280, 256), (60, 640, 256), (100, 1024, 4096)])
def test_clusters_beside_products_in_pairs(T, n, k):
    from tensorline_b200 import ops_gemm, ops_q4
    assert any(kernel == "gemm_q4" and ranges > 1 for _, kernel, _, ranges in ops_q4.plan(T, n, k, torch.cuda.get_device_properties(0).multi_processor_count))
    g = torch.Generator().manual_seed(T)
    w = ops_q4.quantize(torch.randn(n, k, generator=g).cuda()).settle()
    x = torch.randn(T, k, generator=g).to(torch.bfloat16).cuda()
    h, wide = torch.randn(1536, 2048, generator=g).to(torch.bfloat16).cuda(), torch.randn(4096, 2048, generator=g).to(torch.bfloat16).cuda()
    few, many = ops_q4.gemm_q4(x, w), ops_gemm.gemm_tc2(h, wide)
    torch.cuda.synchronize()
    side, got_few, got_many = torch.cuda.Stream(), [], []
    for _ in range(10):
        with torch.cuda.stream(side):
            got_few += [ops_q4.gemm_q4(x, w) for _ in range(4)]
        got_many.append(ops_gemm.gemm_tc2(h, wide))
    torch.cuda.synchronize()
    assert all(torch.equal(y, few) for y in got_few) and all(torch.equal(y, many) for y in got_many)
