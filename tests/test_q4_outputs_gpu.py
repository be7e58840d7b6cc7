"""Outputs in the weights' own memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,at", [(1, 0), (3, 64), (40, -128)])
def test_an_output_in_the_weights_is_refused(T, at):
    from tensorline_b200 import ops_q4
    from tensorline_b200.ops import KernelError
    room = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    codes, scales = torch.randint(0, 16, (128, 128), generator=torch.Generator().manual_seed(1)), torch.ones(128, 1)
    packed = ops_q4.pack(codes.cuda(), scales.to(torch.bfloat16).cuda()).data
    data = room[32768:32768 + packed.numel()].view(packed.shape).copy_(packed)
    w = ops_q4.Q4Weight(data, 128, 128)
    x = torch.randn(T, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    flat = room.view(torch.bfloat16)
    first = 32768 // 2 + (at if at >= 0 else packed.numel() // 2 - 1)
    with pytest.raises(KernelError, match="weights"):
        ops_q4.gemm_q4(x, w, out=flat[first:first + T * 128].view(T, 128))
    before, behind = flat[32768 // 2 - T * 128:32768 // 2].view(T, 128), flat[32768 // 2 + packed.numel() // 2:][:T * 128].view(T, 128)
    want = ops_q4.gemm_q4(x, w)
    for out in (before, behind):                         # right in front of them and behind them
        assert torch.equal(ops_q4.gemm_q4(x, w, out=out), want) and torch.equal(data, packed)
