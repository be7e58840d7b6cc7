"""Weights of 4 bits as models are bound with them."""
import pytest
import torch

from tests.plain.q4_plain import quantized
from tests.plain.qwen2_plain import read_safetensors
from tests.test_engine_gpu import engine
from tests.tiny import write_tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", [torch.bfloat16, torch.float32])
def test_a_tied_head_holds_the_same_values_in_both_engines(tmp_path, store):
    from tensorline_b200 import ops_q4
    folder = write_tiny("A", tmp_path / "m", store_dtype=store)
    table = next(t for n, t in read_safetensors(folder / "model.safetensors").items() if "embed" in n)
    codes, scales, zeros = quantized(table.to(store), 32, True, torch.bfloat16)
    spread = lambda t: t.repeat_interleave(32, dim=1)[:, :table.shape[1]]                # noqa: E731
    want = (spread(scales.double()) * (codes - spread(zeros)).double()).float()
    for dtype in ("bfloat16", "float32"):
        head = engine(folder, dtype, weight_bits=4, weight_group=32, weight_zeros=True, quantize_head=True).model.head.weight
        values = ops_q4.dequantize(head) if isinstance(head, ops_q4.Q4Weight) else head
        assert values.dtype == torch.float32 and torch.equal(values.cpu(), want), dtype


@pytest.mark.parametrize("stored", [torch.float16, torch.float64])
def test_matrices_of_other_types(stored):
    """As a folder's loader has it for what no kernel reads: by way of float32."""
    from tensorline_b200 import ops_q4
    from tensorline_b200.parts import FEED_FORWARDS, PartSpec, Runtime
    g = torch.Generator().manual_seed(3)
    part = FEED_FORWARDS.build(PartSpec("gated_mlp", dict(hidden=64, intermediate=128)), Runtime(torch.device("cuda", 0), torch.bfloat16, weight_bits=4))
    weights = {n: torch.randn(s.shape, generator=g).to(stored).cuda() for n, s in part.expected_tensors("l").items()}
    part.bind(weights, "l")
    codes, scales, _ = quantized(weights["l.down_proj.weight"].float(), 128, False, torch.bfloat16)
    want = (scales.double().repeat_interleave(128, dim=1)[:, :128] * (codes - 8).double()).float()
    assert torch.equal(ops_q4.dequantize(part.w_down).cpu(), want)


@pytest.mark.parametrize("kind", ["gated_mlp", "plain_mlp"])
@pytest.mark.parametrize("cut", ["rows of a wider matrix", "rows between two 16-byte boundaries", "every other value", "one row for all"])
def test_a_feed_forward_of_rows_that_lie_apart(kind, cut):
    """As weights of 16 bits take them."""
    from tensorline_b200.parts import FEED_FORWARDS, PartSpec, Runtime
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(5, 140, generator=g).to(torch.bfloat16).cuda()
    h = {"rows of a wider matrix": lambda: wide[:, :64], "rows between two 16-byte boundaries": lambda: wide[:, 4:68], "every other value": lambda: wide[:, :128:2],
         "one row for all": lambda: wide[0, :64].expand(5, 64)}[cut]()
    assert h.shape == (5, 64) and not h.is_contiguous()
    activation = "silu" if kind == "gated_mlp" else "gelu_tanh"
    for bits in (None, 4):
        part = FEED_FORWARDS.build(PartSpec(kind, dict(hidden=64, intermediate=128, activation=activation)), Runtime(torch.device("cuda", 0), torch.bfloat16, weight_bits=bits))
        part.bind({n: torch.randn(s.shape, generator=g).to(torch.bfloat16).cuda() for n, s in part.expected_tensors("l").items()}, "l")
        got = part.forward(h, None)
        if bits == 4:                                    # (a library's product may add up in another order for them)
            assert torch.equal(got, part.forward(h.contiguous(), None))
