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
