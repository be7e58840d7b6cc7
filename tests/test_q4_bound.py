"""Weights of 4 bits: which values the parts quantize as a model is bound (no GPU: the quantizer is a recorder)."""
import pytest
import torch

from tensorline_b200 import ops_q4
from tensorline_b200.parts import EMBEDDINGS, HEADS, PartSpec, Runtime


@pytest.fixture
def quantized(monkeypatch):
    """What `ops_q4.quantize` is given, in order."""
    seen = []
    monkeypatch.setattr(ops_q4, "quantize", lambda t, *form: seen.append(t.clone()) or ops_q4.pack(torch.zeros(t.shape, dtype=torch.int64), torch.ones(t.shape[0], -(-t.shape[1] // 128))))
    monkeypatch.setattr(ops_q4, "dequantize", lambda q: torch.zeros(q.shape))
    return seen


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("stored", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["weight", ""])
def test_a_tied_head_is_made_from_the_table_as_it_is_stored(quantized, act, stored, name):
    """Not from the embedding's copy, which the bfloat16 engine has rounded: both engines have the same codes and scales."""
    rt = Runtime(torch.device("cpu"), act, weight_bits=4, quantize_head=True)
    table = torch.randn(24, 16, generator=torch.Generator().manual_seed(1)).to(stored)
    embedding = EMBEDDINGS.build(PartSpec("token_table", {"tensor": name}), rt, vocab=24, dim=16)
    head = HEADS.build(PartSpec("linear", {}), rt, vocab=24, dim=16, tied=True)
    weights = {"embed" + (f".{name}" if name else ""): table}
    embedding.bind(weights, "embed")
    head.bind(weights, "head", embedding)
    assert len(quantized) == 1 and quantized[0].dtype == stored and torch.equal(quantized[0], table)
    assert embedding.weight.dtype == (torch.bfloat16 if act == torch.bfloat16 else stored)      # the table itself stays as it is


@pytest.mark.parametrize("stored", [torch.float16, torch.float64])
def test_matrices_of_other_types_by_way_of_float32(quantized, stored):
    from tensorline_b200.parts import FEED_FORWARDS
    rt = Runtime(torch.device("cpu"), torch.bfloat16, weight_bits=4)
    part = FEED_FORWARDS.build(PartSpec("plain_mlp", dict(hidden=16, intermediate=24)), rt)
    g = torch.Generator().manual_seed(2)
    weights = {n: torch.randn(s.shape, generator=g).to(stored) for n, s in part.expected_tensors("l").items()}
    part.bind(weights, "l")
    for seen, name in zip(quantized, ("l.up_proj.weight", "l.down_proj.weight"), strict=True):
        assert seen.dtype == torch.float32 and torch.equal(seen, weights[name].float())
