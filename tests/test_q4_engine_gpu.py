"""The engine with weights of 4 bits: against the plain model with the values that the 4-bit weights stand for, and the bfloat16 engine
against the 32-bit one, which reads those values exactly, for every decoder."""
import importlib
import json

import pytest
import torch

from tests.plain.q4_plain import quantized
from tests.plain.qwen2_plain import PlainQwen2, greedy_generate, read_safetensors
from tests.test_engine_gpu import engine, follows_where_decided, params
from tests.tiny import CONFIGS, random_tokens, write_tiny

pytestmark = pytest.mark.gpu


def folder_of_values(folder, out, group, zeros, head):
    """The model folder with its layers' matrices replaced by what their 4-bit weights stand for, in 32 bits."""
    from tensorline_b200.weights.safetensors_io import write_safetensors
    tensors = read_safetensors(folder / "model.safetensors")
    for name, t in tensors.items():
        if name.endswith("_proj.weight") or (head and name == "lm_head.weight"):
            codes, scales, zs = quantized(t.to(torch.bfloat16), group, zeros, torch.bfloat16)
            spread = lambda x: x.repeat_interleave(group, dim=1)[:, :t.shape[1]]          # noqa: E731
            tensors[name] = (spread(scales.double()) * (codes - (spread(zs) if zeros else 8)).double()).float()
    out.mkdir()
    (out / "config.json").write_text((folder / "config.json").read_text())
    write_safetensors(out / "model.safetensors", tensors)
    return out


@pytest.mark.parametrize("name,group,zeros,head", [("A", 32, False, False), ("B_FULL", 128, True, True), ("C", 64, False, True)])
def test_the_dense_decoder_is_the_plain_model_of_the_values(tmp_path, name, group, zeros, head):
    from tensorline_b200 import ops
    folder = write_tiny(name, tmp_path / "m")
    plain = PlainQwen2(folder_of_values(folder, tmp_path / "q", group, zeros, head))
    prompts = [random_tokens(CONFIGS[name]["vocab_size"], n, seed=30 + n) for n in (1, 5, 17, 32)]
    options = dict(weight_bits=4, weight_group=group, weight_zeros=zeros, quantize_head=head)
    exact = engine(folder, "float32", **options).generate(prompts, params())
    assert [o.token_ids for o in exact] == [greedy_generate(plain, p, 8) for p in prompts]
    before = ops.kernel_counts.copy()
    eng = engine(folder, "bfloat16", **options)
    outs = eng.generate(prompts, params())
    used = ops.kernel_counts - before
    assert sum(follows_where_decided(plain, p, o.token_ids) for p, o in zip(prompts, outs)) >= 1
    assert used["gemm_q4"] and used["quantize_q4"] and bool(used["gemm_q4+gated"]) == (CONFIGS[name]["intermediate_size"] % 64 == 0)
    assert eng.stats()["graph_replays"] > 0
    eager = engine(folder, "bfloat16", cuda_graphs=False, **options).generate(prompts, params())
    assert [o.token_ids for o in eager] == [o.token_ids for o in outs]


DECODERS = [("vutesun", "V1"), ("vutesun", "V4"), ("dekerax", "D1"), ("dekerax", "D4"), ("sumuvik", "S1"), ("sumuvik", "S4"), ("tenalorn", "N1"), ("tenalorn", "N4"),
            ("zosurax", "Z1"), ("zosurax", "Z4"), ("fimolix", "F1"), ("fimolix", "F4")]


@pytest.mark.parametrize("decoder,name", DECODERS)
def test_every_decoder_in_both_engines(tmp_path, decoder, name):
    """Prompts, then single tokens: of the positions four in five within 0.05 of the largest logit, all within the largest (as the decoders' own tests
    have it for weights of 16 bits)."""
    from tensorline_b200 import Engine
    from tensorline_b200.engine.runner import StepEntry
    tiny = importlib.import_module(f"tests.tiny_{decoder}")
    folder = getattr(tiny, f"write_tiny_{decoder}")(name, tmp_path / "m")
    vocab = json.loads((folder / "config.json").read_text()).get("vocab_size") or next(
        v for k, v in json.loads((folder / "config.json").read_text()).items() if "vocab" in k)
    logits = []
    for dtype in ("float32", "bfloat16"):
        eng = Engine(str(folder), dtype=dtype, block_size=tiny.PAGE_SIZE[name], num_blocks=64, max_num_seqs=4, max_model_len=128, weight_bits=4, weight_group=32,
                     weight_zeros=True)
        got = []
        for rid, n in (("a", 21), ("b", 6)):
            eng.cache.admit(rid)
            eng.cache.grow(rid, 0, n + 4)
            eng.runner.start_request(rid, 0)
        prompts = {"a": random_tokens(vocab, 25, seed=1), "b": random_tokens(vocab, 10, seed=2)}
        got.append(eng.runner.step([StepEntry("a", prompts["a"][:21], list(range(21))), StepEntry("b", prompts["b"][:6], list(range(6)))]).double().cpu())
        for i in range(4):
            got.append(eng.runner.step([StepEntry("a", prompts["a"][21 + i:22 + i], [0]), StepEntry("b", prompts["b"][6 + i:7 + i], [0])]).double().cpu())
        logits.append(torch.cat(got))
    assert bool(torch.isfinite(logits[1]).all())
    top = float(logits[0].abs().max())
    err = (logits[1] - logits[0]).abs().amax(1)
    assert float(err.max()) <= top and int((err > 0.05 * top).sum()) <= 0.2 * len(err), (decoder, name, (err / top).tolist())


def test_from_the_command_line(tmp_path, capsys):
    from tensorline_b200 import cli
    folder = write_tiny("B_FULL", tmp_path / "m")
    plain = PlainQwen2(folder_of_values(folder, tmp_path / "q", 64, True, False))
    assert cli.main(["--model", str(folder), "--dtype", "float32", "--prompt-ids", "5,9,200,17", "--max-tokens", "5", "--ignore-eos", "--block-size", "8",
                     "--num-blocks", "16", "--max-num-seqs", "4", "--max-model-len", "64", "--weight-bits", "4", "--weight-group", "64", "--weight-zeros"]) == 0
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    assert [line["token_ids"] for line in lines] == [greedy_generate(plain, [5, 9, 200, 17], 5)]


def test_a_layer_of_a_large_model(tmp_path):
    """Sizes at which every kernel of the products runs (one token, some, a prompt), through the parts: the gated feed-forward and a product whose
    input is a norm's recipe, against float64 from the values."""
    from tensorline_b200.parts import FEED_FORWARDS, PartSpec, Runtime
    from tests.plain.q4_plain import values
    rt = Runtime(torch.device("cuda", 0), torch.bfloat16, 16, weight_bits=4, weight_zeros=True)
    part = FEED_FORWARDS.build(PartSpec("gated_mlp", dict(hidden=1024, intermediate=2048, activation="silu")), rt)
    g = torch.Generator().manual_seed(1)
    weights = {n: (torch.randn(s.shape, generator=g) * s.shape[1] ** -0.5).to(torch.bfloat16).cuda() for n, s in part.expected_tensors("l").items()}
    part.bind(weights, "l")
    gu, down = values(part.w_gate_up).cuda(), values(part.w_down).cuda()
    for T in (1, 8, 16, 40, 100, 400):
        h = torch.randn(T, 1024, generator=g).to(torch.bfloat16).cuda()
        y = part.forward(h, None).double()
        a, u = [t.reshape(T, -1) for t in (h.double() @ gu.t()).view(T, 32, 2, 64).unbind(2)]
        m = a * torch.sigmoid(a) * u
        want = m @ down.t()
        # the inner values and the outputs are rounded to bfloat16, 2^-8 at most; the inner ones' errors add up at most as their norms do
        bound = (m.norm(dim=1, keepdim=True) * down.norm(dim=1)[None] + want.abs()) * 2.0 ** -8 * 1.01
        assert bool(((y - want).abs() <= bound).all()), T
