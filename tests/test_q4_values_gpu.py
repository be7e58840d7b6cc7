"""Decoders with weights of 4 bits beside the same decoders with the values that those weights stand for, quantized by the plain code and stored in 32 bits.

The 32-bit engine reads the values exactly, so its logits are the same bits either way.  The bfloat16 engine is held against them by the rule that the decoders
without experts have for weights of 16 bits, every position within 0.05 of the largest logit, and by that of the others, four positions in five."""
import importlib
import json

import pytest
import torch

from tests.plain.q4_plain import quantized
from tests.plain.qwen2_plain import PlainQwen2, read_safetensors
from tests.test_engine_gpu import NEW_TOKENS, PAGE_SIZE, PROMPT_LENGTHS, engine, follows_where_decided, params
from tests.test_q4_engine_gpu import folder_of_values
from tests.tiny import CONFIGS, random_tokens, write_tiny

pytestmark = pytest.mark.gpu

ALL = [(decoder, name) for decoder, names in (("vutesun", ("V1", "V2", "V3", "V4")), ("dekerax", ("D1", "D2", "D3", "D4", "D5")), ("sumuvik", ("S1", "S2", "S3", "S4", "S5", "S6")),
                                              ("tenalorn", ("N1", "N2", "N3", "N4", "N5", "N6")), ("zosurax", ("Z1", "Z2", "Z3", "Z4", "Z5", "Z6")),
                                              ("fimolix", ("F1", "F2", "F3", "F4", "F5", "F6"))) for name in names]
OPTIONS = dict(num_blocks=64, max_num_seqs=4, max_model_len=128)


def written(decoder, name, out):
    tiny = importlib.import_module(f"tests.tiny_{decoder}")
    folder = getattr(tiny, f"write_tiny_{decoder}")(name, out)
    return folder, tiny.PAGE_SIZE[name], next(v for k, v in json.loads((folder / "config.json").read_text()).items() if "vocab" in k)


def logits(eng, vocab):
    """Two requests: prompts, then four single tokens each."""
    from tensorline_b200.engine.runner import StepEntry
    prompts = {"a": random_tokens(vocab, 25, seed=1), "b": random_tokens(vocab, 10, seed=2)}
    first = {"a": 21, "b": 6}
    for rid, n in first.items():
        eng.cache.admit(rid)
        eng.cache.grow(rid, 0, n + 4)
        eng.runner.start_request(rid, 0)
    got = [eng.runner.step([StepEntry(r, prompts[r][:n], list(range(n))) for r, n in first.items()])]
    for i in range(4):
        got.append(eng.runner.step([StepEntry(r, prompts[r][n + i:n + i + 1], [0]) for r, n in first.items()]))
    return torch.cat([g.double().cpu() for g in got])


def of_values(folder, out, given, group, zeros):
    """The folder with every tensor whose rows the engine gave to its quantizer (`given`: matrices) replaced by the values of the plain quantization."""
    from tensorline_b200.weights.safetensors_io import write_safetensors
    rows = {}
    for m in given:
        rows.setdefault(m.shape[1], set()).update(r.tobytes() for r in m.float().cpu().numpy())
    tensors, names = read_safetensors(folder / "model.safetensors"), []
    for name, t in tensors.items():
        if t.dim() == 2 and "embed" not in name and all(r.tobytes() in rows.get(t.shape[1], ()) for r in t.float().numpy()):
            codes, scales, zs = quantized(t, group, zeros, torch.bfloat16)
            spread = lambda x: x.repeat_interleave(group, dim=1)[:, :t.shape[1]]          # noqa: E731
            tensors[name] = (spread(scales.double()) * (codes - (spread(zs) if zeros else 8)).double()).float()
            names.append(name)
    out.mkdir()
    (out / "config.json").write_text((folder / "config.json").read_text())
    write_safetensors(out / "model.safetensors", tensors)
    return out, names


@pytest.mark.parametrize("decoder,name", ALL)
def test_the_logits_of_the_values(tmp_path, monkeypatch, decoder, name):
    from tensorline_b200 import Engine, ops_q4
    folder, page, vocab = written(decoder, name, tmp_path / "m")
    given, quantize = [], ops_q4.quantize
    monkeypatch.setattr(ops_q4, "quantize", lambda t, *form: given.append(t.clone()) or quantize(t, *form))
    own_head = "head" in read_safetensors(folder / "model.safetensors")                  # (a folder cannot hold a tied head's values beside the table's)
    bits = dict(weight_bits=4, weight_group=32, weight_zeros=True, quantize_head=own_head, block_size=page, **OPTIONS)
    exact = logits(Engine(str(folder), dtype="float32", **bits), vocab)
    values, names = of_values(folder, tmp_path / "v", given, 32, True)
    assert bool(given) == bool(names) and (not given or ("head" in names) == own_head)    # widths that are no multiple of 8 stay as they are
    want = logits(Engine(str(values), dtype="float32", block_size=page, **OPTIONS), vocab)
    assert torch.equal(exact, want)
    err = (logits(Engine(str(folder), dtype="bfloat16", **bits), vocab) - want).abs().amax(1) / want.abs().max()
    if decoder in ("zosurax", "fimolix"):
        assert float(err.max()) <= 0.05, err.tolist()
    else:                                                # a position's experts may change with a rounding
        assert float(err.max()) <= 1.0 and int((err > 0.05).sum()) <= 0.2 * len(err), err.tolist()


@pytest.mark.parametrize("name,group,zeros,head", [("A", 64, True, False), ("B_FULL", 32, False, True), ("B", 32, True, True), ("C", 128, False, False)])
def test_the_dense_decoder_where_the_plain_model_is_decided(tmp_path, name, group, zeros, head):
    """As many decided positions as for weights of 16 bits, windows and longer outputs among them."""
    folder = write_tiny(name, tmp_path / "m")
    plain = PlainQwen2(folder_of_values(folder, tmp_path / "q", group, zeros, head))
    prompts, n_new = [random_tokens(CONFIGS[name]["vocab_size"], n, seed=30 + n) for n in PROMPT_LENGTHS[name]], NEW_TOKENS[name]
    eng = engine(folder, "bfloat16", weight_bits=4, weight_group=group, weight_zeros=zeros, quantize_head=head, block_size=PAGE_SIZE[name], num_blocks=64, max_model_len=160)
    outs = eng.generate(prompts, params(n_new))
    assert sum(follows_where_decided(plain, p, o.token_ids) for p, o in zip(prompts, outs)) >= n_new // 2
