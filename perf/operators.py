"""What the products with 4-bit weights are measured by, beside their plain forms.

    linear      y = x W^T for W held as 4-bit codes with a scale (and a zero point) per row and group of k
    gated       act(x Wg^T) * (x Wu^T), both matrices in 4 bits, gate and up rows alternating in blocks of 64
    quantize    a matrix into that form and back to the values it stands for

A weight is w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group]), codes and zeros 0..15, zero = 8 where none is stored.
It is held as uint8 [ceil(N / 128), ceil(K / 128), bytes]: the block of 128 rows and 128 k that a thread block reads at a time, in it the codes,
the scales [group][row] and the zeros [group][row].  Codes lie as [k / 32][row][k / 8 % 4] words of 32 bits; k % 8 = 4 p + 2 q + h
is at bit 16 h + 8 p + 4 q of its word.  Sizes are those of the published Qwen2.5 layers and of the engine's default steps (1 to 64
requests that decode, prompts of up to 2,048 tokens).
"""
from __future__ import annotations

import math
import zlib

import torch

own = False

SEVEN_B = dict(hidden=3584, inter=18944, qkv=4608, vocab=152064)
FOURTEEN_B = dict(hidden=5120, inter=13824, qkv=7168)


def listed():
    return [
        # one request decodes: its query, key and value rows, the smallest call
        dict(name="qkv_token_1", kind="linear", tokens=1, n=SEVEN_B["qkv"], k=SEVEN_B["hidden"], group=128, zeros=False, scale="bfloat16", out="bfloat16"),
        # eight requests decode: the down projection, a long sum over few rows of weights
        dict(name="down_tokens_8", kind="linear", tokens=8, n=SEVEN_B["hidden"], k=SEVEN_B["inter"], group=128, zeros=False, scale="bfloat16", out="bfloat16"),
        # the output head of eight requests, 32-bit logits, the most weights of a call
        dict(name="head_tokens_8", kind="linear", tokens=8, n=SEVEN_B["vocab"], k=SEVEN_B["hidden"], group=128, zeros=True, scale="bfloat16", out="float32"),
        # an odd number of requests, small groups with zero points and 32-bit scales
        dict(name="down_tokens_45", kind="linear", tokens=45, n=FOURTEEN_B["hidden"], k=FOURTEEN_B["inter"], group=64, zeros=True, scale="float32", out="bfloat16"),
        # a prompt's odd tail beside decoding requests
        dict(name="qkv_prompt_333", kind="linear", tokens=333, n=FOURTEEN_B["qkv"], k=FOURTEEN_B["hidden"], group=128, zeros=False, scale="bfloat16", out="bfloat16"),
        # a whole prompt through the down projection
        dict(name="down_prompt_2048", kind="linear", tokens=2048, n=SEVEN_B["hidden"], k=SEVEN_B["inter"], group=128, zeros=False, scale="bfloat16", out="bfloat16"),
        # the feed-forward's first half for one, eight and 64 requests, and for a whole prompt
        dict(name="gated_token_1", kind="gated", tokens=1, n=2 * SEVEN_B["inter"], k=SEVEN_B["hidden"], group=128, zeros=False, scale="bfloat16", act="silu"),
        dict(name="gated_tokens_8", kind="gated", tokens=8, n=2 * SEVEN_B["inter"], k=SEVEN_B["hidden"], group=128, zeros=False, scale="bfloat16", act="silu"),
        dict(name="gated_tokens_64", kind="gated", tokens=64, n=2 * FOURTEEN_B["inter"], k=FOURTEEN_B["hidden"], group=128, zeros=True, scale="bfloat16", act="gelu_tanh"),
        dict(name="gated_prompt_2048", kind="gated", tokens=2048, n=2 * SEVEN_B["inter"], k=SEVEN_B["hidden"], group=128, zeros=False, scale="bfloat16", act="silu"),
        # loading: the largest matrix of a layer as it is stored, and a small odd one
        dict(name="quantize_gate_up", kind="quantize", n=2 * SEVEN_B["inter"], k=SEVEN_B["hidden"], group=128, zeros=False, scale="bfloat16", of="bfloat16", out="bfloat16"),
        dict(name="quantize_odd", kind="quantize", n=1003, k=1096, group=32, zeros=True, scale="float32", of="float32", out="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gated", "gated", "quantize"])
    case = dict(kind=kind, group=rng.choice([32, 64, 128, 128]), zeros=rng.random() < 0.4, scale=rng.choice(["bfloat16", "bfloat16", "float32"]))
    case["k"] = 8 * _log(rng, 256 // 8, SEVEN_B["inter"] // 8)
    most = 2 * SEVEN_B["inter"] * SEVEN_B["hidden"]                                     # weights of a matrix
    if kind == "quantize":
        case.update(n=_log(rng, 65, min(40000, most // case["k"])), of=rng.choice(["bfloat16", "float32"]), out=rng.choice(["bfloat16", "float32"]))
        return case
    case["tokens"] = _log(rng, 1, 2048)
    n = _log(rng, 128, min(40000, most // case["k"]))
    if kind == "gated":
        case.update(n=128 * max(1, n // 128), act=rng.choice(["silu", "gelu_tanh", "swish_clamped"]))
    else:
        case.update(n=n, out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    return case


def _type(name):
    return {"bfloat16": torch.bfloat16, "float32": torch.float32}[name]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(zlib.crc32(repr((seed, sorted(case.items()))).encode()))
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")               # noqa: E731
    n, k, group, zeros = case["n"], case["k"], case["group"], case["zeros"]
    if case["kind"] == "quantize":                       # rows of unequal size, some groups of zeros
        w = rand(n, k).mul_(0.02).mul_(rand(n, 1).mul_(0.5).exp_())
        w[::97, :group] = 0.0
        return dict(case, w=w.to(_type(case["of"])))
    tiles, blocks, groups = -(-n // 128), -(-k // 128), 128 // group
    # codes as weights of a normal distribution have them, scaled to their group's largest; a zero point moves a group's middle
    zero = (rand(tiles, blocks, groups, 128) * 0.8 + 7.5).round_().clamp_(0, 15).to(torch.uint8) if zeros else None
    codes = torch.empty((tiles, blocks, 4, 128, 16), dtype=torch.uint8, device="cuda")
    for t in range(0, tiles, 256):                       # in pieces: a vocabulary's worth of floats is large
        part = codes[t:t + 256]
        c = (rand(part.shape[0], blocks, 4, 128, 16, 2) * 2.6)
        if zeros:                                        # [tile, block, group, row] -> the 32-k piece's group
            z = zero[t:t + 256].repeat_interleave(4 // groups, dim=2) if groups < 4 else zero[t:t + 256]
            c += z[..., None, None]
        else:
            c += 8.0
        c = c.round_().clamp_(0, 15).to(torch.uint8)
        part.copy_(c[..., 0] | (c[..., 1] << 4))
    scale = (torch.rand((tiles, blocks, groups, 128), generator=g, device="cuda") * 0.008 + 0.004).to(_type(case["scale"]))
    pieces = [codes.reshape(tiles, blocks, -1), scale.reshape(tiles, blocks, -1).view(torch.uint8)]
    if zeros:
        pieces.append(zero.reshape(tiles, blocks, -1))
    x = rand(case["tokens"], k)
    if case["kind"] == "linear" and k > 8192:            # a feed-forward's inner values: products, most of them small
        x = x * rand(case["tokens"], k).mul_(0.5)
    return dict(case, data=torch.cat(pieces, dim=2), x=x.to(torch.bfloat16))


def _weights(state, dtype):
    """The matrix that `data` stands for, [N, K]."""
    n, k, group, zeros, data = state["n"], state["k"], state["group"], state["zeros"], state["data"]
    tiles, blocks, groups = data.shape[0], data.shape[1], 128 // group
    b = data[:, :, :8192].reshape(tiles, blocks, 4, 128, 4, 2, 2)                        # [.., k / 32, row, word, h, p]
    c = torch.stack((b & 15, b >> 4), dim=-1).permute(0, 3, 1, 2, 4, 6, 7, 5)            # [tile, row, block, k / 32, word, p, q, h]
    c = c.reshape(tiles * 128, blocks * groups, group).to(dtype)
    at = 8192 + groups * 128 * _type(state["scale"]).itemsize
    s = data[:, :, 8192:at].contiguous().view(_type(state["scale"])).reshape(tiles, blocks, groups, 128)
    s = s.permute(0, 3, 1, 2).reshape(tiles * 128, blocks * groups, 1).to(dtype)
    if zeros:
        z = data[:, :, at:].reshape(tiles, blocks, groups, 128).permute(0, 3, 1, 2).reshape(tiles * 128, blocks * groups, 1).to(dtype)
    else:
        z = 8.0
    return ((c - z) * s).reshape(tiles * 128, blocks * 128)[:n, :k]


LIMIT, ALPHA = 7.0, 1.702                                # the clamped swish's constants


def _gate(g, u, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    if act == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))) * u
    g, u = g.clamp_max(LIMIT), u.clamp(-LIMIT, LIMIT)
    return g / (1.0 + torch.exp(-ALPHA * g)) * (u + 1.0)


def _halves(w):
    """Gate and up rows of a matrix in which they alternate in blocks of 64."""
    b = w.reshape(w.shape[0] // 128, 2, 64, w.shape[1])
    return b[:, 0].reshape(-1, w.shape[1]), b[:, 1].reshape(-1, w.shape[1])


def _rounded(w, group, zeros, scale_type):
    """The values that quantized weights stand for, in 64 bits: what is next to a border is decided there."""
    n, k = w.shape
    full = -(-k // group) * group
    v = torch.zeros((n, full), dtype=torch.float64, device=w.device)
    v[:, :k] = w
    v = v.reshape(n, full // group, group)
    if zeros:
        lo, hi = v.amin(dim=2, keepdim=True).clamp_max(0.0), v.amax(dim=2, keepdim=True).clamp_min(0.0)
        s = ((hi - lo) / 15.0).float().to(scale_type).double()
        d = torch.where(s > 0, s, torch.ones_like(s))
        z = (-lo / d).round().clamp(0, 15)
        c = ((v / d).round() + z).clamp(0, 15) - z
    else:
        s = (v.abs().amax(dim=2, keepdim=True) / 7.0).float().to(scale_type).double()
        d = torch.where(s > 0, s, torch.ones_like(s))
        c = (v / d).round().clamp(-7, 7)
    return (c * s).reshape(n, full)[:, :k]


def run(state):
    if own:
        from tensorline_b200 import ops_q4
        scale = _type(state["scale"])
        if state["kind"] == "quantize":
            return ops_q4.dequantize(ops_q4.quantize(state["w"], group=state["group"], zeros=state["zeros"], scale_dtype=scale), _type(state["out"]))
        w = ops_q4.Q4Weight(state["data"], state["n"], state["k"], group=state["group"], zeros=state["zeros"], scale_dtype=scale,
                            at_rest=True)                # a model's weights were there long before the call
        if state["kind"] == "linear":
            return ops_q4.gemm_q4(state["x"], w, _type(state["out"]))
        return ops_q4.gemm_q4(state["x"], w, gated=("swish_clamped", LIMIT, ALPHA) if state["act"] == "swish_clamped" else state["act"])
    if state["kind"] == "quantize":
        return _rounded(state["w"], state["group"], state["zeros"], _type(state["scale"])).to(_type(state["out"]))
    x, w = state["x"].float(), _weights(state, torch.float32)
    if state["kind"] == "linear":
        return (x @ w.t()).to(_type(state["out"]))
    gate, up = _halves(w)
    return _gate(x @ gate.t(), x @ up.t(), state["act"]).to(torch.bfloat16)


def work(case):
    n, k = case["n"], case["k"]
    groups = -(-k // case["group"])
    held = n * k / 2 + n * groups * (_type(case["scale"]).itemsize + (0.5 if case["zeros"] else 0.0))
    if case["kind"] == "quantize":                       # read once, written packed, read packed, written as values
        return dict(bytes=n * k * (_type(case["of"]).itemsize + _type(case["out"]).itemsize) + 2 * held, flops=0)
    t = case["tokens"]
    y = t * n * _type(case["out"]).itemsize if case["kind"] == "linear" else t * (n // 2) * 2
    return dict(bytes=held + t * k * 2 + y, flops=2 * t * n * k)


def exact(case, seed):
    s = prepare(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    if case["kind"] == "quantize":
        w = s["w"].double()
        out = torch.empty_like(w)
        for at in range(0, k, group):                    # group by group
            v = w[:, at:at + group]
            if case["zeros"]:
                low, high = torch.minimum(v.min(1).values, torch.zeros(())), torch.maximum(v.max(1).values, torch.zeros(()))
                sc = ((high - low) / 15).to(torch.float32).to(_type(case["scale"])).double()
                safe = sc.masked_fill(sc == 0, 1.0)
                zp = torch.round(-low / safe).clamp(0, 15)
                q = torch.round(v / safe[:, None]) + zp[:, None]
                out[:, at:at + group] = sc[:, None] * (q.clamp(0, 15) - zp[:, None])
            else:
                sc = (torch.maximum(v.max(1).values, -v.min(1).values) / 7).to(torch.float32).to(_type(case["scale"])).double()
                q = torch.round(v / sc.masked_fill(sc == 0, 1.0)[:, None])
                out[:, at:at + group] = sc[:, None] * q.clamp(-7, 7)
        return out
    x, data, groups = s["x"].double(), s["data"], 128 // group
    sums = torch.empty((x.shape[0], n), dtype=torch.float64, device="cuda")
    words = data[:, :, :8192].contiguous().view(torch.int32).reshape(data.shape[0], data.shape[1], 4, 128, 4)
    ends = 8192 + groups * 128 * _type(case["scale"]).itemsize
    scales = data[:, :, 8192:ends].contiguous().view(_type(case["scale"])).reshape(data.shape[0], data.shape[1], groups, 128)
    zero = data[:, :, ends:].reshape(data.shape[0], data.shape[1], groups, 128) if case["zeros"] else None
    for t in range(0, data.shape[0], 32):                # 32 tiles of rows at a time, k by its place in a word
        w = torch.empty((words[t:t + 32].shape[0], 128, data.shape[1], 16, 8), dtype=torch.float64, device="cuda")
        for j in range(8):
            code = (words[t:t + 32] >> (16 * (j & 1) + 8 * (j >> 2) + 4 * (j >> 1 & 1))) & 15
            w[..., j] = code.permute(0, 3, 1, 2, 4).reshape(w.shape[:4])
        w = w.reshape(w.shape[0], 128, data.shape[1], groups, group)
        w -= zero[t:t + 32].permute(0, 3, 1, 2)[..., None].double() if zero is not None else 8.0
        w *= scales[t:t + 32].permute(0, 3, 1, 2)[..., None].double()
        rows = w.reshape(-1, data.shape[1] * 128)[:, :k]
        rows = rows[:max(0, n - t * 128)]
        sums[:, t * 128:t * 128 + rows.shape[0]] = x @ rows.t()
    if case["kind"] == "linear":
        return sums
    pair = sums.reshape(x.shape[0], n // 128, 2, 64)
    a, b = pair[:, :, 0].reshape(x.shape[0], -1), pair[:, :, 1].reshape(x.shape[0], -1)
    if case["act"] == "silu":
        return a * torch.sigmoid(a) * b
    if case["act"] == "gelu_tanh":
        return a * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3)) * b
    a = torch.clamp(a, max=LIMIT)
    return a * torch.sigmoid(ALPHA * a) * (torch.clamp(b, min=-LIMIT, max=LIMIT) + 1.0)
