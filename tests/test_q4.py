"""Weights of 4 bits without a GPU: the stored form, and what is refused."""
import pytest
import torch

from tensorline_b200 import ops_q4
from tensorline_b200.ops import KernelError
from tests.plain.q4_plain import unpack, values


@pytest.mark.parametrize("n,k", [(1, 8), (128, 128), (131, 264), (300, 136)])
@pytest.mark.parametrize("group", ops_q4.GROUPS)
@pytest.mark.parametrize("zeros,scale", [(False, torch.bfloat16), (True, torch.float32)])
def test_packed_weights_are_what_was_packed(n, k, group, zeros, scale):
    g = torch.Generator().manual_seed(n + k)
    per_row = (n, -(-k // group))
    codes, scales = torch.randint(0, 16, (n, k), generator=g), torch.rand(per_row, generator=g).to(scale)
    zs = torch.randint(0, 16, per_row, generator=g) if zeros else None
    w = ops_q4.pack(codes, scales, zs, group)
    assert w.shape == (n, k) and w.nbytes == -(-n // 128) * -(-k // 128) * ops_q4.block_bytes(group, scale, zeros)
    got, got_scales, got_zeros = unpack(w)
    assert torch.equal(got, codes) and torch.equal(got_scales, scales)
    assert got_zeros is None if zs is None else torch.equal(got_zeros, zs)
    first = float(scales[0, 0]) * (int(codes[0, 0]) - (int(zs[0, 0]) if zeros else 8))
    assert float(values(w)[0, 0]) == pytest.approx(first, abs=0)


def test_refused_forms():
    codes, scales = torch.zeros(4, 64, dtype=torch.int64), torch.ones(4, 1)
    for bad in (lambda: ops_q4.pack(codes, scales, group=16), lambda: ops_q4.pack(codes, scales.half()), lambda: ops_q4.pack(codes, scales[:3]),
                lambda: ops_q4.pack(codes + 16, scales), lambda: ops_q4.pack(codes - 1, scales), lambda: ops_q4.pack(codes.float(), scales),
                lambda: ops_q4.pack(codes[:, :60], scales), lambda: ops_q4.pack(codes, scales, torch.full((4, 1), 16)),
                lambda: ops_q4.pack(codes, scales, torch.zeros(4, 1)), lambda: ops_q4.pack(codes[:0], scales[:0]),
                lambda: ops_q4.pack(codes, scales, torch.zeros(4, 2, dtype=torch.int64))):
        with pytest.raises(KernelError):
            bad()
    data = ops_q4.pack(codes, scales).data
    for args, more in (((data, 4, 60), {}), ((data, 0, 64), {}), ((data, 4, 64), {}), ((data, 129, 64), dict(scale_dtype=torch.float32)),
                       ((data, 4, 64), dict(scale_dtype=torch.float16)), ((data, 4, 64), dict(group=48)), ((data.int(), 4, 64), dict(scale_dtype=torch.float32)),
                       ((data, 4, 64), dict(scale_dtype=torch.float32, zeros=True)), ((data.transpose(0, 2), 4, 64), {})):
        with pytest.raises(KernelError):
            ops_q4.Q4Weight(*args, **more)
    assert ops_q4.Q4Weight(data, 4, 64, scale_dtype=torch.float32).shape == (4, 64)


def test_no_path_on_the_host():
    w = ops_q4.pack(torch.zeros(4, 64, dtype=torch.int64), torch.ones(4, 1))
    assert not w.settle().data.is_cuda and w.at_rest
    for call in (lambda: ops_q4.gemm_q4(torch.zeros(2, 64, dtype=torch.bfloat16), w), lambda: ops_q4.quantize(torch.zeros(4, 64)),
                 lambda: ops_q4.dequantize(w)):
        with pytest.raises(KernelError, match="no CPU path"):
            call()


@pytest.mark.parametrize("x,more", [
    (torch.zeros(2, 64), {}), (torch.zeros(2, 72, dtype=torch.bfloat16), {}), (torch.zeros(64, dtype=torch.bfloat16), {}),
    (torch.zeros(2, 64, dtype=torch.bfloat16), dict(out_dtype=torch.float16)), (torch.zeros(2, 64, dtype=torch.bfloat16), dict(gated="relu")),
    (torch.zeros(2, 64, dtype=torch.bfloat16), dict(gated=("swish_clamped", 0.0, 1.0))), (torch.zeros(2, 64, dtype=torch.bfloat16), dict(gated="silu")),
    (torch.zeros(2, 64, dtype=torch.bfloat16), dict(gated=["silu"])), (torch.zeros(2, 64, dtype=torch.bfloat16), dict(gated=("swish_clamped", "7", 1.0)))])
def test_refused_products(x, more):
    w = ops_q4.pack(torch.zeros(4, 64, dtype=torch.int64), torch.ones(4, 1))
    with pytest.raises(KernelError):
        ops_q4.gemm_q4(x, w, **more)


def test_sizes_that_the_entries_have_no_room_for():
    w = ops_q4.pack(torch.zeros(4, 64, dtype=torch.int64), torch.ones(4, 1))
    with pytest.raises(KernelError, match="at most"):
        ops_q4.gemm_q4(torch.empty(2 ** 32 + 1, 64, dtype=torch.bfloat16, device="meta"), w)
    with pytest.raises(KernelError, match="rows"):
        ops_q4.dequantize(ops_q4.Q4Weight(torch.empty(65536, 1, 8448, dtype=torch.uint8, device="meta"), 65536 * 128, 128))
    with pytest.raises(KernelError, match="sizes"):
        ops_q4.Q4Weight(torch.empty(2 ** 25, 1, 8448, dtype=torch.uint8, device="meta"), 2 ** 32, 128)


def test_matrices_that_share_memory():
    n = 10
    for a, a_step, a_bytes, b, b_step, b_bytes, rows in [(1000, 200, 64, 1000 + at, step, wide, n) for at in range(-2300, 2300, 20) for step in (80, 200, 320) for wide in (20, 80)]:
        bytes_of = lambda start, by, wide: {start + r * by + c for r in range(rows) for c in range(wide)}      # noqa: E731
        shared = bool(bytes_of(a, a_step, a_bytes) & bytes_of(b, b_step, b_bytes))
        said = ops_q4._meet(a, a_step, a_bytes, b, b_step, b_bytes, rows)
        assert said >= shared                            # never missed
        if a_step == b_step:
            assert said == shared
    assert not ops_q4._meet(0, 64, 64, 0, 64, 64, 0) and ops_q4._meet(0, 0, 64, 32, 0, 64, 1) and not ops_q4._meet(0, 0, 64, 64, 0, 64, 1)


def test_entries_are_declared_as_they_are_called():
    import ctypes
    import os
    import re
    from tests.test_entry_signatures import KINDS
    found = {}
    for source in ops_q4.SOURCES:
        with open(os.path.join(os.path.dirname(ops_q4.__file__), "csrc", source)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for name, arguments in re.findall(r"TL_EXPORT\s+int\s+(\w+)\s*\(([^)]*)\)\s*\{", text):
            kinds = [re.sub(r"\bconst\b", "", a.strip().rsplit(None, 1)[0] if "*" not in a else "*").strip() for a in arguments.split(",")]
            found[name] = [ctypes.c_void_p if kind == "*" else KINDS[kind] for kind in kinds]
    assert found == {name: list(sig) for name, sig in ops_q4._SIGNATURES.items()}


def test_bytes_of_a_block_are_those_of_the_library():
    lib = ops_q4.lib()
    for group in ops_q4.GROUPS:
        for scale in (torch.bfloat16, torch.float32):
            for zeros in (False, True):
                assert lib.tl_q4_block_bytes(group, int(scale is torch.float32), int(zeros)) == ops_q4.block_bytes(group, scale, zeros)
    assert lib.tl_q4_block_bytes(16, 0, 0) == 0


def test_c_entries_refuse_what_they_do_not_take():
    """No pointer is looked at before the sizes: these end on the host."""
    lib, p = ops_q4.lib(), 1 << 20
    good = dict(x=p, ldx=64, w=p, y=p, ldo=128, T=2, N=128, K=64, form=64, limit=0.0, alpha=1.0, status=p, stream=None)
    for bad in (dict(T=-1), dict(T=0x7fffff01), dict(N=0x7fffff01, ldo=1 << 31), dict(K=0x7fffff08, ldx=1 << 31), dict(N=0), dict(K=0), dict(K=60), dict(form=16), dict(form=64 | 1 << 14), dict(form=-1), dict(form=64 | 1 << 10, N=192),
                dict(ldo=100), dict(ldx=56), dict(ldx=68), dict(x=p + 2), dict(w=p + 8), dict(y=None), dict(status=None)):
        assert lib.tl_gemm_q4(*{**good, **bad}.values()) == 1, bad
    assert lib.tl_gemm_q4(*{**good, "T": 0}.values()) == 0
    for w, out, n, k, form in ((p, p, 0, 64, 64), (p, p, 4, 60, 64), (p, p, 4, 64, 16), (p + 8, p, 4, 64, 64), (p, p + 8, 4, 64, 64), (p, p, 4, 64, 64 | 1 << 10)):
        assert lib.tl_quantize_q4(w, 0, out, n, k, form, None) == 1
        assert lib.tl_dequantize_q4(w, out, 0, n, k, form, None) == 1


def test_options_of_the_command_and_the_engine():
    from tensorline_b200 import cli
    from tensorline_b200.config.engine import EngineConfig
    a = cli._generate_parser().parse_args(["--model", "m", "--weight-bits", "4", "--weight-group", "64", "--weight-zeros", "--quantize-head"])
    assert (a.weight_bits, a.weight_group, a.weight_zeros, a.quantize_head) == (4, 64, True, True)
    a = cli._generate_parser().parse_args(["--model", "m"])
    assert (a.weight_bits, a.weight_group, a.weight_zeros, a.quantize_head) == (None, 128, False, False)
    EngineConfig(weight_bits=4, weight_group=32, weight_zeros=True, quantize_head=True).validate()
    for bad in (dict(weight_bits=8), dict(weight_bits=4, weight_group=48), dict(weight_zeros=True), dict(quantize_head=True)):
        with pytest.raises(ValueError):
            EngineConfig(**bad).validate()
