"""Weights of 4 bits: making them, and products with them (`csrc/gemm_q4.cu`, `csrc/gemm_q4_long.cu`, `csrc/gemv_q4.cu`, `csrc/quantize_q4.cu`).

    w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])

codes and zeros are whole numbers 0..15 (zero = 8 where a matrix has none), scales bfloat16 or float32, a group is 32, 64 or 128 values along k.
A matrix takes half a byte a value and its scales: 0.52 bytes in groups of 128 with bfloat16 scales and no zeros.

    w = quantize(matrix)                          # or pack(codes, scales, zeros), for weights that were quantized elsewhere
    y = gemm_q4(x, w)                             # x [T, K] bfloat16, y [T, N]
    m = gemm_q4(x, gate_up, gated="silu")         # silu(gate) * up, where gate and up rows alternate in blocks of 64
    matrix = dequantize(w)

Launches go to the current stream of the tensors' device.  As with every matrix of this package, K is a multiple of 8.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import ops
from .csrc.build import load_library
from .ops import KernelError, _check, _stream, device_status, num_sms

_P, _I, _F, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong

SOURCES = ["gemm_q4.cu", "gemm_q4_long.cu", "gemv_q4.cu", "quantize_q4.cu"]
_SIGNATURES = {
    "tl_q4_block_bytes": [_I, _I, _I],
    "tl_gemm_q4": [_P, _L, _P, _P, _L, _I, _I, _I, _I, _F, _F, _P, _P],
    "tl_gemm_q4_plan": [_I, _I, _I, _I, _P, _I],
    "tl_quantize_q4": [_P, _I, _P, _I, _I, _I, _P],
    "tl_dequantize_q4": [_P, _P, _I, _I, _I, _I, _P],
}
GROUPS = (32, 64, 128)
ROWS = K_BLOCK = 128                                      # of a stored block
CODE_BYTES = ROWS * K_BLOCK // 2
MOST = 0x7fffff00                                         # tokens, rows and columns
MOST_ROWS = 65535 * ROWS                                  # of a matrix that is quantized or read back
_lib = None


def lib():
    global _lib
    if _lib is None:
        l = load_library("tl_q4", SOURCES)
        for name, sig in _SIGNATURES.items():
            fn = getattr(l, name)
            fn.argtypes = sig
            fn.restype = ctypes.c_int
        _lib = l
    return _lib


def block_bytes(group: int, scale_dtype: torch.dtype, zeros: bool) -> int:
    """Bytes of a stored block of 128 rows and 128 k: codes, scales, zeros."""
    if group not in GROUPS:
        raise KernelError(f"4-bit weights come in groups of {GROUPS} values, not {group}")
    if scale_dtype is not torch.bfloat16 and scale_dtype is not torch.float32:
        raise KernelError(f"scales of 4-bit weights are bfloat16 or float32, not {scale_dtype}")
    return CODE_BYTES + K_BLOCK // group * ROWS * (scale_dtype.itemsize + (1 if zeros else 0))


class Q4Weight:
    """A matrix [n, k] of 4-bit weights in its stored form: `data` uint8 [ceil(n / 128), ceil(k / 128), block_bytes(..)], a block holding

        codes   [4: k / 32][128: row][4: k / 8 % 4] words of 32 bits; k % 8 = 4 p + 2 q + h is at bit 16 h + 8 p + 4 q of its word
        scales  [128 / group][128: row] of `scale_dtype`
        zeros   [128 / group][128: row] uint8, if `zeros`

    (what is stored behind row n and column k is not used).  `at_rest`: the program promises that no kernel which may still be running
    when a product is launched writes `data`; a product then asks for its first weights while the kernel in front of it ends.  Weights that were
    loaded once are at rest as soon as the host has waited for the device (`settle`)."""

    __slots__ = ("data", "n", "k", "group", "zeros", "scale_dtype", "at_rest", "shape", "form")
    is_q4 = True

    def __init__(self, data: torch.Tensor, n: int, k: int, group: int = 128, zeros: bool = False, scale_dtype: torch.dtype = torch.bfloat16,
                 at_rest: bool = False):
        want = (-(-n // ROWS), -(-k // K_BLOCK), block_bytes(group, scale_dtype, zeros))
        if not 1 <= n <= MOST or not 1 <= k <= MOST or k % 8:
            raise KernelError(f"4-bit weights [{n}, {k}]: the sizes are 1 to {MOST} and the second a multiple of 8")
        if data.dtype is not torch.uint8 or data.shape != want or not data.is_contiguous():
            raise KernelError(f"4-bit weights [{n}, {k}] in groups of {group} are a contiguous uint8 {list(want)}, "
                              f"not {data.dtype} {list(data.shape)}")
        if data.data_ptr() % 16:
            raise KernelError("4-bit weights start on a 16-byte boundary")
        self.data, self.n, self.k, self.group, self.zeros, self.scale_dtype, self.at_rest = data, n, k, group, bool(zeros), scale_dtype, at_rest
        self.shape = (n, k)
        self.form = group | (256 if scale_dtype is torch.float32 else 0) | (512 if zeros else 0)      # as the C entries take it

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def settle(self) -> "Q4Weight":
        """Wait for the device; from here on the weights are at rest."""
        if self.data.is_cuda:
            torch.cuda.synchronize(self.data.device)
        self.at_rest = True
        return self


def _device(t: torch.Tensor, *others: torch.Tensor) -> int:
    if not t.is_cuda:
        raise KernelError("kernel called with a CPU tensor: this engine has no CPU path")
    index = t.get_device()
    for o in others:
        if not o.is_cuda or o.get_device() != index:
            raise KernelError(f"tensors on different devices: {t.device} and {o.device}")
    return index


def _on(index: int):
    """A context in which the device `index` is the current one, or None if it is already."""
    return None if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def quantize(w: torch.Tensor, group: int = 128, zeros: bool = False, scale_dtype: torch.dtype = torch.bfloat16) -> Q4Weight:
    """A matrix [N, K], bfloat16 or float32, in 4 bits.  Of a group's values, with the scale rounded to its type (by way of float32):

        without zeros   scale = max |w| / 7;  code = 8 + clamp(rint(w / scale), -7, 7)
        with zeros      lo = min(0, min w), hi = max(0, max w), scale = (hi - lo) / 15;
                        zero = clamp(rint(-lo / scale), 0, 15);  code = clamp(rint(w / scale) + zero, 0, 15)

    rint takes ties to the even number.  A group of zeros stays zeros.  A group that holds an infinity or a value that is no number gets a
    scale that is no number."""
    if w.dim() != 2 or w.dtype not in (torch.bfloat16, torch.float32) or not w.is_contiguous():
        raise KernelError(f"quantize takes a contiguous bfloat16 or float32 matrix, not {w.dtype} {list(w.shape)}")
    index, (n, k) = _device(w), w.shape
    size = block_bytes(group, scale_dtype, zeros)
    if not 1 <= n <= MOST_ROWS or not 1 <= k <= MOST or k % 8 or w.data_ptr() % 16:
        raise KernelError(f"quantize: [{n}, {k}] needs 1 to {MOST_ROWS} rows, a multiple of 8 columns and a base on a 16-byte boundary")
    if (other := _on(index)) is not None:
        with other:
            return quantize(w, group, zeros, scale_dtype)
    blocks = -(-k // K_BLOCK)
    data = torch.empty_strided((-(-n // ROWS), blocks, size), (blocks * size, size, 1), dtype=torch.uint8, device=w.device)
    q = Q4Weight(data, n, k, group, zeros, scale_dtype)
    _check(lib().tl_quantize_q4(w.data_ptr(), int(w.dtype is torch.float32), data.data_ptr(), n, k, q.form, _stream()), "quantize_q4")
    return q


def dequantize(w: Q4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `w` stands for, [N, K]: float32, or those rounded to bfloat16."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise KernelError(f"dequantize gives bfloat16 or float32, not {dtype}")
    if w.n > MOST_ROWS:
        raise KernelError(f"dequantize: {w.n} rows are more than {MOST_ROWS}")
    if (other := _on(_device(w.data))) is not None:
        with other:
            return dequantize(w, dtype)
    out = torch.empty_strided((w.n, w.k), (w.k, 1), dtype=dtype, device=w.data.device)      # (0.8 us less of the host's time than `empty`)
    _check(lib().tl_dequantize_q4(w.data.data_ptr(), out.data_ptr(), int(dtype is torch.float32), w.n, w.k, w.form, _stream()), "dequantize_q4")
    return out


def pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, group: int = 128) -> Q4Weight:
    """Weights that were quantized elsewhere: codes [N, K] whole numbers 0..15, scales [N, ceil(K / group)] bfloat16 or float32, zeros (the
    same shape) whole numbers 0..15 or None: 8.  Works where the tensors are, on the host too; values outside 0..15 are refused."""
    if codes.dim() != 2 or codes.dtype.is_floating_point or codes.dtype.is_complex or codes.dtype == torch.bool:
        raise KernelError(f"pack: codes are whole numbers [N, K], not {codes.dtype} {list(codes.shape)}")
    n, k = codes.shape
    size = block_bytes(group, scales.dtype, zeros is not None)
    if n < 1 or k < 1 or k % 8:
        raise KernelError(f"pack: [{n}, {k}] needs positive sizes, the second a multiple of 8")
    per_row = (n, -(-k // group))
    if tuple(scales.shape) != per_row or (zeros is not None and (tuple(zeros.shape) != per_row or zeros.dtype.is_floating_point)):
        raise KernelError(f"pack: [{n}, {k}] in groups of {group} has scales (and whole zeros) of {list(per_row)}")
    for what, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and (t.device != codes.device or bool(((t < 0) | (t > 15)).any())):
            raise KernelError(f"pack: {what} are 0..15, on the codes' device")
    if scales.device != codes.device:
        raise KernelError("pack: scales are on the codes' device")
    tiles, blocks, groups = -(-n // ROWS), -(-k // K_BLOCK), K_BLOCK // group
    c = torch.full((tiles * ROWS, blocks * K_BLOCK), 8, dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes.to(torch.uint8)
    c = c.view(tiles, ROWS, blocks, 4, 4, 2, 2, 2).permute(0, 2, 3, 1, 4, 7, 5, 6)      # [tile, block, k / 32, row, word, h, p, q]
    pieces = [(c[..., 0] | (c[..., 1] << 4)).reshape(tiles, blocks, CODE_BYTES)]

    def by_block(t, fill):
        full = torch.full((tiles * ROWS, blocks * groups), fill, dtype=t.dtype, device=t.device)
        full[:n, :per_row[1]] = t
        return full.view(tiles, ROWS, blocks, groups).permute(0, 2, 3, 1).contiguous().view(tiles, blocks, groups * ROWS)

    pieces.append(by_block(scales, 0).view(torch.uint8))
    if zeros is not None:
        pieces.append(by_block(zeros.to(torch.uint8), 8))
    data = torch.cat(pieces, dim=2)
    assert data.shape[2] == size
    return Q4Weight(data, n, k, group, zeros is not None, scales.dtype)


KERNELS = ("gemv_q4", "gemm_q4", "gemm_q4_long")


def plan(T: int, n: int, k: int, sms: int) -> list:
    """The launches of a product of T tokens with a matrix [n, k] on a GPU of `sms` SMs: (tokens, kernel, tokens of a tile, ranges of K)."""
    count = lib().tl_gemm_q4_plan(T, n, k, sms, None, 0)
    room = (ctypes.c_int * (4 * count))()
    lib().tl_gemm_q4_plan(T, n, k, sms, room, count)
    return [(room[4 * i], KERNELS[room[4 * i + 1]], room[4 * i + 2], room[4 * i + 3]) for i in range(count)]


@functools.lru_cache(maxsize=4096)
def _launches(T: int, n: int, k: int, index: int) -> int:
    return lib().tl_gemm_q4_plan(T, n, k, num_sms(torch.device("cuda", index)), None, 0)


_GATES = {"silu": 1 << 10, "gelu_tanh": 2 << 10, True: 1 << 10}
_OUT_F32, _AT_REST = 1 << 12, 1 << 13
_status: dict = {}                                        # device index -> address of its status word


def _gate(gated):
    """`gated` as the C entry takes it: (bits, limit, alpha)."""
    if isinstance(gated, tuple):
        if len(gated) == 3 and gated[0] == "swish_clamped" and all(isinstance(v, (int, float)) for v in gated[1:]) and gated[1] > 0:
            return 3 << 10, float(gated[1]), float(gated[2])
    elif isinstance(gated, (str, bool)) and gated in _GATES:
        return _GATES[gated], 0.0, 1.0
    raise KernelError(f"a gated epilogue applies 'silu', 'gelu_tanh' or ('swish_clamped', limit, alpha), not {gated!r}")


def _meet(a: int, a_step: int, a_bytes: int, b: int, b_step: int, b_bytes: int, rows: int) -> bool:
    """Whether two matrices of `rows` rows share memory (addresses, bytes from row to row and of a row); said of some that only interlace too,
    but not of columns of one matrix."""
    if rows == 0 or a + (rows - 1) * a_step + a_bytes <= b or b + (rows - 1) * b_step + b_bytes <= a:
        return False
    if rows > 1 and a_step == b_step:
        ahead = (b - a) % a_step
        return ahead < a_bytes or ahead + b_bytes > a_step
    return True


def _reach(a: int, step: int, wide: int, rows: int, b: int, size: int) -> bool:
    """Whether one of `rows` rows of `wide` bytes, `step` bytes from row to row, from address a on, has a byte of the `size` at b."""
    r = max(0, (b - wide - a) // step + 1)               # the first row that ends behind b
    return r < rows and a + r * step < b + size


# A call takes the host 7 us and the smallest products 5 us, so what is asked of a tensor is asked once, and nothing is built that the call does
# not need (10.5 us with properties of the device and an argument for each of the weights' properties).
def gemm_q4(x: torch.Tensor, w: Q4Weight, out_dtype: torch.dtype = torch.bfloat16, *, gated=False, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] bfloat16 times the matrix that `w` stands for, transposed: [T, N], bfloat16 or float32, sums in float32 and rounded once.
    Rows of x may lie apart (a multiple of 8 values); T may be 0.
    `gated` ("silu", "gelu_tanh" or ("swish_clamped", limit, alpha)): w holds gate and up rows alternating in blocks of 64 (N a multiple of
    128), the result is act(gate) * up, [T, N / 2], from the float32 sums.  `out`: a tensor to write, of the result's shape and type, with rows
    that may lie apart, that shares no memory with x or w."""
    n, k, data = w.n, w.k, w.data
    form, limit, alpha = w.form, 0.0, 1.0
    if gated:
        bits, limit, alpha = _gate(gated)
        form |= bits
        if n % 128:
            raise KernelError(f"gemm_q4: gate and up rows alternate in blocks of 64, {n} rows are no multiple of 128")
    cols = n // 2 if gated else n
    shape = x.shape
    if x.dtype is not torch.bfloat16 or len(shape) != 2 or shape[1] != k or shape[0] > MOST:
        raise KernelError(f"gemm_q4: x is bfloat16 [T, {k}] of at most {MOST} tokens, not {x.dtype} {list(shape)}")
    if out_dtype is torch.float32:
        form |= _OUT_F32
    elif out_dtype is not torch.bfloat16:
        raise KernelError("gemm_q4: output is bfloat16 or float32")
    if w.at_rest:
        form |= _AT_REST
    index, T = x.get_device(), shape[0]
    if index < 0 or data.get_device() != index:
        _device(x, data)                                 # says which
    ptr = x.data_ptr()
    if T > 1:
        ldx, inner = x.stride()
    else:
        ldx, inner = k, x.stride(1)
    if T and (inner != 1 or ldx < k or ldx % 8 or ptr % 16):
        raise KernelError("gemm_q4: x has unit inner stride and rows that start on 16-byte boundaries, one behind the other")
    ldo = cols
    if out is None:
        out = torch.empty_strided((T, cols), (cols, 1), dtype=out_dtype, device=x.device)
    else:
        if T > 1:
            ldo = out.stride(0)
        if out.shape != (T, cols) or out.dtype is not out_dtype or (cols > 1 and out.stride(1) != 1) or ldo < cols:
            raise KernelError(f"gemm_q4: out is {out_dtype} [{T}, {cols}] with unit inner stride")
        _device(x, out)
        if _meet(ptr, ldx * 2, k * 2, out.data_ptr(), ldo * out_dtype.itemsize, cols * out_dtype.itemsize, T):
            raise KernelError("gemm_q4: out shares memory with x")
        if _reach(out.data_ptr(), ldo * out_dtype.itemsize, cols * out_dtype.itemsize, T, data.data_ptr(), data.numel()):
            raise KernelError("gemm_q4: out shares memory with the weights")
    if T == 0:
        return out
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return gemm_q4(x, w, out_dtype, gated=gated, out=out)
    status = _status.get(index)
    if status is None:
        status = _status[index] = device_status(x.device).data_ptr()
    code = (_lib or lib()).tl_gemm_q4(ptr, ldx, data.data_ptr(), out.data_ptr(), ldo, T, n, k, form, limit, alpha, status, torch._C._cuda_getCurrentRawStream(index))
    if T <= 128:                                         # never cut
        _check(code, "gemm_q4+gated" if gated else "gemm_q4")
    else:
        _check(code, "gemm_q4+gated" if gated else "gemm_q4", _launches(T, n, k, index))
    return out


__all__ = ["Q4Weight", "block_bytes", "dequantize", "gemm_q4", "pack", "plan", "quantize", "lib"]
