"""Products with 4-bit weights in every kernel, tile and way of cutting (`tests/q4_shapes.py`), in every form of the weights.

Whole numbers and scales that are powers of two: every sum of theirs is exact in float (below 15 x 3 x 8,200 in steps of 1/4, 21 bits), whatever its order.  What
is stored behind the last row and the last value of a row is poison, tokens and outputs lie in rows of wider matrices."""
import pytest
import torch

from tests.q4_shapes import SHAPES

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
FORMS = [(128, False, BF), (128, True, F32), (64, False, F32), (64, True, BF), (32, False, BF), (32, True, F32)]
GATES = ["silu", "gelu_tanh", ("swish_clamped", 7.0, 1.5)]


def whole(n, k, group, zeros, scale):
    """Weights of 4 bits in whole numbers, and the values that they stand for."""
    from tensorline_b200 import ops_q4
    g = torch.Generator(device="cuda").manual_seed(n + k + group)
    per_row = (n, -(-k // group))
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = 2.0 ** torch.randint(-2, 1, per_row, generator=g, device="cuda").float()
    zs = torch.randint(0, 16, per_row, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    w = ops_q4.pack(codes, scales.to(scale), zs, group)
    spread = lambda t: t.repeat_interleave(group, dim=1)[:, :k]                          # noqa: E731
    values = spread(scales) * (codes.float() - (spread(zs.float()) if zeros else 8.0))
    # poison: rows behind n, values behind k (in the last group that has any, and whole groups)
    tiles, blocks, size = w.data.shape
    groups, rows, left = 128 // group, n - (tiles - 1) * 128, k - (blocks - 1) * 128
    at = 8192 + groups * 128 * scale.itemsize
    code = w.data[:, :, :8192].view(tiles, blocks, 4, 128, 16)
    code[-1, :, :, rows:] = 0xEE
    for word in range(left // 8, 16):
        code[:, -1, word // 4, :, 4 * (word % 4):4 * (word % 4) + 4] = 0x5A
    s = w.data[:, :, 8192:at].view(scale).view(tiles, blocks, groups, 128)
    s[-1, :, :, rows:] = float("nan")
    s[:, -1, -(-left // group):] = float("inf")
    if zeros:
        z = w.data[:, :, at:].view(tiles, blocks, groups, 128)
        z[-1, :, :, rows:] = 255
        z[:, -1, -(-left // group):] = 255
    return w, values.double()


def gates(a, u, gated):
    """(result, the sigmoid's argument) in 64 bits."""
    limit, alpha = gated[1:] if isinstance(gated, tuple) else (None, 1.0)
    if limit:
        a, u = a.clamp_max(limit), u.clamp(-limit, limit) + 1
    z = 2 * (2 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3) if gated == "gelu_tanh" else alpha * a
    return a * torch.sigmoid(z) * u, z


def apart(t, k):
    """[t, k] whole numbers in rows of a wider matrix, whose other values are no numbers."""
    x = torch.full((t + 1, k + 24), float("nan"), dtype=BF, device="cuda")
    x[:t, 8:k + 8] = torch.randint(-3, 4, (t, k), generator=torch.Generator(device="cuda").manual_seed(t + k), device="cuda").to(BF)
    return x[:t, 8:k + 8]


def checked(x, w, dtype, gated, cols):
    """The product into columns of a wider matrix, nothing else of which may change."""
    from tensorline_b200 import ops_q4
    room = torch.full((x.shape[0] + 2, cols + 13), 5.0, dtype=dtype, device="cuda")
    got = ops_q4.gemm_q4(x, w, dtype, gated=gated, out=room[1:-1, 5:cols + 5]).clone()
    room[1:-1, 5:cols + 5] = 5.0
    assert bool((room == 5.0).all())
    return got


@pytest.mark.parametrize("group,zeros,scale", FORMS)
@pytest.mark.parametrize("T,n,gated_n,k", SHAPES)
def test_products(group, zeros, scale, T, n, gated_n, k):
    w, values = whole(n, k, group, zeros, scale)
    x = apart(T, k)
    want = x.double() @ values.t()
    got = checked(x, w, F32, False, n)
    assert torch.equal(got.double(), want)
    assert torch.equal(checked(x, w, BF, False, n), got.to(BF))


@pytest.mark.parametrize("group,zeros,scale", FORMS)
@pytest.mark.parametrize("T,n,gated_n,k", SHAPES)
def test_gated_products(group, zeros, scale, T, n, gated_n, k):
    """The sums are exact.  In halves of 2^-23, of the result: silu 12 (an exponential 4, its share of 1 + e in the reciprocal 2, the sum, the reciprocal, three products,
    u + 1); an argument that is off by 2^-24 a half each moves a sigmoid by its size times that: of gelu's, seven roundings (two constants, four products, a
    sum of terms of one sign), of the clamped swish's, two.  Exponentials below the smallest normal float are off by 2^-126 at most, times the sums."""
    w, values = whole(gated_n, k, group, zeros, scale)
    x = apart(T, k)
    sums = (x.double() @ values.t()).view(T, gated_n // 128, 2, 64)
    a, u = sums[:, :, 0].reshape(T, -1), sums[:, :, 1].reshape(T, -1)
    for gated in GATES:
        want, z = gates(a, u, gated)
        got = checked(x, w, F32, gated, gated_n // 2)
        roundings = {"silu": 0, "gelu_tanh": 7}.get(gated if isinstance(gated, str) else "", 2)
        bound = want.abs() * (13 + roundings * z.abs().clamp_max(104)) * 2.0 ** -24 * 1.001 + a.abs().amax() * (u.abs().amax() + 1) * 2.0 ** -126
        assert bool(((got.double() - want).abs() <= bound).all()), gated
        assert torch.equal(checked(x, w, BF, gated, gated_n // 2), got.to(BF))


@pytest.mark.parametrize("T,n,k", [(100, 2048, 4104), (128, 3584, 4104), (300, 5120, 8200), (129, 9600, 136), (700, 3584, 3080)])
@pytest.mark.parametrize("gated", [False, "silu"])
def test_the_same_bits_in_a_graph_and_behind_other_work(T, n, k, gated):
    from tensorline_b200 import ops_q4
    g = torch.Generator(device="cuda").manual_seed(T)
    w = ops_q4.quantize(torch.randn(n, k, generator=g, device="cuda"), 64, True).settle()
    x = torch.randn(T, k, generator=g, device="cuda").to(BF)
    first = ops_q4.gemm_q4(x, w, F32, gated=gated)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops_q4.gemm_q4(x, w, F32, gated=gated)
        again = ops_q4.gemm_q4(x, w, F32, gated=gated)
    for _ in range(3):
        y.zero_(); again.zero_()
        graph.replay()
        assert torch.equal(y, first) and torch.equal(again, first)


@pytest.mark.parametrize("T,n,k", [(100, 1000, 4104), (300, 5000, 8200), (97, 5000, 520), (700, 3500, 3080)])
def test_values_that_are_no_number_stay_in_their_row_and_column(T, n, k):
    w, values = whole(n, k, 64, True, F32)
    x = apart(T, k)
    scales = w.data[:, :, 8192:8192 + 1024].view(F32).view(w.data.shape[0], w.data.shape[1], 2, 128)
    scales[1, 0, 0, 5] = float("nan")                    # row 133
    x[1, 7], x[T - 1, k - 1] = float("nan"), float("nan")
    got = checked(x, w, F32, False, n)
    rows = [t for t in range(T) if t not in (1, T - 1)]
    cols = [c for c in range(n) if c != 133]
    assert bool(got[:, 133].isnan().all()) and bool(got[1].isnan().all()) and bool(got[T - 1].isnan().all())
    assert torch.equal(got[rows][:, cols].double(), x[rows].double() @ values[cols].t())
