"""Weights of 4 bits: quantization against float64, code for code, and the products at the edges of their tiles.

Whole numbers small enough that every float sum of theirs is exact are compared for equality.  Elsewhere a float sum of K products, scaled by
groups, is off by less than (K + K / group) 2^-23 times the sum of the absolute products, and a result that is rounded to bfloat16 by 2^-8 of
itself."""
import pytest
import torch

from tests.plain.q4_plain import quantized, unpack, values

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
FORMS = [(128, False, BF), (64, True, F32), (32, True, BF), (32, False, F32)]


@pytest.fixture(scope="module")
def q4():
    from tensorline_b200 import ops_q4
    return ops_q4


def whole(q4, n, k, group, zeros, scale, seed=0):
    """Random codes with scales that are powers of two, on the GPU; and their values."""
    g = torch.Generator().manual_seed(seed + n * k)
    per_row = (n, -(-k // group))
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = 2.0 ** torch.randint(-2, 1, per_row, generator=g).float()
    zs = torch.randint(0, 16, per_row, generator=g) if zeros else None
    w = q4.pack(codes.cuda(), scales.to(scale).cuda(), None if zs is None else zs.cuda(), group)
    spread = lambda t: t.repeat_interleave(group, dim=1)[:, :k]                          # noqa: E731
    return w, (spread(scales).double() * (codes - (spread(zs) if zeros else 8)).double()).cuda()


def whole_x(t, k, seed=1):
    return torch.randint(-3, 4, (t, k), generator=torch.Generator().manual_seed(seed + t)).to(BF).cuda()


# ------------------------------------------------------------------ into four bits and back
@pytest.mark.parametrize("n,k", [(1, 8), (130, 136), (257, 1032), (40, 3000)])
@pytest.mark.parametrize("group,zeros,scale", FORMS + [(128, True, BF), (64, False, BF)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_codes_scales_and_zeros(q4, n, k, group, zeros, scale, dtype):
    g = torch.Generator().manual_seed(n)
    m = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 3)).to(dtype)
    m[n // 2, :min(k, group)] = 0.0                      # a group of zeros
    m[0, ::3] = m[0, ::3].abs() + 1                      # mostly above zero
    w = q4.quantize(m.cuda(), group, zeros, scale)
    codes, scales, zs = quantized(m, group, zeros, scale)
    got, got_scales, got_zeros = unpack(w)
    assert torch.equal(got_scales, scales)
    assert zs is None or torch.equal(got_zeros, zs)
    assert torch.equal(got, codes)
    for out in (F32, BF):
        assert torch.equal(q4.dequantize(w, out).cpu(), values(w).float().to(out))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", [BF, F32])
def test_quotients_half_way_between_two_codes(q4, zeros, scale):
    """Scales that are powers of two, values at and one float beside every half-way mark."""
    marks = torch.arange(0, 15 if zeros else 7).float() + 0.5
    rows = []
    for e in (0, -3, 20):
        for sign in ((1,) if zeros else (1, -1)):
            for step in (0, 1, -1):
                v = (marks * 2.0 ** e).view(torch.int32) + step
                row = torch.zeros(32)
                row[:len(marks)] = v.view(torch.float32) * sign
                row[31] = (15.0 if zeros else 7.0) * 2.0 ** e
                rows.append(row)
    m = torch.stack(rows)
    w = q4.quantize(m.cuda(), 32, zeros, scale)
    codes, scales, zs = quantized(m, 32, zeros, scale)
    got, got_scales, got_zeros = unpack(w)
    assert torch.equal(got_scales, scales) and torch.equal(got, codes) and (zs is None or torch.equal(zs, got_zeros))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", [BF, F32])
def test_the_smallest_and_the_largest_values(q4, zeros, scale):
    g = torch.Generator().manual_seed(3)
    m = torch.randn(64, 64, generator=g)
    size = torch.tensor([3e38, 1e30, 1e-30, 1e-36, 1e-38, 1e-40, 1e-42, 1e-44]).repeat(8)[:, None]
    m = (m / m.abs().amax(1, keepdim=True)).double().mul(size.double()).float()
    m[5, 3], m[6, 40], m[7, 0] = float("nan"), float("inf"), float("-inf")
    m[8, :32], m[8, 0] = 1.0, -1e-30                     # the difference of the largest and the smallest is no float
    w = q4.quantize(m.cuda(), 32, zeros, scale)
    codes, scales, zs = quantized(m, 32, zeros, scale)
    got, got_scales, got_zeros = unpack(w)
    assert torch.equal(got_scales.nan_to_num(-1.0), scales.nan_to_num(-1.0)) and int(got_scales.isnan().sum()) == 3
    assert torch.equal(got, codes) and (zs is None or torch.equal(zs, got_zeros))
    out = q4.dequantize(w)
    assert bool(out[5, :32].isnan().all()) and bool(out[6, 32:].isnan().all()) and bool(out[7, :32].isnan().all()) and int(out.isnan().sum()) == 96


def test_what_cannot_be_quantized(q4):
    from tensorline_b200.ops import KernelError
    m = torch.zeros(4, 64, device="cuda")
    for bad in (lambda: q4.quantize(m.half()), lambda: q4.quantize(m.t()), lambda: q4.quantize(m[:, :60].contiguous()), lambda: q4.quantize(m[0]),
                lambda: q4.quantize(m, group=16), lambda: q4.quantize(m, scale_dtype=torch.float16), lambda: q4.quantize(m[:0]),
                lambda: q4.quantize(torch.zeros(4 * 64 + 1, device="cuda")[1:].view(4, 64)), lambda: q4.dequantize(q4.quantize(m), torch.float16)):
        with pytest.raises(KernelError):
            bad()


# ------------------------------------------------------------------ products
@pytest.mark.parametrize("group,zeros,scale", FORMS)
@pytest.mark.parametrize("T", [1, 16, 17, 33, 64, 65, 200])
@pytest.mark.parametrize("n,k", [(1, 8), (128, 128), (200, 264), (1500, 1032)])
def test_whole_numbers_exactly(q4, group, zeros, scale, T, n, k):
    w, m = whole(q4, n, k, group, zeros, scale)
    x = whole_x(T, k)
    want = x.double() @ m.t()
    got = q4.gemm_q4(x, w, F32)
    assert torch.equal(got.double(), want)
    assert torch.equal(q4.gemm_q4(x, w), want.float().to(BF))


@pytest.mark.parametrize("T,n,k", [(1, 4608, 3584), (8, 3584, 18944), (45, 5120, 13824), (9, 40000, 512), (2048, 640, 1024), (333, 7168, 640)])
def test_whole_numbers_at_layer_sizes(q4, T, n, k):
    w, m = whole(q4, n, k, 128, False, BF)
    x = whole_x(T, k)
    assert torch.equal(q4.gemm_q4(x, w, F32).double(), x.double() @ m.t())


@pytest.mark.parametrize("T", [643, 700, 1284])
@pytest.mark.parametrize("gated", [False, "silu"])
def test_tokens_of_a_last_round_by_themselves(q4, T, gated):
    """One or two full rounds of tiles and a few tokens more, which another kernel, or other tiles, take; rows that lie apart."""
    n, k = 3584, 4096
    w, values_ = whole(q4, n, k, 128, False, BF)
    x = whole_x(T, k)
    sums = x.double() @ values_.T
    cols = n // 2 if gated else n
    room = torch.full((T + 1, cols + 24), 7.0, dtype=F32, device="cuda")
    wide = torch.zeros(T, k + 40, dtype=BF, device="cuda")
    wide[:, :k] = x
    q4.gemm_q4(wide[:, :k], w, F32, gated=gated, out=room[:T, :cols])
    if gated:
        sums = sums.view(T, n // 128, 2, 64)
        want = gates(sums[:, :, 0].reshape(T, -1), sums[:, :, 1].reshape(T, -1), gated)
        assert ((room[:T, :cols].double() - want).abs() <= 12 * 2.0 ** -24 * want.abs() + 2.0 ** -100).all()      # (test_gates_of_short_sums_tile_after_tile)
    else:
        assert torch.equal(room[:T, :cols].double(), sums)
    assert (room[T:] == 7).all() and (room[:, cols:] == 7).all()


@pytest.mark.parametrize("group,zeros,scale", FORMS)
@pytest.mark.parametrize("T,n,k", [(3, 333, 2000), (40, 257, 3000), (130, 129, 1544), (1, 100, 18944)])
def test_sums_in_float(q4, group, zeros, scale, T, n, k):
    g = torch.Generator().manual_seed(T)
    w = q4.quantize((torch.randn(n, k, generator=g) * 0.02).cuda(), group, zeros, scale)
    x = torch.randn(T, k, generator=g).to(BF).cuda()
    m = values(w).cuda()
    want, size = x.double() @ m.t(), x.double().abs() @ m.abs().t()
    got = q4.gemm_q4(x, w, F32)
    assert bool(((got.double() - want).abs() <= (k + k / group) * 2.0 ** -23 * size).all())
    assert torch.equal(q4.gemm_q4(x, w), got.to(BF))     # one rounding more


def gates(a, u, gated):
    if gated == "silu":
        return a * torch.sigmoid(a) * u
    if gated == "gelu_tanh":
        return torch.nn.functional.gelu(a, approximate="tanh") * u
    _, limit, alpha = gated
    a = a.clamp_max(limit)
    return a * torch.sigmoid(alpha * a) * (u.clamp(-limit, limit) + 1)


@pytest.mark.parametrize("gated", ["silu", "gelu_tanh", ("swish_clamped", 1.5, 1.7)])
@pytest.mark.parametrize("T,n,k", [(1, 128, 64), (5, 640, 1032), (33, 384, 2048), (64, 38400, 136), (77, 256, 520), (130, 896, 264), (1, 37888, 128)])
def test_gates(q4, gated, T, n, k):
    g = torch.Generator().manual_seed(T)
    w = q4.quantize((torch.randn(n, k, generator=g) * k ** -0.5).cuda(), 64, True, F32)
    x = (torch.randn(T, k, generator=g) * 2).to(BF).cuda()
    m = values(w).cuda()
    z, size = x.double() @ m.t(), x.double().abs() @ m.abs().t() * (k + k / 64) * 2.0 ** -23
    pair = lambda t: t.view(T, n // 128, 2, 64).unbind(2)                                 # noqa: E731
    (a, u), (da, du) = [[h.reshape(T, -1) for h in pair(t)] for t in (z, size)]
    want = gates(a, u, gated)
    slope = 1.2 * (u.abs() + 2) * da + (a.abs() + 0.2) * du + 1.2 * da * du              # the gates' slopes are below 1.2
    # an exponential, a division and three products in float, of an argument that is off by 2^-22 of itself
    own = want.abs() * (8 + 2 * a.abs()) * 2.0 ** -22
    for out in (F32, BF):
        got = q4.gemm_q4(x, w, out, gated=gated)
        assert got.shape == (T, n // 2)
        assert bool(((got.double() - want).abs() <= (slope + own) * 1.01 + (want.abs() * 2.0 ** -8 if out is BF else 0)).all())


def test_gates_of_short_sums_tile_after_tile(q4):
    """Several tiles a block, whose sums are one or two groups: what changes places for one tile is read before the next one's is written."""
    for k, group in ((64, 64), (128, 64), (128, 128)):
        w, values_ = whole(q4, 600 * 64, k, group, False, F32)
        x = whole_x(192, k)
        sums = (x.double() @ values_.T).view(192, 300, 2, 64)
        got = q4.gemm_q4(x, w, F32, gated="silu").double()
        want = gates(sums[:, :, 0].reshape(192, -1), sums[:, :, 1].reshape(192, -1), "silu")
        # Exact sums.  In halves of 2^-23: an exponential e (4), times its share of 1 + e in the reciprocal of that (2), the sum, the reciprocal and
        # three products: 11.  Exponentials below the smallest normal float, 2^-126, weigh sums of less than 2^13.
        assert ((got - want).abs() <= 12 * 2.0 ** -24 * want.abs() + 2.0 ** -100).all()
        assert torch.equal(got, q4.gemm_q4(x, w, F32, gated="silu").double())


def test_far_gates(q4):
    """Gates whose exponential is no float any more: the quotient is small or nothing, never a number that is none."""
    a = torch.tensor([-1e4, -200.0, -100.0, -88.0, 0.0, 88.0, 200.0, 1e4])
    codes = torch.full((128, 32), 8)
    codes[:64, 0], codes[64:, 1] = 9, 9
    w = q4.pack(codes.cuda(), torch.ones(128, 1).cuda(), group=32)
    x = torch.zeros(8, 32)
    x[:, 0], x[:, 1] = a, 2.0 ** 60
    x = x.to(BF).cuda()
    a = x[:, 0].double()
    for gated in ("silu", "gelu_tanh", ("swish_clamped", 1e30, 1.0)):
        got = q4.gemm_q4(x, w, F32, gated=gated)[:, 0].double()
        want = gates(a, x[:, 1].double(), gated if isinstance(gated, str) else ("swish_clamped", 1e30, 1.0))
        assert bool(((got - want).abs() <= want.abs() * (8 + 2 * a.abs().clamp_max(200)) * 2.0 ** -22 + 2.0 ** (60 - 126) * 1e4).all()), (gated, got, want)


@pytest.mark.parametrize("T", [1, 7, 70])
def test_what_lies_behind_the_matrix_is_not_used(q4, T):
    n, k = 140, 136                                      # one group of 32 of the last block has eight values, three have none
    w, m = whole(q4, n, k, 32, True, F32)
    data = w.data.clone()
    codes = data[:, :, :8192].view(2, 2, 4, 128, 16)
    codes[1, :, :, n - 128:] = 0xEE
    codes[:, 1, 1:] = 0x5A                               # k 160 and on
    codes[:, 1, 0, :, 4:] = 0x77                         # k 136 and on
    scales = data[:, :, 8192:8192 + 2048].view(torch.float32).view(2, 2, 4, 128)
    scales[1, :, :, n - 128:] = float("nan")
    scales[:, 1, 1:] = float("inf")
    data[1, :, 8192 + 2048:].view(2, 4, 128)[:, :, n - 128:] = 255
    x = whole_x(T, k)
    got = q4.gemm_q4(x, q4.Q4Weight(data, n, k, 32, True, F32), F32)
    assert torch.equal(got.double(), x.double() @ m.t())


@pytest.mark.parametrize("T", [4, 40, 100])
def test_values_that_are_no_number_stay_in_their_row_and_column(q4, T):
    w, m = whole(q4, 300, 256, 128, False, F32)
    scales = w.data[:, :, 8192:].view(torch.float32).view(3, 2, 1, 128)
    scales[1, 0, 0, 5] = float("nan")                    # row 133
    x = whole_x(T, 256)
    x[1, 7], x[2, 200] = float("nan"), float("inf")
    got = q4.gemm_q4(x, w, F32)
    rows = [t for t in range(T) if t not in (1, 2)]
    cols = [c for c in range(300) if c != 133]
    assert bool(got[:, 133].isnan().all()) and bool(got[1].isnan().all())
    assert torch.equal(got[rows][:, cols].double(), x[rows].double() @ m[cols].t())
    want = (x[2].double() @ m.t())[cols]                 # an infinity times zero is no number
    assert torch.equal(got[2, cols].double().nan_to_num(7.0, 1.0, -1.0), want.nan_to_num(7.0, 1.0, -1.0))


@pytest.mark.parametrize("T", [2, 50, 129])
@pytest.mark.parametrize("gated", [False, "silu"])
def test_rows_that_lie_apart(q4, T, gated):
    w, m = whole(q4, 384, 200, 64, True, BF)
    wide = whole_x(T, 264)
    x = wide[:, 64:]
    assert x.stride(0) == 264 and x.shape[1] == 200
    n = 192 if gated else 384
    room = torch.full((T + 2, n + 9), 5.0, device="cuda")
    got = q4.gemm_q4(x, w, F32, gated=gated, out=room[1:T + 1, 3:n + 3])
    assert torch.equal(got, q4.gemm_q4(x.contiguous(), w, F32, gated=gated))
    if not gated:
        assert torch.equal(got.double(), x.double() @ m.t())
    room[1:T + 1, 3:n + 3] = 5.0
    assert bool((room == 5.0).all())


@pytest.mark.parametrize("T,gated", [(2, False), (2, "silu"), (40, False), (130, "silu")])
def test_rows_more_than_31_bits_apart(q4, T, gated):
    far = 2 ** 31 + 8 if T == 2 else 2 ** 31 // 32
    w, _ = whole(q4, 256, 128, 64, False, BF)
    x = whole_x(T, 128)
    cols = 128 if gated else 256
    room = torch.empty((T - 1) * far + 256, dtype=BF, device="cuda")
    wide = room.as_strided((T, cols), (far, 1))
    assert q4.gemm_q4(x, w, gated=gated, out=wide) is wide
    assert torch.equal(wide, q4.gemm_q4(x, w, gated=gated))
    tokens = room.as_strided((T, 128), (far, 1))
    tokens.copy_(x)
    assert torch.equal(q4.gemm_q4(tokens, w, gated=gated), q4.gemm_q4(x, w, gated=gated))


def test_refusals(q4):
    from tensorline_b200.ops import KernelError
    w, _ = whole(q4, 128, 64, 64, False, BF)
    x = whole_x(4, 64)
    wide = whole_x(4, 80)
    for bad in (lambda: q4.gemm_q4(wide[:, 4:68], w), lambda: q4.gemm_q4(whole_x(4, 68)[:, :64], w), lambda: q4.gemm_q4(whole_x(64, 4).t(), w),
                lambda: q4.gemm_q4(x[:1].expand(4, 64), w), lambda: q4.gemm_q4(x, w, out=torch.empty(4, 128, device="cuda")),
                lambda: q4.gemm_q4(x, w, out=torch.empty(128, 4, dtype=BF, device="cuda").t()), lambda: q4.gemm_q4(x, w, out=torch.empty(4, 128, dtype=BF)),
                lambda: q4.gemm_q4(x, w, out=torch.empty(1, 128, dtype=BF, device="cuda").expand(4, 128))):
        with pytest.raises(KernelError):
            bad()
    assert q4.gemm_q4(x[:0], w).shape == (0, 128) and q4.gemm_q4(x[:0], w, F32, gated=True).shape == (0, 64)
    assert torch.equal(q4.gemm_q4(x[2:3].expand(1, 64), w), q4.gemm_q4(x, w)[2:3])


@pytest.mark.parametrize("T", [1, 40, 200])
def test_outputs_beside_tokens_not_in_them(q4, T):
    from tensorline_b200.ops import KernelError
    w, _ = whole(q4, 128, 128, 64, False, BF)
    room = torch.zeros(T + 1, 256, dtype=BF, device="cuda")
    room[:T, :128] = whole_x(T, 128)
    x, want = room[:T, :128], q4.gemm_q4(whole_x(T, 128), w)
    for out in (x, room[:T, 64:192], room[1:, :128] if T > 1 else x):
        with pytest.raises(KernelError, match="shares memory"):
            q4.gemm_q4(x, w, out=out)
    assert torch.equal(q4.gemm_q4(x, w, out=room[:T, 128:]), want) and torch.equal(room[:T, :128], whole_x(T, 128))


# ------------------------------------------------------------------ streams, graphs, one call behind another
def test_made_and_used_without_a_wait(q4):
    """Weights that the kernel in front is still writing: a product that was not promised anything waits for them."""
    for i in range(20):
        m = torch.full((4096, 4096), float(i + 1), device="cuda").to(BF)
        x = torch.ones(1, 4096, dtype=BF, device="cuda")
        got = q4.gemm_q4(x, q4.quantize(m), F32)
        want = 4096 * 7 * torch.tensor((i + 1) / 7).to(BF).double().item()
        assert bool((got.double() == want).all())


def test_another_stream(q4):
    w, m = whole(q4, 2000, 1024, 128, False, BF)
    x = whole_x(20, 1024)
    want = x.double() @ m.t()
    torch.cuda.synchronize()
    w.settle()
    side, got = torch.cuda.Stream(), []
    with torch.cuda.stream(side):
        for _ in range(8):
            got.append(q4.gemm_q4(x, w, F32))
    here = [q4.gemm_q4(x, w, F32) for _ in range(8)]     # beside those on the other stream
    torch.cuda.synchronize()
    for y in got + here:
        assert torch.equal(y.double(), want)


@pytest.mark.parametrize("T", [1, 30, 64, 300])
def test_two_captured_graphs(q4, T):
    """Nothing is shared between them: replays in any order, on other inputs."""
    made = []
    for seed, gated in ((0, False), (1, "silu")):
        w, m = whole(q4, 512, 640, 32, True, BF, seed)
        w.settle()
        x = whole_x(T, 640)
        q4.gemm_q4(x, w, F32, gated=gated)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = q4.gemm_q4(x, w, F32, gated=gated)
        made.append((graph, x, y, w, m, gated))
    for seed in (5, 6):
        for graph, x, *_ in made:
            x.copy_(whole_x(T, 640, seed))
        for graph, *_ in made + made[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for _, x, y, w, m, gated in made:
            assert torch.equal(y, q4.gemm_q4(x, w, F32, gated=gated))
            if not gated:
                assert torch.equal(y.double(), x.double() @ m.t())


@pytest.mark.parametrize("T,n,k", [(8, 1024, 4096), (100, 4096, 1024), (1, 30000, 256)])
def test_the_same_call_gives_the_same_bits(q4, T, n, k):
    g = torch.Generator().manual_seed(T)
    w = q4.quantize(torch.randn(n, k, generator=g).cuda()).settle()
    x = torch.randn(T, k, generator=g).to(BF).cuda()
    first = q4.gemm_q4(x, w, F32)
    assert all(torch.equal(first, q4.gemm_q4(x, w, F32)) for _ in range(10))


def test_a_feed_forward_as_it_is_used(q4):
    """quantize, the gated product, the product behind it: against the same in float64 from the values that the weights stand for."""
    g = torch.Generator().manual_seed(0)
    T, H, I = 19, 768, 1280
    gate_up = q4.quantize((torch.randn(2 * I, H, generator=g) * H ** -0.5).to(BF).cuda())
    down = q4.quantize((torch.randn(H, I, generator=g) * I ** -0.5).to(BF).cuda(), 64, True)
    x = torch.randn(T, H, generator=g).to(BF).cuda()
    m = q4.gemm_q4(x, gate_up, gated="silu")
    y = q4.gemm_q4(m, down)
    a, u = [t.reshape(T, -1) for t in (x.double() @ values(gate_up).cuda().t()).view(T, I // 64, 2, 64).unbind(2)]
    want = (a * torch.sigmoid(a) * u) @ values(down).cuda().t()
    # two roundings to bfloat16 of at most 2^-8, the inner one of terms whose errors add up at most as their norms do
    inner = (a * torch.sigmoid(a) * u).norm(dim=1, keepdim=True) * 2.0 ** -8 * 1.01
    bound = inner * values(down).cuda().norm(dim=1)[None] + want.abs() * 2.0 ** -8 * 1.01
    assert bool(((y.double() - want).abs() <= bound).all())
