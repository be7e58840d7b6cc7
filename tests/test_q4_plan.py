"""How products with weights of 4 bits are cut into launches (no GPU: the plan is the host's)."""
import math
import random

import pytest

from tensorline_b200 import ops_q4
from tests.q4_shapes import SHAPES, SMS, ways

SIZES = [(t, n, k) for t in (1, 8, 9, 16, 17, 32, 33, 64, 65, 100, 128, 129, 333, 512, 643, 700, 1284, 2048, 2049, 5000, 100_000)
         for n, k in ((1, 8), (128, 128), (640, 8192), (3584, 18944), (37888, 3584), (152064, 3584), (300, 1_000_000))]


@pytest.mark.parametrize("sms", [148, 132, 2, 1])
def test_every_token_is_taken_once_and_every_range_holds_something(sms):
    for T, n, k in SIZES:
        launches = ops_q4.plan(T, n, k, sms)
        blocks = -(-k // 128)
        assert sum(tokens for tokens, *_ in launches) == T and all(tokens > 0 for tokens, *_ in launches)
        assert len(launches) == 1 or T > 128             # what `gemm_q4` counts on
        for tokens, kernel, tile, ranges in launches:
            assert 1 <= ranges <= 8 and -(-blocks // -(-blocks // ranges)) == ranges
            assert tile in {"gemv_q4": (8, 16), "gemm_q4": (32, 64, 128), "gemm_q4_long": (32, 64, 96, 128)}[kernel]
            assert (kernel == "gemv_q4") == (tokens <= 16) and (kernel != "gemv_q4" or tokens <= tile) and (kernel != "gemm_q4_long" or ranges == 1)


def test_sizes_that_no_product_has():
    lib = ops_q4.lib()
    for T, n, k, sms in ((0, 128, 64, 148), (1, 0, 64, 148), (1, 128, 60, 148), (1, 128, 64, 0), (0x7fffff01, 128, 64, 148)):
        assert lib.tl_gemm_q4_plan(T, n, k, sms, None, 0) == 0
    assert lib.tl_gemm_q4_plan(700, 3584, 4096, 148, None, 0) == 2 and lib.tl_gemm_q4_plan(700, 3584, 4096, 148, None, 2) == 0      # nowhere to write them


@pytest.mark.parametrize("T", [65535 * 128, 65535 * 128 + 1, 9_000_000, 0x7fffff00])
@pytest.mark.parametrize("n,k", [(8, 10_000), (8, 20_000), (1, 200_000), (128, 8)])
def test_grids_that_a_launch_can_have(T, n, k):
    """Tiles of tokens are the grid's second dimension in `gemm_q4`, which ends at 65,535; `gemm_q4_long` has one block an SM."""
    for tokens, kernel, tile, _ in ops_q4.plan(T, n, k, 148):
        assert kernel != "gemm_q4" or -(-tokens // tile) <= 65535


def test_the_tested_shapes_take_every_way_that_there_is():
    """Sizes all over the range, drawn: what a plan does with one of them is in `test_q4_shapes_gpu.py`, plain and gated, whatever the prices are changed to."""
    rng = random.Random(5)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))    # noqa: E731
    seen = set()
    for _ in range(20_000):
        n, k = log(1, 160_000), 8 * log(1, 4000)
        seen |= ways(ops_q4.plan(log(1, 5000), n, k, SMS), n)
    for kind in (1, 2):
        tested = set().union(*(ways(ops_q4.plan(shape[0], shape[kind], shape[3], SMS), shape[kind]) for shape in SHAPES))
        assert seen <= tested, sorted(seen - tested)
    assert {tile for kernel, tile, _ in seen if kernel == "gemm_q4"} == {32, 64, 128} and {tile for kernel, tile, _ in seen if kernel == "gemm_q4_long"} >= {64, 96, 128}
    ranges = {r for T, n, _, k in SHAPES for _, kernel, tile, r in ops_q4.plan(T, n, k, SMS) if (kernel, tile) == ("gemm_q4", 128)}
    assert ranges >= {1, 2, 3, 4, 6, 7, 8}
