"""Products with weights of 4 bits into memory that the weights lie in are refused (no GPU: the rule on addresses)."""
from tensorline_b200 import ops_q4


def test_rows_that_reach_into_a_block_of_memory():
    for a in range(0, 400, 7):
        for step, wide in ((40, 40), (50, 20), (300, 10)):
            for b, size in ((100, 1), (100, 30), (130, 200)):
                for rows in (1, 2, 5, 9):
                    written = {a + r * step + c for r in range(rows) for c in range(wide)}
                    assert ops_q4._reach(a, step, wide, rows, b, size) == bool(written & set(range(b, b + size))), (a, step, wide, b, size, rows)
    assert not ops_q4._reach(0, 40, 40, 0, 0, 100)
