"""Tensor memory of the products with 4-bit weights is given back before a block waits for others of its cluster.

A block of two ranges of 128 k (19.9 KB, 30,720 registers, 256 columns) finds room beside one of the products that work in pairs and take all 512 columns
of two SMs.  If it held its columns while it waits for the cluster, its peer could be waiting for columns that one block of such a pair holds, while the
pair's other block waits for these: on two streams, without end.  Shown on the source (nothing is run): what stands between the allocation and the first wait for the cluster."""
import itertools
import os
import re

from tensorline_b200 import ops_q4


def kernel_text():
    with open(os.path.join(os.path.dirname(ops_q4.__file__), "csrc", "gemm_q4.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return text[text.index("gemm_q4_kernel(const"):text.index("int qg_launch(")]


def stuck(gives_back_first: bool) -> bool:
    """Whether some order of the four allocations ends with everybody waiting: two SMs of 512 columns, a cluster A (256 a block), a pair P (512)."""
    for order in itertools.permutations([("A", 0), ("A", 1), ("P", 0), ("P", 1)]):
        free, held, gone = [512, 512], set(), set()
        moved = True
        while moved:
            moved = False
            for block in order:
                kind, sm = block
                need = 256 if kind == "A" else 512
                peer = (kind, 1 - sm)
                if block not in held and block not in gone and free[sm] >= need:
                    free[sm] -= need
                    held.add(block)
                    moved = True
                elif block in held and (peer in held or peer in gone or (kind == "A" and gives_back_first)):
                    free[sm] += need                     # it is through, or through with its columns
                    held.discard(block)
                    gone.add(block)
                    moved = True
        if len(gone) < 4:
            return True
    return False


def test_the_order_matters():
    assert stuck(False) and not stuck(True)


def test_columns_are_given_back_before_the_cluster_is_waited_for():
    text = kernel_text()
    assert text.count("tcgen05.alloc") == text.count("tcgen05.dealloc") == 1
    assert text.index("tcgen05.alloc") < text.index("tcgen05.dealloc") < text.index("pair_cluster_sync")
