"""The warps of the products of many tokens with 4-bit weights share the registers of their block out anew (setmaxnreg), and wait for their share: a build
whose blocks are launched with fewer than the shares' sum is refused instead of waiting without end.  The launcher compiled for the host with stand-ins for
the CUDA calls (no GPU: nothing is launched)."""
import subprocess

from tensorline_b200.csrc.build import ARCH_FLAGS, CSRC, _nvcc

HARNESS = r"""
#include <cuda_runtime.h>
#include <cstdio>
static int registers = 0, launched = 0;
template <typename F> static cudaError_t get_attributes(cudaFuncAttributes* a, F) { *a = {}; a->numRegs = registers; return cudaSuccess; }
template <typename F> static cudaError_t set_attribute(F, cudaFuncAttribute, int) { return cudaSuccess; }
static cudaError_t get_device(int* dev) { *dev = 0; return cudaSuccess; }
template <typename... A> static cudaError_t launch(A...) { ++launched; return cudaSuccess; }
#define cudaFuncGetAttributes get_attributes
#define cudaFuncSetAttribute set_attribute
#define cudaGetDevice get_device
#define cudaLaunchKernelEx launch
#define cudaGetLastError() cudaSuccess
#include "gemm_q4_long.cu"
int main() {
    for (int r : {64, 88, 89, 96, 104}) {
        registers = r;
        CUtensorMap map{};
        Q4Args G{};
        q4_form(&G.form, 128, 0, 0);
        G.T = 64; G.N = 128; G.K = 1024; G.blocks = 8; G.per = 4;
        const int before = launched, status = ql_launch<128, false>(map, QlArgs{G, 64, 1, 1}, 1, 0);
        std::printf("%d %d %d\n", r, status, launched - before);
    }
}
"""


def test_registers_that_the_shares_count_on(tmp_path):
    (tmp_path / "harness.cu").write_text(HARNESS)
    cmd = [_nvcc(), *ARCH_FLAGS, "-O0", "-Xcicc", "-O0", "-Xptxas", "-O0", "-std=c++17", "-I", str(CSRC), "-o", str(tmp_path / "harness"), str(tmp_path / "harness.cu")]
    built = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    assert built.returncode == 0, built.stderr
    run = subprocess.run([str(tmp_path / "harness")], capture_output=True, text=True, timeout=60)
    said = [tuple(map(int, line.split())) for line in run.stdout.splitlines()]
    # a thread's registers are allocated in eights: 89 are 96, and 5 warpgroups of 96 cover 56 + 2 x 80 + 2 x 128
    assert said == [(64, 701, 0), (88, 701, 0), (89, 0, 1), (96, 0, 1), (104, 0, 1)]
