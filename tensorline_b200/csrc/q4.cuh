// Weights of 4 bits as the kernels here hold them.
//
//     w[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])          codes and zeros 0..15, zero = 8 where none is stored
//
// in blocks of 128 rows and 128 k, [ceil(N / 128)][ceil(K / 128)], each of them, without a gap,
//     codes   [4: k / 32][128: row][4: k / 8 % 4] words of 32 bits; k % 8 = 4 p + 2 q + h is at bit 16 h + 8 p + 4 q of its word
//     scales  [128 / group][128: row], bfloat16 or float
//     zeros   [128 / group][128: row] bytes, if there are any
// A thread block streams its blocks with one bulk copy each.  A row's 32 codes are one 16-byte piece, so that a warp reads 32 rows of a block
// from shared memory without a conflict; and the two values of a bfloat16 pair (k, k + 1) are the same four bits of a word's halves, so
// that one and-or makes both of them at once.  What is stored behind row N and column K is never used, whatever it is.
#pragma once
#include "umma_pair.cuh"

namespace {

constexpr int Q4_ROWS = 128, Q4_K = 128, Q4_CODES = Q4_ROWS * Q4_K / 2;

struct Q4Form { int group, groups, scale_f32, zeros, bytes; };      // k a group, groups of a block, ..., bytes of a block

// 0 if there is no such form
inline int q4_form(Q4Form* f, int group, int scale_f32, int zeros) {
    if (group != 32 && group != 64 && group != 128) return 0;
    f->group = group; f->groups = Q4_K / group; f->scale_f32 = scale_f32 != 0; f->zeros = zeros != 0;
    f->bytes = Q4_CODES + f->groups * Q4_ROWS * (f->scale_f32 ? 4 : 2) + (f->zeros ? f->groups * Q4_ROWS : 0);
    return 1;
}

__device__ __forceinline__ float q4_scale(const unsigned char* scales, int at, int f32) {
    return f32 ? reinterpret_cast<const float*>(scales)[at] : __bfloat162float(reinterpret_cast<const bf16*>(scales)[at]);
}

// Eight codes less their zero as four bfloat16 pairs, k in ascending order: 128 + code is a bfloat16 whose last four bits are the code, and
// the difference of two such numbers is exact.  `zz`: 128 + zero in both halves.
__device__ __forceinline__ void q4_values(uint32_t w, __nv_bfloat162 zz, uint32_t* out) {
    const uint32_t at[4] = {0u, 4u, 8u, 12u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = ((w >> at[i]) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), zz);
        out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}
__device__ __forceinline__ __nv_bfloat162 q4_zero(uint32_t z) {
    const uint32_t v = 0x43004300u | z | (z << 16);
    return *reinterpret_cast<const __nv_bfloat162*>(&v);
}

}  // namespace
