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

struct Q4Form { int group, groups, scale_f32, zeros, bytes; };      // k a group, groups of a block, ..., bytes of a block
struct Q4Args {
    const unsigned char* x; long long ldx;               // tokens, bfloat16, rows `ldx` values apart
    const unsigned char* w; int blocks;                  // packed weights; blocks of k a tile of rows has
    void* out; long long ldo; int out_f32;
    int N, K, T;
    Q4Form form;
    int per;                                             // blocks of k a range (grid z)
    int stages, stage_bytes;
    int gate; float limit, alpha;                        // 0: none, 1: silu, 2: gelu, 3: clamped swish; rows 0..63 of a tile are gates, 64..127 theirs
    int at_rest;                                         // the weights have been there since before the kernel in front: they are asked for at once
    int* status;
};

namespace {

constexpr int Q4_ROWS = 128, Q4_K = 128, Q4_CODES = Q4_ROWS * Q4_K / 2;
constexpr int Q4_MOST = 0x7fffff00;                       // tokens, rows and columns: a tile's end is still an int
constexpr int Q4_FEW = 16;                                // tokens up to which gemv_q4.cu takes a product

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
// the difference of two such numbers is exact.  `zz`: 128 + zero in both halves.  The and-or is spelt out with one of its constants in a
// register: left to itself it was two instructions, on the pipe that these kernels use most (35 us instead of 30 for 136 million weights).
__device__ __forceinline__ void q4_values(uint32_t w, uint32_t magic, __nv_bfloat162 zz, uint32_t* out) {
    const uint32_t at[4] = {0u, 4u, 8u, 12u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(v) : "r"(w >> at[i]), "r"(magic));
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), zz);
        out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}
// 128 in both halves, in a register whatever the compiler knows about it
__device__ __forceinline__ uint32_t q4_magic() {
    uint32_t m;
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(m));
    return m;
}
__device__ __forceinline__ __nv_bfloat162 q4_zero(uint32_t z) {
    const uint32_t v = 0x43004300u | z | (z << 16);
    return *reinterpret_cast<const __nv_bfloat162*>(&v);
}

__device__ __forceinline__ uint32_t q4_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
// D (+)= A B with A in tensor memory; by a whole warp, the instruction itself by one lane (umma_pair.cuh has the reason)
__device__ __forceinline__ void q4_mma(uint32_t acc, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(acc), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void q4_commit(uint32_t bar, uint32_t one) {
    asm volatile("{\n\t.reg .pred q;\n\t"
                 "setp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(bar), "r"(one) : "memory");
}

// Shared memory by its 32-bit addresses.  (A pointer whose alignment was rounded up by hand is a generic one to the compiler: loads through it took
// the long way, and every barrier's address was made again from 64 bits.)
__device__ __forceinline__ uint4 q4_lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t q4_lds8(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ float q4_lds_scale(uint32_t scales, int at, int f32) {
    if (f32) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(scales + 4 * at));
        return v;
    }
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(scales + 2 * at));
    return __uint_as_float((uint32_t)v << 16);
}
__device__ __forceinline__ bool q4_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// as mbar_wait
__device__ __forceinline__ bool q4_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    if (q4_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!q4_try(bar, parity)) {
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_CYCLES) {
            *abort_flag = 1;
            atomicCAS(status, 0, code);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void q4_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void q4_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void q4_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }

// a += s x, b += s y: the pairs of float multiply-adds of this architecture
__device__ __forceinline__ void q4_fma2(float s, float x, float y, float& a, float& b) {
    asm("{\n\t.reg .b64 m, v, c;\n\t"
        "mov.b64 m, {%2, %2};\n\tmov.b64 v, {%3, %4};\n\tmov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, m, v, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t}" : "+f"(a), "+f"(b) : "f"(s), "f"(x), "f"(y));
}
__device__ __forceinline__ void q4_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void q4_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ const float* q4_peer(const float* p, int rank) {      // the same shared-memory location in block `rank` of the cluster
    uint64_t out;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<const float*>(out);
}

__device__ __forceinline__ void q4_ld16(uint32_t at, float (&r)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
                   "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]) : "r"(at));
}
__device__ __forceinline__ void q4_ld8(uint32_t at, float (&r)[8]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "r"(at));
}
__device__ __forceinline__ void q4_st32(uint32_t at, const uint32_t (&u)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
                   "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
                   "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
                   "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
                 : "memory");
}

// act(g) u from float sums.  Every activation is g times a sigmoid, whose exponential is of a number below zero: no value of g overflows it.
__device__ __forceinline__ float q4_gate(float g, float u, int kind, float limit, float alpha) {
    float z = g;
    if (kind == 2) z = 1.5957691216057308f * (g + 0.044715f * g * g * g);        // 0.5 (1 + tanh(z / 2)) is the sigmoid of z
    else if (kind == 3) {
        g = g > limit ? limit : g;
        u = u > limit ? limit : u < -limit ? -limit : u;
        z = alpha * g;
        u += 1.0f;
    }
    // (a divide in place of the reciprocal and one Newton step for it, of a number in [1, 2], takes the longer half of a gate's time)
    const float e = expf(-fabsf(z)), d = 1.0f + e;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    return g * (z < 0.f ? e * r : r) * u;
}
__device__ __forceinline__ void q4_store(const Q4Args& G, size_t at, float v) {
    if (G.out_f32) ((float*)G.out)[at] = v;
    else ((bf16*)G.out)[at] = __float2bfloat16_rn(v);
}

// The end of a tile of 128 rows: its sums lie in shared memory, PARTS of [TOKENS][128] floats in each of the cluster's `nz` blocks, one block a
// range of K.  Block z adds up a z-th share of the tokens, in the order of the ranges and their parts, and stores it, through the gate where
// there is one: gates and what they weigh are rows 64 apart.  Thread `tid` of `threads`; behind a barrier of the cluster, and in front of one.
template <int PARTS, int TOKENS>
__device__ __forceinline__ void q4_finish(const Q4Args& G, const float* red, int tile, int t0, int nz, int z, int tid, int threads) {
    const int tokens = min(TOKENS, G.T - t0), share = (tokens + nz - 1) / nz;
    const int lo = min(tokens, z * share), hi = min(tokens, lo + share);
    const float* peer[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) peer[y] = nz > 1 ? q4_peer(red, y < nz ? y : 0) : red;
    const int wide = G.gate ? 64 : 128;                  // outputs a token has in this tile
    const int n0 = tile * wide, n_end = G.gate ? G.N / 2 : G.N;
    for (int at = tid; at < (hi - lo) * wide; at += threads) {
        const int t = lo + at / wide, r = at % wide;
        float a[8 * PARTS], u[8 * PARTS];
#pragma unroll
        for (int y = 0; y < 8; ++y)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                if (y < nz) {
                    a[y * PARTS + p] = peer[y][(p * TOKENS + t) * Q4_ROWS + r];
                    u[y * PARTS + p] = G.gate ? peer[y][(p * TOKENS + t) * Q4_ROWS + r + 64] : 0.f;
                }
        float sa = a[0], su = u[0];
#pragma unroll
        for (int y = 1; y < 8 * PARTS; ++y)
            if (y / PARTS < nz) { sa += a[y]; su += u[y]; }
        if (n0 + r < n_end) q4_store(G, (size_t)(t0 + t) * G.ldo + n0 + r, G.gate ? q4_gate(sa, su, G.gate, G.limit, G.alpha) : sa);
    }
}

// x [T, K] bfloat16 with rows `ld` values apart, boxes of `k` values (64: with the 128-byte swizzle, else without one) by `rows` tokens
inline int q4_map(CUtensorMap* map, const void* x, int T, int K, long long ld, int rows, int k) {
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)T}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)k, (cuuint32_t)rows}, elem[2] = {1, 1};
    const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, elem,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, k == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 101;
}

}  // namespace
