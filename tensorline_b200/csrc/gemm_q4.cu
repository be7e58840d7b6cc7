// Products with weights of 4 bits (q4.cuh): y[t, n] = sum_k x[t, k] w[n, k], x bfloat16, y bfloat16 or float.
//
//     y[t, n] = sum over groups g of  scale[n, g] * ( sum over the group's k of x[t, k] (code[n, k] - zero[n, g]) )
//
// The inner sum is one of the tensor cores': its factors, bfloat16 and whole numbers of at most four bits and a sign, are exact, and so are
// their products in float.  The scale joins in float, as a multiply-add of a group's sum into the output's: no weight is rounded.
//
// A block works on 128 rows of W and BN tokens over a range of K, a block of 128 k at a time.  One warp brings the packed weights (one bulk copy a
// block of k) and the tokens (by TMA, 128-byte swizzle) into a ring; four warps unpack the weights, a row a thread, straight into tensor memory,
// which is where tcgen05.mma takes its 128-row operand from; one warp issues the products; four warps take a finished group's sums out of
// tensor memory, scale and add them in registers.  Weights in tensor memory cost one store of 32 values a warp instead of a swizzled round
// trip through shared memory, and their scale is one number a thread, since a row is a lane.
// Every wait on a barrier is bounded: a block whose wait runs out records a code in `status`, stops and returns.
#include "q4.cuh"

namespace {

constexpr int QG_THREADS = 320;                          // warp 0: copies, 1: tensor memory + products, 2..5: unpacking, 6..9: sums
constexpr int QG_STAGES_MAX = 12;

template <int BN> struct QgShape {
    static constexpr int X_HALF = BN * 128, X_BYTES = 2 * X_HALF;         // BN tokens x 64 k, twice
    static constexpr int NA = BN <= 16 ? 3 : BN <= 64 ? 2 : 4;            // unpacked blocks in turn, 64 columns each
    static constexpr int ND = BN <= 32 ? 4 : 2;                           // groups' sums in turn
    static constexpr int PER_SM = BN <= 64 ? 2 : 1;
    static constexpr uint32_t COLS = BN <= 64 ? 256 : 512;
    static constexpr int D_COL = NA * 64;
    static constexpr int SMEM_MOST = PER_SM == 2 ? 112 * 1024 : 226 * 1024;
    static_assert(D_COL + ND * BN <= (int)COLS, "tensor memory");
};

struct QgArgs {
    const unsigned char* w; int blocks;                  // packed weights; blocks of k a tile of rows has
    void* out; int out_f32, ldo;
    int N, K, T;
    Q4Form form;
    int per;                                             // blocks of k a range (grid z)
    int stages, stage_bytes;
    int gate; float limit, alpha;                        // 0: none, 1: silu, 2: gelu, 3: clamped swish; rows 0..63 of a tile are gates, 64..127 theirs
    int at_rest;                                         // the weights have been there since before the kernel in front: they are asked for at once
    int* status;
};

__device__ __forceinline__ uint32_t qg_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
// D (+)= A B with A in tensor memory; by a whole warp, the instruction itself by one lane (umma_pair.cuh has the reason)
__device__ __forceinline__ void qg_mma(uint32_t acc, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(acc), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void qg_commit(uint64_t* bar, uint32_t one) {
    asm volatile("{\n\t.reg .pred q;\n\t"
                 "setp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(smem_addr(bar)), "r"(one) : "memory");
}
__device__ __forceinline__ void qg_ld16(uint32_t at, float (&r)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
                   "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]) : "r"(at));
}
__device__ __forceinline__ void qg_st32(uint32_t at, const uint32_t (&u)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
                   "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
                   "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
                   "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
                 : "memory");
}
__device__ __forceinline__ void qg_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ const float* qg_peer(const float* p, int rank) {      // the same shared-memory location in block `rank` of the cluster
    uint64_t out;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<const float*>(out);
}

// act(g) u from float sums.  Every activation is g times a sigmoid, whose exponential is of a number below zero: no value of g overflows it.
__device__ __forceinline__ float qg_gate(float g, float u, int kind, float limit, float alpha) {
    float z = g;
    if (kind == 2) z = 1.5957691216057308f * (g + 0.044715f * g * g * g);        // 0.5 (1 + tanh(z / 2)) is the sigmoid of z
    else if (kind == 3) {
        g = g > limit ? limit : g;
        u = u > limit ? limit : u < -limit ? -limit : u;
        z = alpha * g;
        u += 1.0f;
    }
    const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
    return g * (z < 0.f ? e * r : r) * u;
}
__device__ __forceinline__ void qg_store(const QgArgs& G, size_t at, float v) {
    if (G.out_f32) ((float*)G.out)[at] = v;
    else ((bf16*)G.out)[at] = __float2bfloat16_rn(v);
}

template <int BN>
__global__ void __launch_bounds__(QG_THREADS, QgShape<BN>::PER_SM)
gemm_q4_kernel(const __grid_constant__ CUtensorMap map_x, const QgArgs G) {
    using Sh = QgShape<BN>;
    constexpr int NA = Sh::NA, ND = Sh::ND;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);      // a stage: tokens, then packed weights
    const int S = G.stages;
    uint64_t* w_full = reinterpret_cast<uint64_t*>(ring + (size_t)S * G.stage_bytes);
    uint64_t* x_full = w_full + S;
    uint64_t* empty = x_full + S;                        // 4 unpacking warps, 4 summing warps, the products
    uint64_t* a_full = empty + S;                        // [NA] 4 unpacking warps
    uint64_t* a_empty = a_full + NA;                     // [NA] the products
    uint64_t* d_full = a_empty + NA;                     // [ND] the products
    uint64_t* d_empty = d_full + ND;                     // [ND] 4 summing warps
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + ND);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, t0 = blockIdx.y * BN, nz = gridDim.z;
    const int k0 = blockIdx.z * G.per, n_k = min(G.blocks, k0 + G.per) - k0;      // > 0: the launcher leaves no range empty
    const int all_groups = (G.K + G.form.group - 1) / G.form.group;
    auto groups_of = [&](int i) { return min(G.form.groups, all_groups - (k0 + i) * G.form.groups); };      // a last block's groups behind K are left out

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(w_full + s, 1); mbar_init(x_full + s, 1); mbar_init(empty + s, 9); }
        for (int b = 0; b < NA; ++b) { mbar_init(a_full + b, 4); mbar_init(a_empty + b, 1); }
        for (int b = 0; b < ND; ++b) { mbar_init(d_full + b, 1); mbar_init(d_empty + b, 4); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(Sh::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int quarter = warp & 3;                        // the lanes of tensor memory a warp reaches: 32 * (warp % 4)
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    float acc[BN];                                       // of the summing warps: a row's outputs

    if (warp == 0) {
        if (lane == 0) {
            // ------------------------------------------------------------ copies
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            const unsigned char* src = G.w + ((size_t)tile * G.blocks + k0) * G.form.bytes;
            auto load_w = [&](int i, int s) {
                mbar_expect_tx(w_full + s, G.form.bytes);
                qg_bulk(smem_addr(ring + (size_t)s * G.stage_bytes) + Sh::X_BYTES, src + (size_t)i * G.form.bytes, G.form.bytes, w_full + s);
            };
            auto load_x = [&](int i, int s) {
                const uint32_t dst = smem_addr(ring + (size_t)s * G.stage_bytes);
                mbar_expect_tx(x_full + s, Sh::X_BYTES);
                tma_box(dst, &map_x, x_full + s, (k0 + i) * Q4_K, t0);
                tma_box(dst + Sh::X_HALF, &map_x, x_full + s, (k0 + i) * Q4_K + 64, t0);
            };
            const int ahead = min(n_k, S);
            if (!G.at_rest) grid_dependency_wait();
            for (int i = 0; i < ahead; ++i) load_w(i, i);
            if (G.at_rest) grid_dependency_wait();
            grid_dependency_trigger();
            for (int i = 0; i < ahead; ++i) load_x(i, i);
            for (int i = ahead, s = 0, turn = 0; i < n_k; ++i) {
                if (!mbar_wait(empty + s, turn & 1, abort_flag, G.status, 71)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == S) { s = 0; ++turn; }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- products
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(Q4_ROWS >> 4) << 24);
        const uint32_t one = qg_elect();
        const int steps = G.form.group / 16;
        grid_dependency_wait();                          // the bounded waits start counting once the tokens can land
        int d = 0, s = 0, turn = 0;
        bool ok = true;
        for (int i = 0; i < n_k && ok; ++i) {
            const int b = i % NA;
            ok = mbar_wait(x_full + s, turn & 1, abort_flag, G.status, 72) && mbar_wait(a_full + b, (i / NA) & 1, abort_flag, G.status, 72);
            const int gs = groups_of(i);
            const uint32_t x = smem_addr(ring + (size_t)s * G.stage_bytes);
            for (int g = 0; g < gs && ok; ++g, ++d) {
                const int c = d % ND;
                if (d >= ND) ok = mbar_wait(d_empty + c, (d / ND - 1) & 1, abort_flag, G.status, 73);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int k = 0; k < steps; ++k) {
                    const int at = g * steps + k;        // 16 k: 8 columns of weights, 32 bytes of tokens
                    qg_mma(tmem + Sh::D_COL + c * BN, tmem + b * 64 + at * 8, desc_kmajor(x + (at >> 2) * Sh::X_HALF + (at & 3) * 32), idesc, k > 0, one);
                }
                qg_commit(d_full + c, one);
            }
            if (!ok) break;
            qg_commit(a_empty + b, one);
            qg_commit(empty + s, one);
            if (++s == S) { s = 0; ++turn; }
        }
    } else if (warp < 6) {
        // ---------------------------------------------------------------- unpacking
        const int row = quarter * 32 + lane, zeros_at = Q4_CODES + G.form.groups * Q4_ROWS * (G.form.scale_f32 ? 4 : 2);
        const int piece_group = G.form.group / 32;       // pieces of 32 k a group
        if (!G.at_rest) grid_dependency_wait();
        for (int i = 0, s = 0, turn = 0; i < n_k; ++i) {
            const int b = i % NA;
            if (!mbar_wait(w_full + s, turn & 1, abort_flag, G.status, 74)) break;
            const unsigned char* st = ring + (size_t)s * G.stage_bytes + Sh::X_BYTES;
            if (i >= NA && !mbar_wait(a_empty + b, (i / NA - 1) & 1, abort_flag, G.status, 74)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[32];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int piece = 2 * half + j;
                    const uint4 q = *reinterpret_cast<const uint4*>(st + (piece * Q4_ROWS + row) * 16);
                    const __nv_bfloat162 zz = q4_zero(G.form.zeros ? st[zeros_at + (piece / piece_group) * Q4_ROWS + row] : 8u);
                    q4_values(q.x, zz, v + 16 * j);
                    q4_values(q.y, zz, v + 16 * j + 4);
                    q4_values(q.z, zz, v + 16 * j + 8);
                    q4_values(q.w, zz, v + 16 * j + 12);
                }
                qg_st32(lanes + b * 64 + half * 32, v);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) { mbar_arrive(a_full + b); mbar_arrive(empty + s); }
            if (++s == S) { s = 0; ++turn; }
        }
    } else {
        // ---------------------------------------------------------------- sums
        const int row = quarter * 32 + lane;
#pragma unroll
        for (int c = 0; c < BN; ++c) acc[c] = 0.f;
        grid_dependency_wait();                          // the output may still be read by the kernel in front
        bool ok = true;
        for (int i = 0, s = 0, turn = 0, d = 0; i < n_k && ok; ++i) {
            if (!mbar_wait(w_full + s, turn & 1, abort_flag, G.status, 75)) { ok = false; break; }
            const unsigned char* scales = ring + (size_t)s * G.stage_bytes + Sh::X_BYTES + Q4_CODES;
            const int gs = groups_of(i);
            float sc[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) sc[g] = g < gs ? q4_scale(scales, g * Q4_ROWS + row, G.form.scale_f32) : 0.f;
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + s);
            if (++s == S) { s = 0; ++turn; }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (g >= gs) break;
                const int c = d % ND;
                if (!mbar_wait(d_full + c, (d / ND) & 1, abort_flag, G.status, 75)) { ok = false; break; }
                ++d;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = lanes + Sh::D_COL + c * BN;
#pragma unroll
                for (int c0 = 0; c0 < BN; c0 += 16) {
                    float r[16];
                    qg_ld16(at + c0, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[c0 + j] = fmaf(sc[g], r[j], acc[c0 + j]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(d_empty + c);
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");   // the other summing warps have read their scales out of the ring
        if (ok && nz == 1 && !G.gate) {
            const int n = tile * Q4_ROWS + row;
            if (n < G.N) {
#pragma unroll
                for (int c = 0; c < BN; ++c)
                    if (t0 + c < G.T) qg_store(G, (size_t)(t0 + c) * G.ldo + n, acc[c]);
            }
        } else if (ok) {                                 // the sums to shared memory, [token][row]: the ring is idle, every copy has been waited for
            float* red = reinterpret_cast<float*>(ring);
#pragma unroll
            for (int c = 0; c < BN; ++c) red[c * Q4_ROWS + row] = acc[c];
        }
    }
    if (nz > 1 || G.gate) {
        // The ranges of K of a tile are a cluster.  Block z adds up a z-th share of the tile's tokens over all blocks, in the ranges' order, and
        // stores it, through the gate where there is one: gates and what they weigh are rows 64 apart.
        if (nz > 1) pair_cluster_sync(); else __syncthreads();
        if (warp >= 2 && !*abort_flag) {
            const float* red = reinterpret_cast<const float*>(ring);
            const int tokens = min(BN, G.T - t0), share = (tokens + nz - 1) / nz;
            const int lo = min(tokens, (int)blockIdx.z * share), hi = min(tokens, lo + share);
            const float* peer[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) peer[z] = nz > 1 ? qg_peer(red, z < nz ? z : 0) : red;
            const int wide = G.gate ? 64 : 128;          // outputs a token has in this tile
            const int n0 = tile * wide, n_end = G.gate ? G.N / 2 : G.N;
            for (int at = (int)threadIdx.x - 64; at < (hi - lo) * wide; at += QG_THREADS - 64) {
                const int t = lo + at / wide, r = at % wide;
                float a[8], u[8];
#pragma unroll
                for (int z = 0; z < 8; ++z)
                    if (z < nz) {
                        a[z] = peer[z][t * Q4_ROWS + r];
                        u[z] = G.gate ? peer[z][t * Q4_ROWS + r + 64] : 0.f;
                    }
                float sa = a[0], su = u[0];
#pragma unroll
                for (int z = 1; z < 8; ++z)
                    if (z < nz) { sa += a[z]; su += u[z]; }
                if (n0 + r < n_end) qg_store(G, (size_t)(t0 + t) * G.ldo + n0 + r, G.gate ? qg_gate(sa, su, G.gate, G.limit, G.alpha) : sa);
            }
        }
        if (nz > 1) pair_cluster_sync();                 // nobody leaves while its shared memory is read
    }
    // -------------------------------------------------------------------- teardown
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_flag) {                                   // copies in flight land before the shared memory is handed on
        const long long begin = clock64();
        while (clock64() - begin < 2000000LL) { }
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::COLS) : "memory");
    }
}

// x [T, K] bfloat16 with rows `ld` values apart, boxes of 64 k by `rows` tokens, 128-byte swizzle
int qg_map(CUtensorMap* map, const void* x, int T, int K, long long ld, int rows) {
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)T}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)rows}, elem[2] = {1, 1};
    const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, elem,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 101;
}

template <int BN>
int qg_launch(const CUtensorMap& map, QgArgs G, int tiles, int splits, cudaStream_t stream) {
    using Sh = QgShape<BN>;
    constexpr int BARS = (3 * QG_STAGES_MAX + 2 * Sh::NA + 2 * Sh::ND) * 8 + 16;
    static bool raised[TL_MAX_DEVICES] = {};
    int e = tl_raise_smem(gemm_q4_kernel<BN>, raised, Sh::SMEM_MOST);
    if (e) return e;
    G.stage_bytes = (Sh::X_BYTES + G.form.bytes + 1023) & ~1023;
    G.stages = (Sh::SMEM_MOST - 1024 - BARS) / G.stage_bytes;
    if (G.stages > QG_STAGES_MAX) G.stages = QG_STAGES_MAX;
    if (G.stages > G.per) G.stages = G.per;
    size_t ring = (size_t)G.stages * G.stage_bytes;      // it holds the sums, [BN][128] floats, in the end
    if (ring < (size_t)BN * Q4_ROWS * 4) { G.stages = (int)(((size_t)BN * Q4_ROWS * 4 + G.stage_bytes - 1) / G.stage_bytes); ring = (size_t)G.stages * G.stage_bytes; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, (G.T + BN - 1) / BN, splits);
    cfg.blockDim = dim3(QG_THREADS);
    cfg.dynamicSmemBytes = ring + 1024 + BARS;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (tl_dependent_launch_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 1; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = splits;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t ce = cudaLaunchKernelEx(&cfg, gemm_q4_kernel<BN>, map, G);
    return ce != cudaSuccess ? (int)ce : tl_launch_status();
}

}  // namespace

// Bytes of a block of 128 rows and 128 k, 0: there is no such form.
TL_EXPORT int tl_q4_block_bytes(int group, int scale_f32, int zeros) {
    Q4Form f;
    return q4_form(&f, group, scale_f32, zeros) ? f.bytes : 0;
}

// y[T, ldo] = x[T, ldx] w^T over weights of 4 bits, N x K.  `gate` 1..3: rows of w are gates and what they weigh, alternating in blocks of 64
// (N % 128 == 0), and y [T, N / 2] is act(gate) * up: 1 silu, 2 the tanh form of gelu, 3 the clamped swish with `limit` and `alpha`.
// `at_rest`: no kernel of this stream that could still be running writes the weights.  Returns 0, a CUDA error or 1 for what it does not take.
TL_EXPORT int tl_gemm_q4(const void* x, long long ldx, const void* w, void* y, int out_f32, int ldo, int T, int N, int K, int group, int scale_f32,
                         int zeros, int gate, float limit, float alpha, int at_rest, int* status, cudaStream_t stream) {
    QgArgs G{};
    if (T < 0 || N < 1 || K < 1 || (K & 7) || !q4_form(&G.form, group, scale_f32, zeros)) return 1;
    if (gate < 0 || gate > 3 || (gate && (N & 127)) || ldo < (gate ? N / 2 : N)) return 1;
    if (T == 0) return 0;
    if (ldx < K || (ldx & 7) || ((uintptr_t)x & 15) || ((uintptr_t)w & 15) || !y || !status) return 1;
    int e = load_encode();
    if (e) return e;
    G.w = (const unsigned char*)w; G.blocks = (K + Q4_K - 1) / Q4_K;
    G.out = y; G.out_f32 = out_f32; G.ldo = ldo; G.N = N; G.K = K; G.T = T;
    G.gate = gate; G.limit = limit; G.alpha = alpha; G.at_rest = at_rest; G.status = status;
    const int bn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
    const int tiles = (N + Q4_ROWS - 1) / Q4_ROWS, t_tiles = (T + bn - 1) / bn;
    if (t_tiles > 65535) return 1;
    const int room = tl_num_sms() * (bn <= 64 ? 2 : 1);
    const long long work = (long long)tiles * t_tiles;
    int splits = work < room ? (int)(room / work) : 1;
    if (splits > 8) splits = 8;
    if (splits > G.blocks) splits = G.blocks;
    G.per = (G.blocks + splits - 1) / splits;
    splits = (G.blocks + G.per - 1) / G.per;
    CUtensorMap map;
    if ((e = qg_map(&map, x, T, K, ldx, bn))) return e;
    switch (bn) {
        case 16: return qg_launch<16>(map, G, tiles, splits, stream);
        case 32: return qg_launch<32>(map, G, tiles, splits, stream);
        case 64: return qg_launch<64>(map, G, tiles, splits, stream);
        default: return qg_launch<128>(map, G, tiles, splits, stream);
    }
}
