// Products with weights of 4 bits (q4.cuh): y[t, n] = sum_k x[t, k] w[n, k], x bfloat16, y bfloat16 or float.
//
//     y[t, n] = sum over groups g of  scale[n, g] * ( sum over the group's k of x[t, k] (code[n, k] - zero[n, g]) )
//
// The inner sum is one of the tensor cores': its factors, bfloat16 and whole numbers of at most four bits and a sign, are exact, and so are
// their products in float.  The scale joins in float, as a multiply-add of a group's sum into the output's: no weight is rounded.
//
// A block works on 128 rows of W and BN tokens over a range of K, a block of 128 k at a time.  One warp brings the packed weights (one bulk copy a
// block of k) and the tokens (by TMA, 128-byte swizzle) into a ring; four warps unpack the weights, a row a thread, straight into tensor memory,
// which is where tcgen05.mma takes its 128-row operand from; one warp issues the products; four warps (eight at 128 tokens) take a finished group's sums out of
// tensor memory, scale and add them in registers.  Weights in tensor memory cost one store of 32 values a warp instead of a swizzled round
// trip through shared memory, and their scale is one number a thread, since a row is a lane.
// What bounds it: hand-overs between those warps, 540 ns a block of k at 64 tokens and 1.4 times that for two thread blocks an SM (unpacking alone 230,
// the weights' way from memory 190).  Measured in a CUDA graph on weights that are not in L2: 37,888 x 3,584 gated, 32 tokens 22.7 us, 64 tokens 29.4 us
// (floor 10.7); 3,584 x 18,944, 64 tokens 20 us (5.8), 128 tokens 24.8 (10.7); 5,120 x 13,824 in groups of 64 with zeros and float scales, 45 tokens 23.5 us (6.4).
// Every wait on a barrier is bounded: a block whose wait runs out records a code in `status`, stops and returns.
#include "q4.cuh"

int gemv_q4_ranges(int tiles, int blocks, int sms);                // gemv_q4.cu
int gemv_q4(Q4Args G, int splits, cudaStream_t stream);
int gemm_q4_long(const Q4Args& G, int bn, cudaStream_t stream);     // gemm_q4_long.cu

namespace {

constexpr int QG_STAGES_MAX = 12, QG_TILES_MOST = 65535;           // tiles of tokens: a grid's second dimension

template <int BN> struct QgShape {
    static constexpr int X_HALF = BN * 128, X_BYTES = 2 * X_HALF;         // BN tokens x 64 k, twice
    static constexpr int NA = BN <= 64 ? 2 : 4;                           // unpacked blocks in turn, 64 columns each
    static constexpr int ND = BN <= 32 ? 4 : 2;                           // groups' sums in turn
    static constexpr int PER_SM = BN <= 64 ? 2 : 1;
    static constexpr int PARTS = BN == 128 ? 2 : 1, CW = BN / PARTS;      // of the tokens, a summing warp one (two at 64: 1 to 8 % slower, at 128: 10 % faster)
    static constexpr int THREADS = 32 * (6 + 4 * PARTS);                  // warp 0: copies, 1: tensor memory + products, 2..5: unpacking, 6..: sums
    static constexpr uint32_t COLS = BN <= 64 ? 256 : 512;
    static constexpr int D_COL = NA * 64;
    static constexpr int SMEM_MOST = PER_SM == 2 ? 112 * 1024 : 226 * 1024;
    static_assert(D_COL + ND * BN <= (int)COLS, "tensor memory");
};

template <int BN, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(QgShape<BN>::THREADS, QgShape<BN>::PER_SM)
gemm_q4_kernel(const __grid_constant__ CUtensorMap map_x, const Q4Args G) {
    using Sh = QgShape<BN>;
    constexpr int NA = Sh::NA, ND = Sh::ND, GROUPS = Q4_K / GROUP, CW = Sh::CW, SUMS = 4 * Sh::PARTS;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;             // a stage: tokens, then packed weights
    const int S = G.stages;
    const uint32_t full = ring + S * G.stage_bytes;
    const uint32_t empty = full + 8 * S;                 // 4 unpacking warps, all summing warps
    const uint32_t a_full = empty + 8 * S;               // [NA] 4 unpacking warps
    const uint32_t a_empty = a_full + 8 * NA;            // [NA] all summing warps: its products are done
    const uint32_t d_full = a_empty + 8 * NA;            // [ND] the products
    const uint32_t d_empty = d_full + 8 * ND;            // [ND] all summing warps
    float* red = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)));       // the sums, [token][row], in the ring once it is idle

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, t0 = blockIdx.y * BN, nz = gridDim.z;
    const int k0 = blockIdx.z * G.per, n_k = min(G.blocks, k0 + G.per) - k0;      // > 0: the launcher leaves no range empty
    const int last = (G.K + GROUP - 1) / GROUP - (k0 + n_k - 1) * GROUPS;                  // groups of the last block that begin before K
    auto groups_of = [&](int i) { return GROUPS == 1 || i + 1 < n_k ? GROUPS : min(GROUPS, last); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { q4_init(full + 8 * s, 1); q4_init(empty + 8 * s, 4 + SUMS); }
        for (int b = 0; b < NA; ++b) { q4_init(a_full + 8 * b, 4); q4_init(a_empty + 8 * b, SUMS); }
        for (int b = 0; b < ND; ++b) { q4_init(d_full + 8 * b, 1); q4_init(d_empty + 8 * b, SUMS); }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(Sh::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int quarter = warp & 3;                        // the lanes of tensor memory a warp reaches: 32 * (warp % 4)
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    float acc[CW];                                       // of the summing warps: a row's outputs

    if (warp == 0) {
        if (lane == 0) {
            // ------------------------------------------------------------ copies
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            const unsigned char* src = G.w + ((size_t)tile * G.blocks + k0) * G.form.bytes;
            auto load_w = [&](int i, int s) {
                q4_expect(full + 8 * s, Sh::X_BYTES + G.form.bytes);
                q4_bulk(ring + s * G.stage_bytes + Sh::X_BYTES, src + (size_t)i * G.form.bytes, G.form.bytes, full + 8 * s);
            };
            auto load_x = [&](int i, int s) {
                const uint32_t dst = ring + s * G.stage_bytes;
                q4_box(dst, &map_x, full + 8 * s, (k0 + i) * Q4_K, t0);
                q4_box(dst + Sh::X_HALF, &map_x, full + 8 * s, (k0 + i) * Q4_K + 64, t0);
            };
            const int ahead = min(n_k, S);
            if (!G.at_rest) grid_dependency_wait();
            for (int i = 0; i < ahead; ++i) load_w(i, i);
            if (G.at_rest) grid_dependency_wait();
            grid_dependency_trigger();
            for (int i = 0; i < ahead; ++i) load_x(i, i);
            for (int i = ahead, s = 0, turn = 0; i < n_k; ++i) {
                if (!q4_wait(empty + 8 * s, turn & 1, abort_flag, G.status, 71)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == S) { s = 0; ++turn; }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- products
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(Q4_ROWS >> 4) << 24);
        const uint32_t one = q4_elect();
        grid_dependency_wait();                          // the bounded waits start counting once the tokens can land
        int d = 0, s = 0;
        bool ok = true;
        for (int i = 0; i < n_k && ok; ++i) {
            const int b = i % NA;
            ok = q4_wait(a_full + 8 * b, (i / NA) & 1, abort_flag, G.status, 72);
            const int gs = groups_of(i);
            const uint64_t x = desc_kmajor(ring + s * G.stage_bytes);
            const uint32_t a = tmem + b * 64;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                if (g >= gs || !ok) break;
                const int c = d % ND;
                if (d >= ND) ok = q4_wait(d_empty + 8 * c, (d / ND - 1) & 1, abort_flag, G.status, 73);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int k = 0; k < GROUP / 16; ++k) {
                    constexpr int STEP = 16;             // 16 k: 8 columns of weights, 32 bytes of tokens (2 of a descriptor's units of 16)
                    const int at = g * (GROUP / STEP) + k;
                    q4_mma(tmem + Sh::D_COL + c * BN, a + at * 8, x + ((at >> 2) * Sh::X_HALF + (at & 3) * 32) / 16, idesc, k > 0, one);
                }
                q4_commit(d_full + 8 * c, one);
                ++d;
            }
            if (!ok) break;
            if (++s == S) s = 0;
        }
    } else if (warp < 6) {
        // ---------------------------------------------------------------- unpacking
        const int row = quarter * 32 + lane, zeros_at = Q4_CODES + G.form.groups * Q4_ROWS * (G.form.scale_f32 ? 4 : 2);
        grid_dependency_wait();                          // as above
        const uint32_t magic = q4_magic();
        for (int i = 0, s = 0, turn = 0; i < n_k; ++i) {
            const int b = i % NA;
            if (!q4_wait(full + 8 * s, turn & 1, abort_flag, G.status, 74)) break;
            const uint32_t st = ring + s * G.stage_bytes + Sh::X_BYTES;
            uint4 q[4];
            uint32_t z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                q[j] = q4_lds128(st + (j * Q4_ROWS + row) * 16);
                z[j] = ZEROS ? q4_lds8(st + zeros_at + (j * 32 / GROUP) * Q4_ROWS + row) : 8u;
            }
            if (i >= NA && !q4_wait(a_empty + 8 * b, (i / NA - 1) & 1, abort_flag, G.status, 74)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[32];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 p = q[2 * half + j];
                    const __nv_bfloat162 zz = q4_zero(z[2 * half + j]);
                    q4_values(p.x, magic, zz, v + 16 * j);
                    q4_values(p.y, magic, zz, v + 16 * j + 4);
                    q4_values(p.z, magic, zz, v + 16 * j + 8);
                    q4_values(p.w, magic, zz, v + 16 * j + 12);
                }
                q4_st32(lanes + b * 64 + half * 32, v);
                if (half == 0) {                         // the codes are in registers: the stage is free
                    __syncwarp();
                    if (lane == 0) q4_arrive(empty + 8 * s);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) q4_arrive(a_full + 8 * b);
            if (++s == S) { s = 0; ++turn; }
        }
    } else {
        // ---------------------------------------------------------------- sums
        const int row = quarter * 32 + lane, part = (warp - 6) >> 2;
#pragma unroll
        for (int c = 0; c < CW; ++c) acc[c] = 0.f;
        grid_dependency_wait();                          // the output may still be read by the kernel in front
        bool ok = true;
        for (int i = 0, s = 0, d = 0; i < n_k && ok; ++i) {
            const uint32_t scales = ring + s * G.stage_bytes + Sh::X_BYTES + Q4_CODES, done = empty + 8 * s;
            const int gs = groups_of(i);
            if (++s == S) s = 0;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                if (g >= gs) break;
                const int c = d % ND;
                // over when the products are, and so is the stage's copy, which they came after
                if (!q4_wait(d_full + 8 * c, (d / ND) & 1, abort_flag, G.status, 75)) { ok = false; break; }
                ++d;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (g == gs - 1 && lane == 0) q4_arrive(a_empty + 8 * (i % NA));
                const float sc = q4_lds_scale(scales, g * Q4_ROWS + row, G.form.scale_f32);
                const uint32_t at = lanes + Sh::D_COL + c * BN + part * CW;
                constexpr int AT_ONCE = 16;
#pragma unroll
                for (int c0 = 0; c0 < CW; c0 += AT_ONCE) {
                    float r[AT_ONCE / 16][16];
#pragma unroll
                    for (int j = 0; j < AT_ONCE / 16; ++j) q4_ld16(at + c0 + 16 * j, r[j]);
                    tmem_ld_wait();
                    if (c0 + AT_ONCE >= CW) {            // the last of them are in registers
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            q4_arrive(d_empty + 8 * c);
                            if (g == gs - 1) q4_arrive(done);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < AT_ONCE; j += 2) q4_fma2(sc, r[j / 16][j % 16], r[j / 16][j % 16 + 1], acc[c0 + j], acc[c0 + j + 1]);
                }
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"n"(32 * (SUMS + 1)) : "memory");   // the other summing warps have read their scales out of the ring; warp 1 gives tensor memory back
        if (ok && nz == 1 && !G.gate) {
            const int n = tile * Q4_ROWS + row;
            if (n < G.N) {
#pragma unroll
                for (int c = 0; c < CW; ++c)
                    if (t0 + part * CW + c < G.T) q4_store(G, (size_t)(t0 + part * CW + c) * G.ldo + n, acc[c]);
            }
        } else if (ok) {                                 // the sums to shared memory, [token][row]: the ring is idle, every copy has been waited for
#pragma unroll
            for (int c = 0; c < CW; ++c) red[(part * CW + c) * Q4_ROWS + row] = acc[c];
        }
    }
    // Tensor memory goes back as soon as the sums have left it, before anyone waits for the cluster: a block that holds columns waits for its own copies
    // only.  (On two streams this kernel's clusters and a product in pairs, which takes all columns of two SMs, could each hold what the other waits for.)
    if (warp == 1) {
        asm volatile("bar.sync 1, %0;" ::"n"(32 * (SUMS + 1)) : "memory");
        if (*abort_flag) {                               // products in flight end first
            const long long begin = clock64();
            while (clock64() - begin < 2000000LL) { }
        }
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::COLS) : "memory");
    }
    if (nz > 1 || G.gate) {
        if (nz > 1) pair_cluster_sync(); else __syncthreads();
        if (warp >= 2 && !*abort_flag) q4_finish<1, BN>(G, red, tile, t0, nz, blockIdx.z, (int)threadIdx.x - 64, Sh::THREADS - 64);
        if (nz > 1) pair_cluster_sync();                 // nobody leaves while its shared memory is read
    }
    // -------------------------------------------------------------------- teardown
    __syncthreads();
    if (*abort_flag) {                                   // copies in flight land before the shared memory is handed on
        const long long begin = clock64();
        while (clock64() - begin < 2000000LL) { }
    }
}

template <int BN, int GROUP, bool ZEROS>
int qg_launch(const CUtensorMap& map, Q4Args G, int tiles, int splits, cudaStream_t stream) {
    using Sh = QgShape<BN>;
    constexpr int BARS = (2 * QG_STAGES_MAX + 2 * Sh::NA + 2 * Sh::ND) * 8 + 16;
    static bool raised[TL_MAX_DEVICES] = {};
    int e = tl_raise_smem(gemm_q4_kernel<BN, GROUP, ZEROS>, raised, Sh::SMEM_MOST);
    if (e) return e;
    G.stage_bytes = (Sh::X_BYTES + G.form.bytes + 1023) & ~1023;
    G.stages = (Sh::SMEM_MOST - 1024 - BARS) / G.stage_bytes;
    if (G.stages > QG_STAGES_MAX) G.stages = QG_STAGES_MAX;
    if (G.stages > G.per) G.stages = G.per;
    size_t ring = (size_t)G.stages * G.stage_bytes;      // it holds the sums, [BN][128] floats, in the end
    if (ring < (size_t)BN * Q4_ROWS * 4) { G.stages = (int)(((size_t)BN * Q4_ROWS * 4 + G.stage_bytes - 1) / G.stage_bytes); ring = (size_t)G.stages * G.stage_bytes; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, (G.T + BN - 1) / BN, splits);
    cfg.blockDim = dim3(Sh::THREADS);
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
    const cudaError_t ce = cudaLaunchKernelEx(&cfg, gemm_q4_kernel<BN, GROUP, ZEROS>, map, G);
    return ce != cudaSuccess ? (int)ce : tl_launch_status();
}

template <int BN>
int qg_launch_form(const CUtensorMap& map, const Q4Args& G, int tiles, int splits, cudaStream_t stream) {
    if (G.form.zeros)
        return G.form.group == 128 ? qg_launch<BN, 128, true>(map, G, tiles, splits, stream) :
               G.form.group == 64 ? qg_launch<BN, 64, true>(map, G, tiles, splits, stream) : qg_launch<BN, 32, true>(map, G, tiles, splits, stream);
    return G.form.group == 128 ? qg_launch<BN, 128, false>(map, G, tiles, splits, stream) :
           G.form.group == 64 ? qg_launch<BN, 64, false>(map, G, tiles, splits, stream) : qg_launch<BN, 32, false>(map, G, tiles, splits, stream);
}

// How a product's tokens are gone through, and about how long that takes.
struct QgPlan { int bn, long_, splits, first; double us; };      // tokens of a tile; of gemm_q4_long.cu?; ranges of K; tokens before the rest is planned anew

// Ranges of K in clusters, for one launch over `tiles` of `bn` tokens.  An SM that has two thread blocks takes 1.4 times as long for a block of k of
// each; of 148 SMs about 133 get a block in clusters of two or three, 118 in clusters of four and 98 in larger ones (of two a SM 266, of seven and
// more 252), and clusters that find no room begin when others have ended.  Measured at 1, 2 .. 8 ranges, us:  45 tokens, 40 tiles x 108 blocks of k
// 57 33 24 25 22 19 28 26;  64, 28 x 148: 77 44 31 25 27 24 23 20;  64, 216 x 40: 37 38 47 48 50 56;  128, 28 x 148: 70 44 32 25 41 36;
// 128, 74 x 28: 18 19 28 33;  90, 16 x 32: 19 15 12 9.8 9.2 8.7.
QgPlan qg_ranges(long long tiles, int blocks, int bn, int sms) {
    const int two = bn <= 64;
    QgPlan p{bn, 0, 1, 0, 0};
    for (int s = 1; s <= 8 && s <= blocks; ++s) {
        const int per = (blocks + s - 1) / s;
        if ((blocks + per - 1) / per != s) continue;     // a range would be empty
        const long long total = tiles * s, alone = s == 1 || sms == 1 ? sms : s <= 3 ? sms * 9 / 10 : s == 4 ? sms * 4 / 5 : sms * 2 / 3;
        const long long both = s == 1 ? 2 * sms : s <= 6 ? sms * 9 / 5 : sms * 17 / 10;
        const double turns = total <= alone ? 1 : two ? 1.4 * ((total + both - 1) / both) : (total + alone - 1) / alone;
        const double us = two ? turns * (per + 4) * (bn == 32 ? 0.5 : 0.6) + 2 : turns * (per * 0.44 + (s == 1 ? 5.5 : 9));
        if (s == 1 || us < p.us) { p.splits = s; p.us = us; }
    }
    return p;
}

// One launch.  The blocks of gemm_q4_long.cu, one a SM, take a block of k through in 410, 420, 450 and 520 ns at 32, 64, 96 and 128 tokens: of its
// tiles, the one with which they are done first.  Up to 64 tokens, and where there are so few tiles that many SMs would have none, ranges of K
// in clusters are faster.  Measured, us, here / there:  128 tokens, 28 tiles x 148 blocks of k 25 / 65;  74 x 28 18 / 15.6;  256 tokens, 28 x 148 45 / 68.
QgPlan qg_one(int T, int m_tiles, int blocks, int sms) {
    const int here = T <= 32 ? 32 : T <= 64 ? 64 : 128;
    QgPlan p = qg_ranges((long long)m_tiles * ((T + here - 1) / here), blocks, here, sms);
    if (T > 64)
        for (int bn = 128; bn >= 32; bn -= 32) {
            const long long items = (long long)m_tiles * ((T + bn - 1) / bn), rounds = (items + sms - 1) / sms;
            const double us = (double)rounds * blocks * (0.37 + 0.0011 * bn) + 3;
            if (us < p.us || (!p.long_ && (T + here - 1) / here > QG_TILES_MOST)) p = QgPlan{bn, 1, 0, 0, us};
        }
    return p;
}

// Many tokens leave SMs idle in their last round of tiles, nearly all of them at worst: the tokens of that round may be better off by themselves, in
// tiles of another size or in ranges of K.  Measured, us, at once / so:  2,048 tokens, 28 tiles of rows x 148 blocks of k (448 tiles, four more than
// three rounds take) 340 / 275;  700 tokens 136 / 100;  1,500 tokens, 40 x 108 239 / 206;  2,048 tokens, 1,188 x 28 2,245 / 1,985.
QgPlan qg_plan(int T, int m_tiles, int blocks, int sms) {
    QgPlan p = qg_one(T, m_tiles, blocks, sms);
    for (int bn = 128; T > 128 && bn >= 64; bn -= 32) {
        const long long rounds = ((long long)m_tiles * ((T + bn - 1) / bn) + sms - 1) / sms - 1;      // full ones
        const long long first = rounds * sms / m_tiles * bn;
        if (first <= 0 || first >= T) continue;
        const double us = (double)rounds * blocks * (0.37 + 0.0011 * bn) + 5 + qg_one(T - (int)first, m_tiles, blocks, sms).us;
        if (us < p.us) p = QgPlan{bn, 1, 0, (int)first, us};
    }
    return p;
}

// The next launch of a product of T tokens, and the tokens it takes.
enum { QG_GEMV, QG_HERE, QG_LONG };
struct QgLaunch { int tokens, kernel, bn, splits; };
QgLaunch qg_next(int T, int m_tiles, int blocks, int sms) {
    if (T <= Q4_FEW) return QgLaunch{T, QG_GEMV, T <= 8 ? 8 : 16, gemv_q4_ranges(m_tiles, blocks, sms)};
    const QgPlan p = qg_plan(T, m_tiles, blocks, sms);
    return QgLaunch{p.first ? p.first : T, p.long_ ? QG_LONG : QG_HERE, p.bn, p.long_ ? 1 : p.splits};
}

int qg_run(Q4Args G, const QgLaunch& p, cudaStream_t stream) {
    if (p.kernel == QG_GEMV) return gemv_q4(G, p.splits, stream);
    if (p.kernel == QG_LONG) return gemm_q4_long(G, p.bn, stream);
    const int tiles = (G.N + Q4_ROWS - 1) / Q4_ROWS;
    G.per = (G.blocks + p.splits - 1) / p.splits;
    CUtensorMap map;
    const int e = q4_map(&map, G.x, G.T, G.K, G.ldx, p.bn, 64);
    if (e) return e;
    switch (p.bn) {
        case 32: return qg_launch_form<32>(map, G, tiles, p.splits, stream);
        case 64: return qg_launch_form<64>(map, G, tiles, p.splits, stream);
        default: return qg_launch_form<128>(map, G, tiles, p.splits, stream);
    }
}

}  // namespace

// Bytes of a block of 128 rows and 128 k, 0: there is no such form.
TL_EXPORT int tl_q4_block_bytes(int group, int scale_f32, int zeros) {
    Q4Form f;
    return q4_form(&f, group, scale_f32, zeros) ? f.bytes : 0;
}

// y[T, ldo] = x[T, ldx] w^T over weights of 4 bits, N x K.  `form`: k a group, and from bit 8 on: scales are float, there are zeros, (two bits) the
// gate, y is float, no kernel of this stream that could still be running writes the weights.  Gate 1..3: rows of w are gates and what they
// weigh, alternating in blocks of 64 (N % 128 == 0), and y [T, N / 2] is act(gate) * up: 1 silu, 2 the tanh form of gelu, 3 the clamped
// swish with `limit` and `alpha`.  Returns 0, a CUDA error or 1 for what it does not take.
TL_EXPORT int tl_gemm_q4(const void* x, long long ldx, const void* w, void* y, long long ldo, int T, int N, int K, int form, float limit, float alpha,
                         int* status, cudaStream_t stream) {
    Q4Args G{};
    const int gate = form >> 10 & 3, out_f32 = form >> 12 & 1;
    if (form < 0 || form >> 14 || T < 0 || T > Q4_MOST || N < 1 || N > Q4_MOST || K < 1 || K > Q4_MOST || (K & 7) || !q4_form(&G.form, form & 255, form >> 8 & 1, form >> 9 & 1)) return 1;
    if ((gate && (N & 127)) || ldo < (gate ? N / 2 : N)) return 1;
    if (T == 0) return 0;
    if (ldx < K || (ldx & 7) || ((uintptr_t)x & 15) || ((uintptr_t)w & 15) || !y || !status) return 1;
    const int at_rest = form >> 13 & 1;
    int e = load_encode();
    if (e) return e;
    G.x = (const unsigned char*)x; G.ldx = ldx; G.w = (const unsigned char*)w; G.blocks = (K + Q4_K - 1) / Q4_K;
    G.out = y; G.out_f32 = out_f32; G.ldo = ldo; G.N = N; G.K = K; G.T = T;
    G.gate = gate; G.limit = limit; G.alpha = alpha; G.at_rest = at_rest; G.status = status;
    const int m_tiles = (N + Q4_ROWS - 1) / Q4_ROWS, sms = tl_num_sms();
    for (int left = T; left > 0;) {
        const QgLaunch p = qg_next(left, m_tiles, G.blocks, sms);
        G.T = p.tokens;
        if ((e = qg_run(G, p, stream))) return e;
        left -= p.tokens;
        G.x += (size_t)p.tokens * G.ldx * 2;
        G.out = (unsigned char*)G.out + (size_t)p.tokens * G.ldo * (out_f32 ? 4 : 2);
    }
    return 0;
}

// The launches that `tl_gemm_q4` makes of a product of T tokens with N x K weights on `sms` SMs: their number, 0 for sizes that it does not take.  The
// first `room` of them to `launches`, four ints each: its tokens, its kernel (0 gemv_q4.cu, 1 this file's, 2 gemm_q4_long.cu), the
// tokens of a tile, the ranges of K.
TL_EXPORT int tl_gemm_q4_plan(int T, int N, int K, int sms, int* launches, int room) {
    if (T < 1 || T > Q4_MOST || N < 1 || N > Q4_MOST || K < 1 || K > Q4_MOST || (K & 7) || sms < 1 || (room > 0 && !launches)) return 0;
    int n = 0;
    for (int left = T; left > 0; ++n) {
        const QgLaunch p = qg_next(left, (N + Q4_ROWS - 1) / Q4_ROWS, (K + Q4_K - 1) / Q4_K, sms);
        if (n < room) { launches[4 * n] = p.tokens; launches[4 * n + 1] = p.kernel; launches[4 * n + 2] = p.bn; launches[4 * n + 3] = p.splits; }
        left -= p.tokens;
    }
    return n;
}
