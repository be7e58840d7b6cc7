// Products of many tokens with weights of 4 bits (q4.cuh): the sums of gemm_q4.cu in persistent blocks, one a SM.
//
// A block works on 128 rows of W and BN tokens (32 to 128).  Eight warps in two groups unpack every other block of 128 k into tensor memory (a
// row a thread), one warp issues eight products of 16 k a block, eight warps scale a finished group's sums and add them to the outputs', which
// they hold in registers, 64 a thread at most.  Tensor memory: four blocks of unpacked weights (64 columns each) and two groups' sums (2 x 128),
// all of it.  The ring of copies and the buffers run on from one tile to the next.
// What bounds it: the summing warps' chain.  A block of k takes 1,000 cycles at 128 tokens, of which the tensor cores need 520; the summing warps have one thing
// to do behind the other, most of it waiting (125 cycles for the products, of which 80 however long ago they were over, twice 200 for a load of
// 32 columns from tensor memory; 125 for their multiply-adds, which share their pipe with the unpacking, 70 for two arrivals).  Measured in a CUDA
// graph, 37,888 x 3,584 gated: 96 tokens 35 us (floor 16), 2,048 tokens 631 to 651 us (floor 341: 0.86 PFLOP/s); 7,168 x 5,120, 333 tokens: 42 us (15).
// Not faster: pairs of blocks on 256 rows and 192 tokens (half as many bytes of tokens; they hand over through the cluster, about 500 cycles a time,
// with no tensor memory left to hide it: 1,250 cycles a block of k and 5 a token), sixteen summing warps of 32 tokens (2 % slower: 80 registers
// are too few), tokens and weights in rings of their own (7 %: one commit more), two warps that issue products, more warps that unpack.
#include "q4.cuh"

namespace {

constexpr int QL_THREADS = 640;                          // warp 0: copies, 1: tensor memory + products, 4..11: unpacking, 12..19: sums
// registers a thread of those groups of warps: 56 + 2 x 80 + 2 x 128 of the 5 x 96 that the block is launched with
constexpr int QL_REGS_COPY = 56, QL_REGS_UNPACK = 80, QL_REGS_SUM = 128;
static_assert(QL_REGS_COPY + 2 * QL_REGS_UNPACK + 2 * QL_REGS_SUM <= 5 * 96, "a larger share would be waited for without end");
constexpr int QL_MOST = 128, QL_CW = QL_MOST / 2;        // tokens of a tile, of a summing warp
constexpr int QL_NA = 4, QL_ND = 2, QL_D_COL = QL_NA * 64;      // unpacked blocks of k in turn (64 columns), groups' sums in turn
constexpr int QL_STAGES_MAX = 12, QL_SMEM = 226 * 1024, QL_HAND = 2 * 2 * 16 * 64 * 4;      // gates and what they weigh change places: [in turn: 2][half][16][64]
static_assert(QL_D_COL + QL_ND * QL_MOST <= 512, "tensor memory");

struct QlArgs { Q4Args g; int bn, m_tiles, t_tiles; };

// Half of a tile's tokens goes out, 32 rows a warp: `cw` of them, from t0 on.
template <typename TY>
__device__ __forceinline__ bool ql_tile_out(const Q4Args& G, const float (&acc)[QL_CW], int cw, int tile, int t0, int quarter, int lane, float* hand, uint32_t handed,
                                            int& hands, volatile int* abort_flag) {
    auto put = [](TY* at, float v) {
        if constexpr (sizeof(TY) == 4) *at = v; else *at = __float2bfloat16_rn(v);
    };
    const int left = G.T - t0;                           // tokens that there are
    if (!G.gate) {
        const int n = tile * Q4_ROWS + quarter * 32 + lane, count = n < G.N ? left : 0;
        TY* to = (TY*)G.out + t0 * G.ldo + n;
#pragma unroll
        for (int c0 = 0; c0 < QL_CW; c0 += 16) {
            if (c0 >= cw) break;
#pragma unroll
            for (int c = c0; c < c0 + 16; ++c, to += G.ldo)
                if (c < count) put(to, acc[c]);
        }
        return true;
    }
    // Gates are rows 0..63 of a tile and lie in other warps than what they weigh: of 16 tokens at a time the one side hands over its values of the
    // first eight, the other of the second, and each finishes eight.  (Two buffers in turn: whoever writes one again has waited for the
    // hand-over in between, which nobody makes before it has read the one.)
    const bool up = quarter >= 2;
    const int f = (quarter & 1) * 32 + lane, first = up ? 8 : 0;
    TY* to = (TY*)G.out + (t0 + first) * G.ldo + tile * 64 + f;
#pragma unroll
    for (int c0 = 0; c0 < QL_CW; c0 += 16, to += 8 * G.ldo) {
        if (c0 >= cw) break;
        float* h = hand + (hands & 1) * (2 * 16 * 64) + f;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[(up ? j : 8 + j) * 64] = up ? acc[c0 + j] : acc[c0 + 8 + j];
        __syncwarp();
        if (lane == 0) q4_arrive(handed);
        if (!q4_wait(handed, hands & 1, abort_flag, G.status, 86)) return false;
        ++hands;
#pragma unroll
        for (int j = 0; j < 8; ++j, to += G.ldo) {
            const float mine = up ? acc[c0 + 8 + j] : acc[c0 + j], other = h[(first + j) * 64];
            const float y = q4_gate(up ? other : mine, up ? mine : other, G.gate, G.limit, G.alpha);
            if (c0 + first + j < left) put(to, y);
        }
    }
    return true;
}

template <int GROUP, bool ZEROS>
__global__ void __launch_bounds__(QL_THREADS, 1)
gemm_q4_long_kernel(const __grid_constant__ CUtensorMap map_x, const QlArgs A) {
    constexpr int NA = QL_NA, ND = QL_ND, GROUPS = Q4_K / GROUP;
    const Q4Args& G = A.g;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;             // a stage: tokens, packed weights
    const int S = G.stages, BN = A.bn, x_half = BN * 128, x_bytes = 2 * x_half;
    float* hand = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)) + S * G.stage_bytes);
    const uint32_t full = ring + S * G.stage_bytes + QL_HAND;
    const uint32_t empty = full + 8 * S;                 // 4 unpacking warps, 8 summing warps
    const uint32_t a_full = empty + 8 * S;               // [NA] 4 unpacking warps
    const uint32_t a_empty = a_full + 8 * NA;            // [NA] the products
    const uint32_t d_full = a_empty + 8 * NA;            // [ND] the products
    const uint32_t d_empty = d_full + 8 * ND;            // [ND] 8 summing warps
    const uint32_t handed = d_empty + 8 * ND;            // [2] the 4 summing warps of a half

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = blockIdx.x, step = gridDim.x, items = A.m_tiles * A.t_tiles, n_k = G.blocks;
    const int last = (G.K + GROUP - 1) / GROUP - (n_k - 1) * GROUPS;                         // groups of the last block that begin before K

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { q4_init(full + 8 * s, 1); q4_init(empty + 8 * s, 12); }
        for (int b = 0; b < NA; ++b) { q4_init(a_full + 8 * b, 4); q4_init(a_empty + 8 * b, 1); }
        for (int b = 0; b < ND; ++b) { q4_init(d_full + 8 * b, 1); q4_init(d_empty + 8 * b, 8); }
        for (int h = 0; h < 2; ++h) q4_init(handed + 8 * h, 4);
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);

    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(QL_REGS_COPY));
      if (warp == 0) {
        // ---------------------------------------------------------------- copies
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            const unsigned char* src = nullptr;          // the tile's weights
            int t0 = 0;                                  // and tokens
            auto begin = [&](int item) {
                src = G.w + (size_t)(item / A.t_tiles) * n_k * G.form.bytes;
                t0 = (item % A.t_tiles) * BN;
            };
            auto load_w = [&](int c, int s) {
                q4_expect(full + 8 * s, x_bytes + G.form.bytes);
                q4_bulk(ring + s * G.stage_bytes + x_bytes, src + (size_t)c * G.form.bytes, G.form.bytes, full + 8 * s);
            };
            auto load_x = [&](int c, int s) {
                const uint32_t dst = ring + s * G.stage_bytes;
                q4_box(dst, &map_x, full + 8 * s, c * Q4_K, t0);
                q4_box(dst + x_half, &map_x, full + 8 * s, c * Q4_K + 64, t0);
            };
            const int ahead = min(S, n_k);
            begin(first);
            if (!G.at_rest) grid_dependency_wait();
            for (int c = 0; c < ahead; ++c) load_w(c, c);
            if (G.at_rest) grid_dependency_wait();
            grid_dependency_trigger();
            for (int c = 0; c < ahead; ++c) load_x(c, c);
            int s = 0, turn = 0, it = 0;
            bool ok = true;
            for (int item = first; item < items && ok; item += step) {
                begin(item);
                for (int c = 0; c < n_k; ++c, ++it) {
                    if (it >= ahead) {
                        if (it >= S && !q4_wait(empty + 8 * s, (turn - 1) & 1, abort_flag, G.status, 81)) { ok = false; break; }
                        load_w(c, s);
                        load_x(c, s);
                    }
                    if (++s == S) { s = 0; ++turn; }
                }
            }
        }
      } else if (warp == 1) {
        // ---------------------------------------------------------------- products
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(Q4_ROWS >> 4) << 24);
            const uint32_t one = q4_elect();
            grid_dependency_wait();                      // the bounded waits start counting once the tokens can land
            int d = 0, s = 0, n = 0;                     // groups, stage, blocks so far
            bool ok = true;
            for (int item = first; item < items && ok; item += step) {
                for (int c = 0; c < n_k && ok; ++c, ++n) {
                    const int b = n % NA, gs = GROUPS == 1 || c + 1 < n_k ? GROUPS : last;
                    // (the unpacking warps have waited for the stage, its tokens too)
                    if (!q4_wait(a_full + 8 * b, (n / NA) & 1, abort_flag, G.status, 82)) { ok = false; break; }
                    const uint64_t x = desc_kmajor(ring + s * G.stage_bytes);
                    const uint32_t a = tmem + b * 64;
                    if (++s == S) s = 0;
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        if (g >= gs || !ok) break;
                        const int e = d % ND;
                        if (d >= ND) ok = q4_wait(d_empty + 8 * e, (d / ND - 1) & 1, abort_flag, G.status, 83);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                        for (int k = 0; k < GROUP / 16; ++k) {
                            constexpr int STEP = 16;     // 16 k: 8 columns of weights, 32 bytes of tokens (2 of a descriptor's units of 16)
                            const int at = g * (GROUP / STEP) + k;
                            q4_mma(tmem + QL_D_COL + e * QL_MOST, a + at * 8, x + (at >> 2) * (x_half / 16) + (at & 3) * 2, idesc, k > 0, one);
                        }
                        q4_commit(d_full + 8 * e, one);
                        ++d;
                    }
                    if (ok) q4_commit(a_empty + 8 * b, one);
                }
            }
      }
    } else if (warp < 12) {
        // ---------------------------------------------------------------- unpacking: every other block of k a group of four warps
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(QL_REGS_UNPACK));
        const int row = quarter * 32 + lane, zeros_at = Q4_CODES + GROUPS * Q4_ROWS * (G.form.scale_f32 ? 4 : 2);
        const uint32_t magic = q4_magic();
        grid_dependency_wait();                          // as above
        const int mine = (warp - 4) >> 2;
        const int blocks = ((items - first + step - 1) / step) * n_k;                    // of k, of all of its tiles
        int s = mine, turn = 0;
        for (int n = mine; n < blocks; n += 2) {
            const int b = n % NA;
            if (!q4_wait(full + 8 * s, turn & 1, abort_flag, G.status, 84)) break;
            const uint32_t st = ring + s * G.stage_bytes + x_bytes;
            const uint32_t done = empty + 8 * s;
            uint4 q[4];
            uint32_t z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                q[j] = q4_lds128(st + (j * Q4_ROWS + row) * 16);
                z[j] = ZEROS ? q4_lds8(st + zeros_at + (j * 32 / GROUP) * Q4_ROWS + row) : 8u;
            }
            if (n >= NA && !q4_wait(a_empty + 8 * b, (n / NA - 1) & 1, abort_flag, G.status, 84)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            s += 2;                                      // S is even: a stage stays with its group
            if (s >= S) { s -= S; ++turn; }
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
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) { q4_arrive(a_full + 8 * b); q4_arrive(done); }
        }
    } else {
        // ---------------------------------------------------------------- sums: 32 rows and half of the tokens a warp
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(QL_REGS_SUM));
        const int row = quarter * 32 + lane, half = (warp - 12) >> 2, cw = BN / 2;
        grid_dependency_wait();                          // the output may still be read by the kernel in front
        int s = 0, d = 0, hands = 0;                     // times that values changed places
        bool ok = true;
        for (int item = first; item < items && ok; item += step) {
            float acc[QL_CW];
#pragma unroll
            for (int c = 0; c < QL_CW; ++c) acc[c] = 0.f;
            for (int c = 0; c < n_k && ok; ++c) {
                const uint32_t scales = ring + s * G.stage_bytes + x_bytes + Q4_CODES, done = empty + 8 * s;
                const int gs = GROUPS == 1 || c + 1 < n_k ? GROUPS : last;
                if (++s == S) s = 0;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    if (g >= gs) break;
                    const int e = d % ND;
                    // over when the products are, and so is the stage's copy, which they came after
                    if (!q4_wait(d_full + 8 * e, (d / ND) & 1, abort_flag, G.status, 85)) { ok = false; break; }
                    ++d;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const float sc = q4_lds_scale(scales, g * Q4_ROWS + row, G.form.scale_f32);
                    const uint32_t at = lanes + QL_D_COL + e * QL_MOST + half * cw;
#pragma unroll
                    for (int c0 = 0; c0 < QL_CW; c0 += 32) {     // 32 columns at a time: a load's way takes 100 cycles
                        if (c0 >= cw) break;
                        float r[32];
                        if (c0 + 32 <= cw) tmem_ld32(at + c0, r);
                        else q4_ld16(at + c0, *reinterpret_cast<float(*)[16]>(&r));
                        tmem_ld_wait();
                        if (c0 + 32 >= cw) {             // the last of them are in registers
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) {
                                q4_arrive(d_empty + 8 * e);
                                if (g == gs - 1) q4_arrive(done);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            if (j < 16 || c0 + 32 <= cw) q4_fma2(sc, r[j], r[j + 1], acc[c0 + j], acc[c0 + j + 1]);
                    }
                }
            }
            if (!ok) break;
            const int tile = item / A.t_tiles, t0 = (item % A.t_tiles) * BN + half * cw;
            float* h = hand + half * (16 * 64);
            if (G.out_f32) ok = ql_tile_out<float>(G, acc, cw, tile, t0, quarter, lane, h, handed + 8 * half, hands, abort_flag);
            else ok = ql_tile_out<bf16>(G, acc, cw, tile, t0, quarter, lane, h, handed + 8 * half, hands, abort_flag);
        }
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int GROUP, bool ZEROS>
int ql_launch(const CUtensorMap& map, const QlArgs& A, int blocks, cudaStream_t stream) {
    static bool raised[TL_MAX_DEVICES] = {};
    const int dev = tl_device_index();
    if (dev >= 0 && !raised[dev]) {                      // the shares are of what this build's blocks are launched with
        cudaFuncAttributes a;
        const cudaError_t ce = cudaFuncGetAttributes(&a, gemm_q4_long_kernel<GROUP, ZEROS>);
        if (ce != cudaSuccess) return (int)ce;
        if (5 * ((a.numRegs + 7) & ~7) < QL_REGS_COPY + 2 * QL_REGS_UNPACK + 2 * QL_REGS_SUM) return (int)cudaErrorLaunchOutOfResources;
    }
    const int e = tl_raise_smem(gemm_q4_long_kernel<GROUP, ZEROS>, raised, QL_SMEM);
    if (e) return e;
    return launch_after_wait(gemm_q4_long_kernel<GROUP, ZEROS>, dim3(blocks), dim3(QL_THREADS), QL_SMEM, stream, map, A);
}

}  // namespace

// The product of G.T tokens in tiles of `bn` (a multiple of 32, at most 128); `G` is filled in but for the ring (gemm_q4.cu).
int gemm_q4_long(const Q4Args& G, int bn, cudaStream_t stream) {
    QlArgs A{G, bn, (G.N + Q4_ROWS - 1) / Q4_ROWS, (G.T + bn - 1) / bn};
    constexpr int BARS = (2 * QL_STAGES_MAX + 2 * QL_NA + 2 * QL_ND + 2) * 8;
    A.g.stage_bytes = (bn * 256 + G.form.bytes + 1023) & ~1023;
    A.g.stages = (QL_SMEM - 1024 - QL_HAND - BARS) / A.g.stage_bytes;
    if (A.g.stages > QL_STAGES_MAX) A.g.stages = QL_STAGES_MAX;
    A.g.stages &= ~1;                                    // a stage belongs to one group of unpacking warps
    const long long items = (long long)A.m_tiles * A.t_tiles;
    const int blocks = items < tl_num_sms() ? (int)items : tl_num_sms();
    if (blocks < 1) return 1;
    CUtensorMap map;
    int e = load_encode();
    if (e || (e = q4_map(&map, G.x, G.T, G.K, G.ldx, bn, 64))) return e;
    if (G.form.zeros)
        return G.form.group == 128 ? ql_launch<128, true>(map, A, blocks, stream) : G.form.group == 64 ? ql_launch<64, true>(map, A, blocks, stream)
                                                                                                    : ql_launch<32, true>(map, A, blocks, stream);
    return G.form.group == 128 ? ql_launch<128, false>(map, A, blocks, stream) : G.form.group == 64 ? ql_launch<64, false>(map, A, blocks, stream)
                                                                                                 : ql_launch<32, false>(map, A, blocks, stream);
}
