// Products of many tokens with weights of 4 bits (q4.cuh): the sums of gemm_q4.cu on pairs of thread blocks.
//
// Two blocks on neighbouring SMs work on 256 rows of W and BN tokens (32 to 192): tcgen05.mma.cta_group::2, W in tensor memory on the 256-row
// side, the tokens in shared memory, half of them in either block.  A block unpacks its own 128 rows of a block of 128 k into its tensor memory
// (four warps, a row a thread); the leader issues eight products of 16 k; eight warps of each block scale a finished group's sums and add them
// to the outputs', which they hold in registers, 96 a thread at most.  Tensor memory: two blocks of unpacked weights (64 columns each) and two
// groups' sums (2 x 192): all of it.
// The pairs are persistent; the ring of copies and both kinds of buffers run on from one tile to the next, so that nothing starts anew.
// What bounds it: eight products of 256 x BN x 16 take 4 BN cycles, and a round of hand-overs through the block (copies, unpacking, products, sums,
// each about 200 cycles of waiting and arriving beside its work) takes as long as about 160 tokens; wide tiles hide it.
#include "q4.cuh"

namespace {

constexpr int QP_THREADS = 512;                          // warp 0: copies, 1: tensor memory + products, 4..7: unpacking, 8..15: sums
// registers a thread of those three groups of warps: 48 + 96 + 2 x 184 of the 4 x 128 that the block is launched with
constexpr int QP_REGS_COPY = 48, QP_REGS_UNPACK = 96, QP_REGS_SUM = 184;
static_assert(QP_REGS_COPY + QP_REGS_UNPACK + 2 * QP_REGS_SUM <= 512, "a larger share would be waited for without end");
constexpr int QP_MOST = 192, QP_CW = QP_MOST / 2;        // tokens of a pair, of a summing warp
constexpr int QP_NA = 4, QP_ND = 2, QP_D_COL = QP_NA * 32;      // halves of unpacked blocks (64 k, 32 columns), groups' sums
constexpr int QP_STAGES_MAX = 12, QP_SMEM = 226 * 1024, QP_HAND = 2 * 2 * 16 * 64 * 4;      // gates and what they weigh change places: [2][half][16][64]
static_assert(QP_D_COL + QP_ND * QP_MOST <= 512, "tensor memory");

struct QpArgs { Q4Args g; int bn, m_tiles, t_tiles; };

__device__ __forceinline__ void qp_mma(uint32_t acc, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(acc), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}

template <int GROUP, bool ZEROS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(QP_THREADS, 1)
gemm_q4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const QpArgs A) {
    constexpr int NA = QP_NA, ND = QP_ND, GROUPS = Q4_K / GROUP;
    const Q4Args& G = A.g;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);      // a stage: half of the tokens, packed weights
    const int S = G.stages, BN = A.bn, x_half = (BN / 2) * 128, x_bytes = 2 * x_half;
    float* hand = reinterpret_cast<float*>(ring + (size_t)S * G.stage_bytes);
    uint64_t* w_full = reinterpret_cast<uint64_t*>(hand + QP_HAND / 4);
    uint64_t* x_full = w_full + S;                       // the leader's: both blocks' tokens
    uint64_t* empty = x_full + S;                        // 4 unpacking warps, 8 summing warps
    uint64_t* a_full = empty + S;                        // [NA] the leader's: 4 unpacking warps of both blocks
    uint64_t* a_empty = a_full + NA;                     // [NA] the products
    uint64_t* d_full = a_empty + NA;                     // [ND] the products
    uint64_t* d_empty = d_full + ND;                     // [ND] the leader's: 8 summing warps of both blocks
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + ND);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = pair_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, items = A.m_tiles * A.t_tiles, n_k = G.blocks;
    const int last = (G.K + GROUP - 1) / GROUP - (n_k - 1) * GROUPS;                         // groups of the last block that begin before K

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(w_full + s, 1); mbar_init(x_full + s, 1); mbar_init(empty + s, 12); }
        for (int b = 0; b < NA; ++b) { mbar_init(a_full + b, 8); mbar_init(a_empty + b, 1); }
        for (int b = 0; b < ND; ++b) { mbar_init(d_full + b, 1); mbar_init(d_empty + b, 16); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) pair_tmem_alloc(tmem_slot);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    pair_cluster_sync();                                 // both blocks' barriers exist before anyone signals them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);

    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(QP_REGS_COPY));
      if (warp == 0) {
        // ---------------------------------------------------------------- copies (both blocks)
        const uint32_t one = pair_elect(), lead = rank == 0 ? one : 0u;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        const int row_tiles = (G.N + Q4_ROWS - 1) / Q4_ROWS;
        auto load_w = [&](int item, int c, int s) {      // (the second block of the last pair may have no rows: it reads its peer's)
            const int tile = min(2 * (item / A.t_tiles) + (int)rank, row_tiles - 1);
            if (one) {
                mbar_expect_tx(w_full + s, G.form.bytes);
                q4_bulk(smem_addr(ring + (size_t)s * G.stage_bytes) + x_bytes, G.w + ((size_t)tile * n_k + c) * G.form.bytes, G.form.bytes, w_full + s);
            }
        };
        auto load_x = [&](int item, int c, int s) {
            const int t0 = (item % A.t_tiles) * BN + (int)rank * (BN / 2);
            const uint32_t dst = smem_addr(ring + (size_t)s * G.stage_bytes), bar = pair_peer(smem_addr(x_full + s), 0);
            pair_expect(x_full + s, 2 * x_bytes, lead);
            pair_load(dst, &map_x, bar, c * Q4_K, t0, one);
            pair_load(dst + x_half, &map_x, bar, c * Q4_K + 64, t0, one);
        };
        const int ahead = min(S, n_k);
        if (!G.at_rest) grid_dependency_wait();
        for (int c = 0; c < ahead; ++c) load_w(pair, c, c);
        if (G.at_rest) grid_dependency_wait();
        grid_dependency_trigger();
        for (int c = 0; c < ahead; ++c) load_x(pair, c, c);
        int s = 0, turn = 0, it = 0;
        bool ok = true;
        for (int item = pair; item < items && ok; item += pairs) {
            for (int c = 0; c < n_k; ++c, ++it) {
                if (it >= ahead) {
                    if (it >= S && !mbar_wait(empty + s, (turn - 1) & 1, abort_flag, G.status, 81)) { ok = false; break; }
                    load_w(item, c, s);
                    load_x(item, c, s);
                }
                if (++s == S) { s = 0; ++turn; }
            }
        }
      } else if (warp == 1 && rank == 0) {
        // ---------------------------------------------------------------- products (the leader)
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((2 * Q4_ROWS) >> 4) << 24);
            const uint32_t one = pair_elect();
            grid_dependency_wait();                      // the bounded waits start counting once the tokens can land
            int d = 0, s = 0, turn = 0, n = 0;           // groups, stage and its round, halves so far
            bool ok = true, x_there = false, a_there = false, d_there = false;
            for (int item = pair; item < items && ok; item += pairs) {
                for (int c = 0; c < n_k && ok; ++c) {
                    const int gs = GROUPS == 1 || c + 1 < n_k ? GROUPS : last;
                    ok = x_there || mbar_wait(x_full + s, turn & 1, abort_flag, G.status, 82);
                    const uint64_t x = desc_kmajor(smem_addr(ring + (size_t)s * G.stage_bytes));
                    if (++s == S) { s = 0; ++turn; }
#pragma unroll
                    for (int h = 0; h < 2; ++h, ++n) {
                        const int b = n % NA;
                        ok = ok && (a_there || mbar_wait(a_full + b, (n / NA) & 1, abort_flag, G.status, 82));
                        if (!ok) break;
                        // whether the next ones are there is asked now: an answer takes 80 cycles, and these products longer
                        a_there = q4_peek(a_full + (n + 1) % NA, ((n + 1) / NA) & 1);
                        if (h == 1) x_there = q4_peek(x_full + s, turn & 1);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t a = tmem + b * 32;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {    // 16 k: 8 columns of weights, 32 bytes of tokens (2 of a descriptor's units of 16)
                            constexpr int STEPS = GROUP / 16;
                            const int at = h * 4 + k, g = at / STEPS, e = d % ND;
                            if (g >= gs) continue;
                            if (at % STEPS == 0) {
                                if (d >= ND && !d_there) ok = mbar_wait(d_empty + e, (d / ND - 1) & 1, abort_flag, G.status, 83);
                                if (!ok) break;
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                                d_there = d + 1 >= ND && q4_peek(d_empty + (d + 1) % ND, ((d + 1) / ND - 1) & 1);
                            }
                            qp_mma(tmem + QP_D_COL + e * QP_MOST, a + k * 8, x + h * (x_half / 16) + k * 2, idesc, at % STEPS > 0, one);
                            if (at % STEPS == STEPS - 1) { pair_commit(d_full + e, one); ++d; }
                        }
                        if (ok) pair_commit(a_empty + b, one);
                    }
                }
            }
      }
    } else if (warp < 8) {
        // ---------------------------------------------------------------- unpacking
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(QP_REGS_UNPACK));
        const int row = quarter * 32 + lane, zeros_at = Q4_CODES + GROUPS * Q4_ROWS * (G.form.scale_f32 ? 4 : 2);
        const uint32_t magic = q4_magic();
        if (!G.at_rest) grid_dependency_wait();
        int s = 0, turn = 0, n = 0;
        bool ok = true, w_there = false, a_there = false;
        for (int item = pair; item < items && ok; item += pairs) {
            for (int c = 0; c < n_k && ok; ++c) {
                if (!w_there && !mbar_wait(w_full + s, turn & 1, abort_flag, G.status, 84)) { ok = false; break; }
                const unsigned char* st = ring + (size_t)s * G.stage_bytes + x_bytes;
                uint64_t* done = empty + s;
                uint4 q[4];
                uint32_t z[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    q[j] = *reinterpret_cast<const uint4*>(st + (j * Q4_ROWS + row) * 16);
                    z[j] = ZEROS ? st[zeros_at + (j * 32 / GROUP) * Q4_ROWS + row] : 8u;
                }
                if (++s == S) { s = 0; ++turn; }
#pragma unroll
                for (int half = 0; half < 2; ++half, ++n) {
                    const int b = n % NA;
                    if (n >= NA && !a_there && !mbar_wait(a_empty + b, (n / NA - 1) & 1, abort_flag, G.status, 84)) { ok = false; break; }
                    a_there = n + 1 >= NA && q4_peek(a_empty + (n + 1) % NA, ((n + 1) / NA - 1) & 1);
                    if (half == 1) w_there = q4_peek(w_full + s, turn & 1);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
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
                    q4_st32(lanes + b * 32, v);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        pair_arrive(pair_peer(smem_addr(a_full + b), 0));
                        if (half == 1) mbar_arrive(done);
                    }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- sums: 32 rows and half of the tokens a warp
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(QP_REGS_SUM));
        const int row = quarter * 32 + lane, half = (warp - 8) >> 2, cw = BN / 2;
        grid_dependency_wait();                          // the output may still be read by the kernel in front
        int s = 0, turn = 0, d = 0;
        bool ok = true, w_there = false, d_there = false;
        for (int item = pair; item < items && ok; item += pairs) {
            float acc[QP_CW];
#pragma unroll
            for (int c = 0; c < QP_CW; ++c) acc[c] = 0.f;
            for (int c = 0; c < n_k && ok; ++c) {
                if (!w_there && !mbar_wait(w_full + s, turn & 1, abort_flag, G.status, 85)) { ok = false; break; }
                const unsigned char* scales = ring + (size_t)s * G.stage_bytes + x_bytes + Q4_CODES;
                uint64_t* done = empty + s;
                const int gs = GROUPS == 1 || c + 1 < n_k ? GROUPS : last;
                float sc[GROUPS];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) sc[g] = g < gs ? q4_scale(scales, g * Q4_ROWS + row, G.form.scale_f32) : 0.f;
                if (++s == S) { s = 0; ++turn; }
                __syncwarp();
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    if (g >= gs) break;
                    const int e = d % ND;
                    if (!d_there && !mbar_wait(d_full + e, (d / ND) & 1, abort_flag, G.status, 85)) { ok = false; break; }
                    ++d;
                    if (g == gs - 1) {
                        if (lane == 0) mbar_arrive(done);      // the block's products are done
                        w_there = q4_peek(w_full + s, turn & 1);
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = lanes + QP_D_COL + e * QP_MOST + half * cw;
#pragma unroll
                    for (int c0 = 0; c0 < QP_CW; c0 += 16) {
                        if (c0 >= cw) break;
                        float r[16];
                        q4_ld16(at + c0, r);
                        tmem_ld_wait();
                        if (c0 + 16 >= cw) {             // the last of them are in registers
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) pair_arrive(pair_peer(smem_addr(d_empty + e), 0));
                            d_there = q4_peek(d_full + d % ND, (d / ND) & 1);
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 2) q4_fma2(sc[g], r[j], r[j + 1], acc[c0 + j], acc[c0 + j + 1]);
                    }
                }
            }
            if (!ok) break;
            const int tile = 2 * (item / A.t_tiles) + (int)rank, t0 = (item % A.t_tiles) * BN + half * cw;
            if (!G.gate) {
                const int n = tile * Q4_ROWS + row;
                if (n < G.N) {
                    const size_t base = (size_t)t0 * G.ldo + n;
#pragma unroll
                    for (int c = 0; c < QP_CW; ++c)
                        if (c < cw && t0 + c < G.T) q4_store(G, base + (size_t)c * G.ldo, acc[c]);
                }
            } else {
                // Gates are rows 0..63 of a tile and lie in other warps than what they weigh: of 16 tokens at a time the one side hands over its
                // values of the first eight, the other of the second, and each finishes eight.
                const bool up = quarter >= 2;
                const int f = (quarter & 1) * 32 + lane, n = tile * 64 + f;
#pragma unroll
                for (int c0 = 0; c0 < QP_CW; c0 += 16) {
                    if (c0 >= cw) break;
                    float* h = hand + (((c0 >> 4) & 1) * 2 + half) * 16 * 64;
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[(up ? j : 8 + j) * 64 + f] = up ? acc[c0 + j] : acc[c0 + 8 + j];
                    if (half) asm volatile("bar.sync 2, 128;" ::: "memory"); else asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int t = t0 + c0 + (up ? 8 : 0) + j;
                        const float mine = up ? acc[c0 + 8 + j] : acc[c0 + j], other = h[((up ? 8 : 0) + j) * 64 + f];
                        const float y = q4_gate(up ? other : mine, up ? mine : other, G.gate, G.limit, G.alpha);
                        if (n < G.N / 2 && t < G.T) q4_store(G, (size_t)t * G.ldo + n, y);
                    }
                }
            }
        }
    }
    // -------------------------------------------------------------------- teardown
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_flag) {                                   // copies in flight land before the shared memory is handed on
        const long long begin = clock64();
        while (clock64() - begin < 2000000LL) { }
    }
    pair_cluster_sync();
    if (warp == 1) pair_tmem_free(tmem);
}

template <int GROUP, bool ZEROS>
int qp_launch(const CUtensorMap& map, const QpArgs& A, int pairs, cudaStream_t stream) {
    static bool raised[TL_MAX_DEVICES] = {};
    const int e = tl_raise_smem(gemm_q4_pair_kernel<GROUP, ZEROS>, raised, QP_SMEM);
    if (e) return e;
    return launch_after_wait(gemm_q4_pair_kernel<GROUP, ZEROS>, dim3(2 * pairs), dim3(QP_THREADS), QP_SMEM, stream, map, A);
}

}  // namespace

// The product of G.T tokens in tiles of `bn` (a multiple of 32, at most 192); `G` is filled in but for the ring (gemm_q4.cu).
int gemm_q4_pair(const Q4Args& G, int bn, cudaStream_t stream) {
    QpArgs A{G, bn, (G.N + 2 * Q4_ROWS - 1) / (2 * Q4_ROWS), (G.T + bn - 1) / bn};
    constexpr int BARS = (3 * QP_STAGES_MAX + 2 * QP_NA + 2 * QP_ND) * 8 + 16;
    A.g.stage_bytes = (bn * 128 + G.form.bytes + 1023) & ~1023;
    A.g.stages = (QP_SMEM - 1024 - QP_HAND - BARS) / A.g.stage_bytes;
    if (A.g.stages > QP_STAGES_MAX) A.g.stages = QP_STAGES_MAX;
    const long long items = (long long)A.m_tiles * A.t_tiles;
    const int room = tl_num_sms() / 2, pairs = items < room ? (int)items : room;
    if (pairs < 1) return 1;
    CUtensorMap map;
    int e = load_encode();
    if (e || (e = q4_map(&map, G.x, G.T, G.K, G.ldx, bn / 2, 64))) return e;
    if (G.form.zeros)
        return G.form.group == 128 ? qp_launch<128, true>(map, A, pairs, stream) : G.form.group == 64 ? qp_launch<64, true>(map, A, pairs, stream)
                                                                                                  : qp_launch<32, true>(map, A, pairs, stream);
    return G.form.group == 128 ? qp_launch<128, false>(map, A, pairs, stream) : G.form.group == 64 ? qp_launch<64, false>(map, A, pairs, stream)
                                                                                               : qp_launch<32, false>(map, A, pairs, stream);
}
