// Products of few tokens with weights of 4 bits (q4.cuh, gemm_q4.cu): what a step of single tokens spends its time on.
// y[t, n] = sum over groups of scale * (whole-number sums of the tensor cores), as there.
//
// A block works on 128 rows of W over a range of K.  One warp brings packed weights, two blocks of 128 k at a time, and their tokens into a ring by
// bulk copies; eight warps, four for either of the two, unpack 32 rows each into the registers that mma.sync takes as its 16-row operand and
// multiply them there.  No weight goes through shared or tensor memory unpacked, and nobody waits for anyone but the copies: at 23 bytes a
// cycle and SM a block of 128 x 128 weights has to be through in about 370 cycles, and its hand-overs to and from tcgen05 (an arrival, a
// wait and a commit each) took longer.  The order of k within a product is free, so a lane takes eight k that follow one another from one word
// of codes and from one 16-byte piece of a token.
// What bounds it: latency with few warps.  No pipe is full (8 tokens, a cold launch: a scheduler issues in 49 % of the cycles, the ALU, which takes seven of the
// 11 instructions for eight values, is used in 43 %): a scheduler has four working warps, and between two instructions of one lie 8.1 cycles, of
// which it waits 1.8 for copies and loads, 1.1 for the instruction before, 1.0 for a pipe and 1.3 for its turn.  A block of 128 x 128 takes 440 cycles so, where
// memory needs 370; beside that whole tiles are dealt out (1,188 tiles on 296 places are four rounds and four tiles more), and every tile begins and ends anew.
// Measured in a CUDA graph on weights that are not in L2, 37,888 x 3,584 gated (70 MB): 1 token 16.8 us, 8 tokens 17.3, 16 tokens 21.0 (floor 10.7: 4.1
// of 6.5 TB/s); 152,064 x 3,584 with zeros, 8 tokens 71 us (44); 3,584 x 18,944, 8 tokens 13.7 us (5.4); 4,608 x 3,584, 1 token 5.6 us (1.3: half of
// it begins and ends a launch).
#include "q4.cuh"

namespace {

constexpr int GV_GROUPS = 2, GV_WORKERS = 4 * GV_GROUPS, GV_THREADS = 32 * (GV_WORKERS + 1);
constexpr int GV_X_ROW = GV_GROUPS * Q4_K * 2;            // bytes of a token in a stage
constexpr int GV_STAGES_MAX = 12, GV_SMEM_MOST = 112 * 1024;

__device__ __forceinline__ void gv_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT tiles of eight tokens
template <int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(GV_THREADS, 2)
gemv_q4_kernel(const __grid_constant__ CUtensorMap map_x, const Q4Args G) {
    constexpr int TOKENS = 8 * NT, X_BYTES = TOKENS * GV_X_ROW, GROUPS = Q4_K / GROUP;
    extern __shared__ __align__(128) unsigned char ring[];      // a stage: tokens, [TOKENS][GV_GROUPS * 128 k], then GV_GROUPS blocks of weights
    const int S = G.stages;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + (size_t)S * G.stage_bytes);
    uint64_t* empty = full + S;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + S);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, nz = gridDim.z, k0 = blockIdx.z * G.per, n_k = min(G.blocks, k0 + G.per) - k0;
    const int n_st = (n_k + GV_GROUPS - 1) / GV_GROUPS;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, GV_WORKERS); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    if (warp == GV_WORKERS) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            const unsigned char* src = G.w + ((size_t)tile * G.blocks + k0) * G.form.bytes;
            auto load_w = [&](int i, int s) {
                const uint32_t bytes = min(GV_GROUPS, n_k - i * GV_GROUPS) * G.form.bytes;
                mbar_expect_tx(full + s, X_BYTES + bytes);
                q4_bulk(smem_addr(ring + (size_t)s * G.stage_bytes) + X_BYTES, src + (size_t)i * GV_GROUPS * G.form.bytes, bytes, smem_addr(full + s));
            };
            auto load_x = [&](int i, int s) {
                tma_box(smem_addr(ring + (size_t)s * G.stage_bytes), &map_x, full + s, (k0 + i * GV_GROUPS) * Q4_K, 0);
            };
            if (!G.at_rest) grid_dependency_wait();
            for (int i = 0; i < min(n_st, S); ++i) load_w(i, i);
            if (G.at_rest) grid_dependency_wait();
            grid_dependency_trigger();
            for (int i = 0; i < min(n_st, S); ++i) load_x(i, i);
            for (int i = S, s = 0, turn = 0; i < n_st; ++i) {
                if (!mbar_wait(empty + s, turn & 1, abort_flag, G.status, 76)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == S) { s = 0; ++turn; }
            }
        }
    } else {
        const int g = lane >> 2, t = lane & 3, row0 = (warp & 3) * 32 + g, mine = warp >> 2;     // rows row0, + 8, + 16, + 24; its block of a stage
        const int last = (G.K + GROUP - 1) / GROUP - (k0 + n_k - 1) * GROUPS;            // groups of the last block that begin before K
        const uint32_t magic = q4_magic();
        float acc[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[m][j][c] = 0.f;
        grid_dependency_wait();                          // the output may still be read by the kernel in front
        for (int st = 0, s = 0, turn = 0; st < n_st; ++st) {
            const int i = st * GV_GROUPS + mine;
            if (i >= n_k || !mbar_wait(full + s, turn & 1, abort_flag, G.status, 77)) break;
            const unsigned char* x = ring + (size_t)s * G.stage_bytes + g * GV_X_ROW + mine * (Q4_K * 2) + t * 16;
            const unsigned char* block = ring + (size_t)s * G.stage_bytes + X_BYTES + mine * G.form.bytes;
            const unsigned char* w = block + row0 * 16 + t * 4;
            const unsigned char* scales = block + Q4_CODES;
            const unsigned char* zeros = scales + GROUPS * Q4_ROWS * (G.form.scale_f32 ? 4 : 2);
            const int gs = i + 1 < n_k ? GROUPS : last;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
                float sum[2][NT][4];                     // of two tiles of 16 rows
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) sum[0][j][c] = sum[1][j][c] = 0.f;
                __nv_bfloat162 zz[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) zz[m] = q4_zero(ZEROS ? zeros[gr * Q4_ROWS + row0 + 8 * m] : 8u);
#pragma unroll
                for (int p = gr * (GROUP / 32); p < (gr + 1) * (GROUP / 32); ++p) {
                    uint4 v[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) v[j] = *reinterpret_cast<const uint4*>(x + p * 64 + j * 8 * GV_X_ROW);
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        uint32_t a[4], b[4];             // rows row0 + 16 m and + 8, eight k each
                        q4_values(*reinterpret_cast<const uint32_t*>(w + (p * Q4_ROWS + 16 * m) * 16), magic, zz[2 * m], a);
                        q4_values(*reinterpret_cast<const uint32_t*>(w + (p * Q4_ROWS + 16 * m + 8) * 16), magic, zz[2 * m + 1], b);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            gv_mma(sum[m][j], a[0], b[0], a[1], b[1], v[j].x, v[j].y);
                            gv_mma(sum[m][j], a[2], b[2], a[3], b[3], v[j].z, v[j].w);
                        }
                    }
                }
                if (GROUPS > 1 && gr >= gs) continue;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const float lo = q4_scale(scales, gr * Q4_ROWS + row0 + 16 * m, G.form.scale_f32);
                    const float hi = q4_scale(scales, gr * Q4_ROWS + row0 + 16 * m + 8, G.form.scale_f32);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        acc[m][j][0] = fmaf(lo, sum[m][j][0], acc[m][j][0]);
                        acc[m][j][1] = fmaf(lo, sum[m][j][1], acc[m][j][1]);
                        acc[m][j][2] = fmaf(hi, sum[m][j][2], acc[m][j][2]);
                        acc[m][j][3] = fmaf(hi, sum[m][j][3], acc[m][j][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + s);
            if (++s == S) { s = 0; ++turn; }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * GV_WORKERS) : "memory");   // every copy has been waited for and read: the ring takes the sums, [group][token][row]
        float* red = reinterpret_cast<float*>(ring) + (warp >> 2) * TOKENS * Q4_ROWS;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) red[(8 * j + 2 * t + (c & 1)) * Q4_ROWS + row0 + 16 * m + 8 * (c >> 1)] = acc[m][j][c];
    }
    if (nz > 1) pair_cluster_sync(); else __syncthreads();
    if (warp < GV_WORKERS && !*abort_flag)
        q4_finish<GV_GROUPS, TOKENS>(G, reinterpret_cast<const float*>(ring), tile, 0, nz, blockIdx.z, threadIdx.x, 32 * GV_WORKERS);
    if (nz > 1) pair_cluster_sync();                     // nobody leaves while its shared memory is read
    if (*abort_flag) {                                   // copies in flight land before the shared memory is handed on
        const long long begin = clock64();
        while (clock64() - begin < 2000000LL) { }
    }
}

template <int NT, int GROUP, bool ZEROS>
int gv_launch(const CUtensorMap& map, Q4Args G, int tiles, int splits, cudaStream_t stream) {
    constexpr int BARS = 2 * GV_STAGES_MAX * 8 + 16, X_BYTES = 8 * NT * GV_X_ROW, SUMS = GV_GROUPS * 8 * NT * Q4_ROWS * 4;
    static bool raised[TL_MAX_DEVICES] = {};
    int e = tl_raise_smem(gemv_q4_kernel<NT, GROUP, ZEROS>, raised, GV_SMEM_MOST);
    if (e) return e;
    G.stage_bytes = (X_BYTES + GV_GROUPS * G.form.bytes + 127) & ~127;
    const int n_st = (G.per + GV_GROUPS - 1) / GV_GROUPS;
    G.stages = (GV_SMEM_MOST - BARS) / G.stage_bytes;
    if (G.stages > GV_STAGES_MAX) G.stages = GV_STAGES_MAX;
    if (G.stages > n_st) G.stages = n_st;
    static_assert(X_BYTES + GV_GROUPS * Q4_CODES >= SUMS, "a stage takes the sums");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, 1, splits);
    cfg.blockDim = dim3(GV_THREADS);
    cfg.dynamicSmemBytes = (size_t)G.stages * G.stage_bytes + BARS;
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
    const cudaError_t ce = cudaLaunchKernelEx(&cfg, gemv_q4_kernel<NT, GROUP, ZEROS>, map, G);
    return ce != cudaSuccess ? (int)ce : tl_launch_status();
}

template <int NT>
int gv_launch_form(const CUtensorMap& map, const Q4Args& G, int tiles, int splits, cudaStream_t stream) {
    if (G.form.zeros)
        return G.form.group == 128 ? gv_launch<NT, 128, true>(map, G, tiles, splits, stream) :
               G.form.group == 64 ? gv_launch<NT, 64, true>(map, G, tiles, splits, stream) : gv_launch<NT, 32, true>(map, G, tiles, splits, stream);
    return G.form.group == 128 ? gv_launch<NT, 128, false>(map, G, tiles, splits, stream) :
           G.form.group == 64 ? gv_launch<NT, 64, false>(map, G, tiles, splits, stream) : gv_launch<NT, 32, false>(map, G, tiles, splits, stream);
}

}  // namespace

// Ranges of K a tile: the fewest blocks of k, one behind the other, on the SM that has most.  An SM gets through a block of k in the same time
// whether one thread block works on it or two do, so with more of them than SMs every SM counts twice; clusters of many blocks leave some SMs
// of a GPC empty (of 148 SMs about 132 get a block in clusters of two or three, 100 in larger ones, where two blocks go to one SM first).  Measured
// at 1, 2 .. 8 ranges, us:  28 tiles x 148 blocks 45 24 17.5 17 17 16 14.7 13.6;  40 x 108: 33 18 13.2 16 14.5 13.3 17 16;  36 x 28: 9.7 6.2
// 5.6 6.0 5.4 6.2 6.2 6.2;  86 x 16: 6.4 7.2 7.8 6.9 7.0 9.5 9.3 9.1;  296 x 28: 17 21 27 29 27 29 32 32.
int gemv_q4_ranges(int tiles, int blocks, int sms) {
    int best = 1;
    long long least = 0;
    for (int s = 1; s <= 8 && s <= blocks; ++s) {
        const int per = (blocks + s - 1) / s;
        if ((blocks + per - 1) / per != s) continue;     // a range would be empty
        const long long total = (long long)tiles * s, alone = s == 1 ? sms : s <= 3 ? sms * 9 / 10 : sms * 2 / 3;
        const long long both = s == 1 ? 2 * sms : s <= 6 ? sms * 9 / 5 : sms * 8 / 5;
        const long long cost = (total <= alone ? 1 : 2 * ((total + both - 1) / both)) * (per + 4);      // a block begins and ends in the time of four blocks of k
        if (s == 1 || cost < least) { best = s; least = cost; }
    }
    return best;
}

// The product for G.T <= Q4_FEW tokens; `G` is filled in but for the ranges of K and the ring (gemm_q4.cu).
int gemv_q4(Q4Args G, int splits, cudaStream_t stream) {
    const int tiles = (G.N + Q4_ROWS - 1) / Q4_ROWS;
    G.per = (G.blocks + splits - 1) / splits;
    CUtensorMap map;
    int e = load_encode();
    if (e || (e = q4_map(&map, G.x, G.T, G.K, G.ldx, G.T <= 8 ? 8 : 16, GV_X_ROW / 2))) return e;
    return G.T <= 8 ? gv_launch_form<1>(map, G, tiles, splits, stream) : gv_launch_form<2>(map, G, tiles, splits, stream);
}
