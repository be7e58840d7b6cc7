// Matrices into weights of 4 bits (q4.cuh) and back.
//
// Of a group's values, real numbers here, with (.) rounded to the scale's type by way of float:
//     without zeros   scale = (max |w| / 7),                          code = 8 + clamp(rint(w / scale), -7, 7)
//     with zeros      lo = min(0, min w), hi = max(0, max w), scale = ((hi - lo) / 15),
//                     zero = clamp(rint(-lo / scale), 0, 15),         code = clamp(rint(w / scale) + zero, 0, 15)
// rint: to the nearest whole number, ties to the even one.  A scale of zero leaves codes that stand for zeros; a group that holds a value that
// is no number or infinite has a scale that is no number, so that whoever reads it sees it.
//
// Both kernels move a matrix once and are bound by that: a block of threads takes 128 rows and 128 k, 16 lanes a row, eight k a lane (one word
// of codes).  Quotients are decided exactly without 64-bit arithmetic, see q4_rint.
#include "q4.cuh"

namespace {

constexpr int QQ_THREADS = 256;

// The nearest whole number to w / s, ties to even, for 0 < s and |w| <= 32 s.  The quotient by the reciprocal is off by less than 2^-18, so
// its nearest whole number c is the right one or its neighbour; w - c s has no more bits than a float, and its half-way mark is s / 2.
// Scales below 2^-100, whose reciprocals and halves may be none, divide in 64 bits.
__device__ __forceinline__ float q4_rint(float w, float s, float inv) {
    if (s < 7.888609e-31f) return (float)rint((double)w / (double)s);
    float c = rintf(w * inv);
    const float left = fmaf(-s, c, w), half = 0.5f * s;
    const bool odd = ((int)c) & 1;
    if (fabsf(left) > half || (odd && fabsf(left) == half)) c += left > 0.f ? 1.f : -1.f;
    return c;
}

// (hi - lo) / 15 rounded to float: the difference is exact in float more often than not, and an exact difference's quotient is rounded once
// either way (fifteenths have no long runs of equal bits, so rounding to 64 bits in between changes nothing).
__device__ __forceinline__ float q4_fifteenth(float lo, float hi) {
    const float d = hi - lo, back = d + lo;
    if (isfinite(d) && back == hi && hi - d == lo) return d / 15.0f;
    return (float)(((double)hi - (double)lo) / 15.0);
}

template <typename T>
__global__ void __launch_bounds__(QQ_THREADS)
quantize_q4_kernel(const T* __restrict__ w, unsigned char* __restrict__ out, int N, int K, int blocks, const Q4Form form) {
    __shared__ __align__(16) unsigned char tile[Q4_CODES + 4 * Q4_ROWS * 4 + 4 * Q4_ROWS];
    grid_dependency_wait();
    const int kb = blockIdx.x, row0 = blockIdx.y * Q4_ROWS;
    const int lane = threadIdx.x & 31, m = lane & 15, k = kb * Q4_K + 8 * m;
    const int lanes = form.group / 8, scales_at = Q4_CODES, zeros_at = scales_at + form.groups * Q4_ROWS * (form.scale_f32 ? 4 : 2);
    for (int r = (threadIdx.x >> 5) * 2 + (lane >> 4); r < Q4_ROWS; r += QQ_THREADS / 16) {
        float v[8] = {};
        if (row0 + r < N && k < K) {                     // K % 8 == 0
            const T* src = w + (size_t)(row0 + r) * K + k;
            if (sizeof(T) == 2) {
                const uint4 q = *reinterpret_cast<const uint4*>(src);
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(u[j] << 16); v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u); }
            } else {
                const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            }
        }
        float lo = 0.f, hi = 0.f;
        bool odd = false;                                // a value that is no number, or infinite
#pragma unroll
        for (int j = 0; j < 8; ++j) { lo = fminf(lo, v[j]); hi = fmaxf(hi, v[j]); odd |= !isfinite(v[j]); }
        for (int o = 1; o < lanes; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            odd |= __shfl_xor_sync(0xffffffffu, (int)odd, o) != 0;
        }
        float s = odd ? 0.f : form.zeros ? q4_fifteenth(lo, hi) : fmaxf(-lo, hi) / 7.0f;
        if (!form.scale_f32) s = __bfloat162float(__float2bfloat16_rn(s));
        const float inv = 1.0f / s;                      // not used where it is none
        const float zero = !form.zeros ? 8.f : s > 0.f ? fminf(fmaxf(q4_rint(-lo, s, inv), 0.f), 15.f) : 0.f;
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float c = s > 0.f ? q4_rint(v[j], s, inv) : 0.f;
            c = form.zeros ? fminf(fmaxf(c + zero, 0.f), 15.f) : fminf(fmaxf(c, -7.f), 7.f) + 8.f;
            word |= (uint32_t)c << (16 * (j & 1) + 4 * ((j >> 1) & 1) + 8 * (j >> 2));
        }
        reinterpret_cast<uint32_t*>(tile)[((m >> 2) * Q4_ROWS + r) * 4 + (m & 3)] = word;
        if (m % lanes == 0) {
            const int at = (m / lanes) * Q4_ROWS + r;
            if (odd) s = __int_as_float(0x7fc00000);
            if (form.scale_f32) reinterpret_cast<float*>(tile + scales_at)[at] = s;
            else reinterpret_cast<bf16*>(tile + scales_at)[at] = __float2bfloat16_rn(s);
            if (form.zeros) tile[zeros_at + at] = (unsigned char)zero;
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(out + ((size_t)blockIdx.y * blocks + kb) * form.bytes);
    for (int i = threadIdx.x; i < form.bytes / 16; i += QQ_THREADS) dst[i] = reinterpret_cast<const uint4*>(tile)[i];
}

__device__ __forceinline__ void q4_store8(float* dst, const float (&v)[8]) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void q4_store8(bf16* dst, const float (&v)[8]) {
    uint4 q;
    uint32_t* u = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<uint4*>(dst) = q;
}

// The values in float, rounded once more where T is bfloat16.
template <typename T>
__global__ void __launch_bounds__(QQ_THREADS)
dequantize_q4_kernel(const unsigned char* __restrict__ w, T* __restrict__ out, int N, int K, int blocks, const Q4Form form) {
    grid_dependency_wait();
    const int kb = blockIdx.x, row0 = blockIdx.y * Q4_ROWS;
    const unsigned char* src = w + ((size_t)blockIdx.y * blocks + kb) * form.bytes;
    const unsigned char* scales = src + Q4_CODES;
    const unsigned char* zeros = scales + form.groups * Q4_ROWS * (form.scale_f32 ? 4 : 2);
    const int lane = threadIdx.x & 31, m = lane & 15, k = kb * Q4_K + 8 * m;
    if (k >= K) return;
    for (int r = (threadIdx.x >> 5) * 2 + (lane >> 4); r < Q4_ROWS && row0 + r < N; r += QQ_THREADS / 16) {
        const uint32_t word = reinterpret_cast<const uint32_t*>(src)[((m >> 2) * Q4_ROWS + r) * 4 + (m & 3)];
        const int at = (8 * m / form.group) * Q4_ROWS + r;
        const float s = q4_scale(scales, at, form.scale_f32);
        const int zero = form.zeros ? zeros[at] : 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s * (float)((int)((word >> (16 * (j & 1) + 4 * ((j >> 1) & 1) + 8 * (j >> 2))) & 15u) - zero);
        q4_store8(out + (size_t)(row0 + r) * K + k, v);
    }
}

int q4_grid(dim3* grid, int N, int K) {
    const int tiles = (N + Q4_ROWS - 1) / Q4_ROWS;
    *grid = dim3((K + Q4_K - 1) / Q4_K, tiles);
    return tiles <= 65535;
}

}  // namespace

// Weights of 4 bits [ceil(N / 128)][ceil(K / 128)][block] from w [N, K], bfloat16 or float; K % 8 == 0.  `form_bits`: k a group, from bit 8 on: scales are float, there are zeros.
TL_EXPORT int tl_quantize_q4(const void* w, int w_f32, void* out, int N, int K, int form_bits, cudaStream_t stream) {
    Q4Form form;
    dim3 grid;
    if (N < 1 || K < 1 || (K & 7) || form_bits < 0 || form_bits >> 10 || !q4_form(&form, form_bits & 255, form_bits >> 8 & 1, form_bits >> 9 & 1) || !q4_grid(&grid, N, K) || ((uintptr_t)w & 15) || ((uintptr_t)out & 15)) return 1;
    return w_f32 ? launch_after_wait(quantize_q4_kernel<float>, grid, dim3(QQ_THREADS), 0, stream, (const float*)w, (unsigned char*)out, N, K, (int)grid.x, form)
                 : launch_after_wait(quantize_q4_kernel<bf16>, grid, dim3(QQ_THREADS), 0, stream, (const bf16*)w, (unsigned char*)out, N, K, (int)grid.x, form);
}

// The values that weights of 4 bits stand for, [N, K] bfloat16 or float.
TL_EXPORT int tl_dequantize_q4(const void* w, void* out, int out_f32, int N, int K, int form_bits, cudaStream_t stream) {
    Q4Form form;
    dim3 grid;
    if (N < 1 || K < 1 || (K & 7) || form_bits < 0 || form_bits >> 10 || !q4_form(&form, form_bits & 255, form_bits >> 8 & 1, form_bits >> 9 & 1) || !q4_grid(&grid, N, K) || ((uintptr_t)w & 15) || ((uintptr_t)out & 15)) return 1;
    return out_f32 ? launch_after_wait(dequantize_q4_kernel<float>, grid, dim3(QQ_THREADS), 0, stream, (const unsigned char*)w, (float*)out, N, K, (int)grid.x, form)
                   : launch_after_wait(dequantize_q4_kernel<bf16>, grid, dim3(QQ_THREADS), 0, stream, (const unsigned char*)w, (bf16*)out, N, K, (int)grid.x, form);
}
