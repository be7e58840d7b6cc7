// Matrices into weights of 4 bits (q4.cuh) and back.
//
// Of a group's values, real numbers here, with (.) rounded to the scale's type by way of float:
//     without zeros   scale = (max |w| / 7),                          code = 8 + clamp(rint(w / scale), -7, 7)
//     with zeros      lo = min(0, min w), hi = max(0, max w), scale = ((hi - lo) / 15),
//                     zero = clamp(rint(-lo / scale), 0, 15),         code = clamp(rint(w / scale) + zero, 0, 15)
// rint: to the nearest whole number, ties to the even one.  A scale of zero leaves codes that stand for zeros; a group that holds a value that
// is no number or infinite has a scale that is no number, so that whoever reads it sees it.
//
// Both kernels move a matrix once: a block of threads takes 128 rows and 128 k, 16 lanes a row, eight k a lane (one word of codes).  Reading back is
// bound by that; making codes from bfloat16 by its instructions, 17 a value, although quotients are decided exactly without 64-bit arithmetic
// (q4_round).  Measured, 37,888 x 3,584 in groups of 128: codes from bfloat16 86 us (floor 52), from float 95 (94); values in bfloat16 54 us
// (52), in float 98 (94).
#include "q4.cuh"

namespace {

constexpr int QQ_THREADS = 256;                          // of a block that reads back

// The nearest whole number to w / s, ties to even, as the last bits of a float: added to 1.5 2^23, a value is rounded to a whole number.  For
// 2^-100 <= s and |w| <= 16 s.  The quotient by the reciprocal is off by less than 2^-18, so this is the nearest number to w / s or, around
// a half-way mark, its neighbour: w - c s has no more bits than a float, and where it is s / 2 or more, `q4_mend` takes another look.
constexpr float Q4_MAGIC = 12582912.0f;
__device__ __forceinline__ float q4_round(float w, float s, float inv, float& far) {
    const float t = __fmaf_rn(w, inv, Q4_MAGIC);
    far = fmaxf(far, fabsf(__fmaf_rn(-s, t - Q4_MAGIC, w)));
    return t;
}
// two at a time, in this architecture's pairs of float operations
__device__ __forceinline__ void q4_round2(float w0, float w1, float s, float inv, float& t0, float& t1, float& far) {
    float l0, l1;
    asm("{\n\t.reg .b64 w, i, m, t, n, c, l;\n\t"
        "mov.b64 w, {%4, %5};\n\tmov.b64 i, {%6, %6};\n\tmov.b64 m, {%8, %8};\n\tmov.b64 n, {%9, %9};\n\t"
        "fma.rn.f32x2 t, w, i, m;\n\t"
        "add.rn.f32x2 c, t, n;\n\t"
        "mov.b64 i, {%7, %7};\n\t"
        "fma.rn.f32x2 l, i, c, w;\n\t"
        "mov.b64 {%0, %1}, t;\n\tmov.b64 {%2, %3}, l;\n\t}"
        : "=f"(t0), "=f"(t1), "=f"(l0), "=f"(l1) : "f"(w0), "f"(w1), "f"(inv), "f"(-s), "f"(Q4_MAGIC), "f"(-Q4_MAGIC));
    far = fmaxf(far, fmaxf(fabsf(l0), fabsf(l1)));
}
__device__ __forceinline__ float q4_mend(float w, float s, float t) {
    const float left = __fmaf_rn(-s, t - Q4_MAGIC, w), far = fabsf(left), half = 0.5f * s;
    return far > half || (far == half && (__float_as_int(t) & 1)) ? t + (left > 0.f ? 1.f : -1.f) : t;
}
// smaller scales, whose reciprocals and halves may be none
__device__ __forceinline__ int q4_rint_small(float w, float s) { return (int)rint((double)w / (double)s); }
constexpr float Q4_SMALL = 7.888609e-31f;                // 2^-100

__device__ __forceinline__ float q4_max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float q4_min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// (hi - lo) / 15 rounded to float: the difference is exact in float more often than not, and an exact difference's quotient is rounded once
// either way (fifteenths have no long runs of equal bits, so rounding to 64 bits in between changes nothing).
__device__ __forceinline__ float q4_fifteenth(float lo, float hi) {
    const float d = hi - lo, back = d + lo;
    if (isfinite(d) && back == hi && hi - d == lo) return d / 15.0f;
    return (float)(((double)hi - (double)lo) / 15.0);
}

// eight values as they lie in memory
__device__ __forceinline__ void q4_widen(const uint4 (&q)[1], float (&v)[8]) {
    const uint32_t u[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(u[j] << 16); v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u); }
}
__device__ __forceinline__ void q4_widen(const uint4 (&q)[2], float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        v[4 * j] = __uint_as_float(q[j].x); v[4 * j + 1] = __uint_as_float(q[j].y);
        v[4 * j + 2] = __uint_as_float(q[j].z); v[4 * j + 3] = __uint_as_float(q[j].w);
    }
}

// A thread's rows are asked for at once (one behind the other they were 1.3 times the time): eight of bfloat16, four of float, whose
// registers leave room for fewer threads (four rows of bfloat16: 4 % slower, eight of float: 30 %).  The group is the kernel's own, so that the
// lanes' exchange is a straight run of instructions (a loop over them: 113 us instead of 86).
template <typename T> constexpr int QQ_MAKE = sizeof(T) == 2 ? 256 : 512;
template <typename T, bool ZEROS, int GROUP>
__global__ void __launch_bounds__(QQ_MAKE<T>)
quantize_q4_kernel(const T* __restrict__ w, unsigned char* __restrict__ out, int N, int K, int blocks, const Q4Form form) {
    constexpr int PIECES = sizeof(T) / 2, THREADS = QQ_MAKE<T>, ROUNDS = Q4_ROWS / (THREADS / 16);
    __shared__ __align__(16) unsigned char tile[Q4_CODES + 4 * Q4_ROWS * 4 + 4 * Q4_ROWS];
    grid_dependency_wait();
    const int kb = blockIdx.x, row0 = blockIdx.y * Q4_ROWS;
    const int lane = threadIdx.x & 31, m = lane & 15, k = kb * Q4_K + 8 * m, r0 = (threadIdx.x >> 5) * 2 + (lane >> 4);
    constexpr int lanes = GROUP / 8, scales_at = Q4_CODES;
    const int zeros_at = scales_at + Q4_K / GROUP * Q4_ROWS * (form.scale_f32 ? 4 : 2);
    uint4 raw[ROUNDS][PIECES];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int r = row0 + r0 + i * (THREADS / 16);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            raw[i][j] = make_uint4(0u, 0u, 0u, 0u);
            if (r < N && k < K) raw[i][j] = __ldcs(reinterpret_cast<const uint4*>(w + (size_t)r * K + k) + j);      // K % 8 == 0; read once
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int r = r0 + i * (THREADS / 16);
        float v[8];
        q4_widen(raw[i], v);
        float lo = 0.f, hi = 0.f;                        // without zeros `hi` is the largest magnitude; no number, or infinite, if a value is
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi = q4_max_nan(hi, ZEROS ? v[j] : fabsf(v[j]));
            if (ZEROS) lo = q4_min_nan(lo, v[j]);
        }
#pragma unroll
        for (int o = 1; o < lanes; o <<= 1) {
            hi = q4_max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            if (ZEROS) lo = q4_min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        const bool odd = !isfinite(hi) || !isfinite(lo);
        float s = odd ? 0.f : ZEROS ? q4_fifteenth(lo, hi) : hi / 7.0f;
        if (!form.scale_f32) s = __bfloat162float(__float2bfloat16_rn(s));
        int zero = 8;
        uint32_t word = 0;
        if (s >= Q4_SMALL) {
            float inv, far = 0.f, t[8];
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
            if (ZEROS) {
                float z = 0.f;
                zero = __float_as_int(q4_mend(-lo, s, q4_round(-lo, s, inv, z))) - __float_as_int(Q4_MAGIC);      // 0 .. 15: the scale is within 2^-8
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2) q4_round2(v[j], v[j + 1], s, inv, t[j], t[j + 1], far);
            if (far >= 0.5f * s)
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = q4_mend(v[j], s, t[j]);
            // Whole numbers -7 .. 7, or with the zero 0 .. 16, of which 16 is cut off.  What the eight floats' bits have beside them is the same for each.
            const float most = Q4_MAGIC + (float)(15 - zero);
            word = (uint32_t)(zero - __float_as_int(Q4_MAGIC)) * 0x11111111u;
#pragma unroll
            for (int j = 0; j < 8; ++j) word += (uint32_t)__float_as_int(ZEROS ? fminf(t[j], most) : t[j]) << (16 * (j & 1) + 4 * ((j >> 1) & 1) + 8 * (j >> 2));
        } else {
            if (ZEROS) zero = s > 0.f ? min(max(q4_rint_small(-lo, s), 0), 15) : 0;
            for (int j = 0; j < 8; ++j) {
                const int c = s > 0.f ? min(max(q4_rint_small(v[j], s) + zero, ZEROS ? 0 : 1), 15) : zero;
                word |= (uint32_t)c << (16 * (j & 1) + 4 * ((j >> 1) & 1) + 8 * (j >> 2));
            }
        }
        reinterpret_cast<uint32_t*>(tile)[((m >> 2) * Q4_ROWS + r) * 4 + (m & 3)] = word;
        if (m % lanes == 0) {
            const int at = (m / lanes) * Q4_ROWS + r;
            if (odd) s = __int_as_float(0x7fc00000);
            if (form.scale_f32) reinterpret_cast<float*>(tile + scales_at)[at] = s;
            else reinterpret_cast<bf16*>(tile + scales_at)[at] = __float2bfloat16_rn(s);
            if (ZEROS) tile[zeros_at + at] = (unsigned char)zero;
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(out + ((size_t)blockIdx.y * blocks + kb) * form.bytes);
    for (int i = threadIdx.x; i < form.bytes / 16; i += THREADS) dst[i] = reinterpret_cast<const uint4*>(tile)[i];
}

__device__ __forceinline__ void q4_store8(float* dst, const float (&v)[8]) {      // (two stores of 16 bytes, 32 apart: 142 us instead of 98 for 136 million)
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                 "f"(v[6]), "f"(v[7]) : "memory");
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
    constexpr int ROUNDS = Q4_ROWS / (QQ_THREADS / 16);
    const int r0 = (threadIdx.x >> 5) * 2 + (lane >> 4), group = 8 * m / form.group * Q4_ROWS;
    uint32_t words[ROUNDS];
    float scale[ROUNDS];
    int zero[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {                   // a stored block is whole, whatever the matrix's last rows
        const int r = r0 + i * (QQ_THREADS / 16);
        words[i] = reinterpret_cast<const uint32_t*>(src)[((m >> 2) * Q4_ROWS + r) * 4 + (m & 3)];
        scale[i] = q4_scale(scales, group + r, form.scale_f32);
        zero[i] = form.zeros ? zeros[group + r] : 8;
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int r = row0 + r0 + i * (QQ_THREADS / 16);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = scale[i] * (float)((int)((words[i] >> (16 * (j & 1) + 4 * ((j >> 1) & 1) + 8 * (j >> 2))) & 15u) - zero[i]);
        if (r < N) q4_store8(out + (size_t)r * K + k, v);
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
    auto run = [&](auto kernel, auto matrix) { return launch_after_wait(kernel, grid, dim3(w_f32 ? QQ_MAKE<float> : QQ_MAKE<bf16>), 0, stream, matrix, (unsigned char*)out, N, K, (int)grid.x, form); };
    auto typed = [&](auto matrix, auto zeros) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(matrix)>>;
        constexpr bool Z = decltype(zeros)::value;
        return form.group == 128 ? run(quantize_q4_kernel<T, Z, 128>, matrix) : form.group == 64 ? run(quantize_q4_kernel<T, Z, 64>, matrix)
                                                                              : run(quantize_q4_kernel<T, Z, 32>, matrix);
    };
    if (w_f32) return form.zeros ? typed((const float*)w, std::true_type()) : typed((const float*)w, std::false_type());
    return form.zeros ? typed((const bf16*)w, std::true_type()) : typed((const bf16*)w, std::false_type());
}

// The values that weights of 4 bits stand for, [N, K] bfloat16 or float (on a 32-byte boundary).
TL_EXPORT int tl_dequantize_q4(const void* w, void* out, int out_f32, int N, int K, int form_bits, cudaStream_t stream) {
    Q4Form form;
    dim3 grid;
    if (N < 1 || K < 1 || (K & 7) || form_bits < 0 || form_bits >> 10 || !q4_form(&form, form_bits & 255, form_bits >> 8 & 1, form_bits >> 9 & 1) || !q4_grid(&grid, N, K) || ((uintptr_t)w & 15) || ((uintptr_t)out & (out_f32 ? 31 : 15))) return 1;
    return out_f32 ? launch_after_wait(dequantize_q4_kernel<float>, grid, dim3(QQ_THREADS), 0, stream, (const unsigned char*)w, (float*)out, N, K, (int)grid.x, form)
                   : launch_after_wait(dequantize_q4_kernel<bf16>, grid, dim3(QQ_THREADS), 0, stream, (const unsigned char*)w, (bf16*)out, N, K, (int)grid.x, form);
}
