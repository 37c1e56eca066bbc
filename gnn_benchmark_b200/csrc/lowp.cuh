// Element types of the low-precision path: 16-byte vectors of fp32 / bf16 / fp16 as fp32 registers, and the
// e4m3 blocks that the 8-bit operands and optimiser moments are held in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace gnnagg {

// Block scaling: a = max |u| over the block, at least 2^-96 (so that its reciprocal stays finite);
// code = e4m3(u * (448 * (1 / a))), value = code * (a * (1 / 448)).  Every step is rounded to nearest on its
// own, so that the codes are the same however a caller computes them.
constexpr float kE4m3Max = 448.0f;
constexpr float kBlockTiny = 1.262177448e-29f;  // 2^-96
static_assert(kBlockTiny == 1.0f / 79228162514264337593543950336.0f, "2^-96");

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
// Largest magnitudes are compared as bit patterns: the order of |x|, with NaN above infinity, so a block that
// holds a NaN or an infinity gets a NaN or infinite scale and reads back as NaN instead of losing it.
__device__ __forceinline__ float block_amax(uint32_t bits) {
    return __uint_as_float(max(bits, __float_as_uint(kBlockTiny)));
}
__device__ __forceinline__ float block_factor(float amax) { return __fmul_rn(__frcp_rn(amax), kE4m3Max); }
__device__ __forceinline__ float block_scale(float amax) { return __fmul_rn(amax, 1.0f / kE4m3Max); }

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ float4 from_e4m3x4(uint32_t v) {
    const __half2 lo(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xFFFFu), __NV_E4M3));
    const __half2 hi(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> 16), __NV_E4M3));
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    return make_float4(a.x, a.y, b.x, b.y);
}

enum : int { kTypeF32 = GNNAGG_F32, kTypeBf16 = GNNAGG_BF16, kTypeF16 = GNNAGG_F16 };

inline int type_size(int type) { return type == kTypeF32 ? 4 : (type == kTypeBf16 || type == kTypeF16 ? 2 : 0); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float load_as_f32(const void *p, int type, int64_t i) {
    return type == kTypeF32    ? static_cast<const float *>(p)[i]
           : type == kTypeBf16 ? to_f32(static_cast<const __nv_bfloat16 *>(p)[i])
                               : to_f32(static_cast<const __half *>(p)[i]);
}

// 16 bytes global -> shared; completed as the copies of 4 bytes are (common.cuh).
__device__ __forceinline__ void cp_async_16(void *smem, const void *gmem) {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
}

template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);  // elements of one 16-byte access
};

// A 16-byte vector as fp32 values and back, one instruction an element and one for two (element by element the
// compiler takes two each).
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &u, float (&f)[Vec<T>::N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (std::is_same<T, float>::value) {
            f[i] = __uint_as_float(w[i]);
        } else if (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of an fp32
            f[2 * i % Vec<T>::N] = __uint_as_float(w[i] << 16);
            f[(2 * i + 1) % Vec<T>::N] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[2 * i % Vec<T>::N] = v.x, f[(2 * i + 1) % Vec<T>::N] = v.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[Vec<T>::N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = f[2 * i % Vec<T>::N], b = f[(2 * i + 1) % Vec<T>::N];
        if (std::is_same<T, float>::value) {
            w[i] = __float_as_uint(f[i]);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t *>(&v);
        } else {
            const __half2 v = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t *>(&v);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Vec<T>::N consecutive elements at p, of which `valid` exist (the others read as zero), as they lie in memory: a
// 16-bit row held this way takes half the registers of its fp32 values.  VEC: one 16-byte access (p aligned, all
// valid); otherwise element by element.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_raw(const T *p, int valid) {
    if (VEC) return __ldcs(reinterpret_cast<const uint4 *>(p));
    uint4 u = make_uint4(0, 0, 0, 0);
    T *e = reinterpret_cast<T *>(&u);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
        if (i < valid) e[i] = p[i];
    return u;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_raw(T *p, int valid, const uint4 &u) {
    if (VEC) {
        __stcs(reinterpret_cast<uint4 *>(p), u);
    } else {
        const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i)
            if (i < valid) p[i] = e[i];
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T *p, int valid, float (&f)[Vec<T>::N]) {
    unpack16<T>(load_raw<T, VEC>(p, valid), f);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(T *p, int valid, const float (&f)[Vec<T>::N]) {
    store_raw<T, VEC>(p, valid, pack16<T>(f));
}

// A thread's 16 bytes of a row as pieces of P neighbouring elements, one access each: piece q starts at column first +
// q * step (columns from F on read as zero and are not written).  P = Vec<T>::N is a 16-byte vector; with smaller P, for
// rows that do not allow it, neighbouring threads take neighbouring pieces, so that a warp's access is contiguous.
template <int BYTES>
struct Access;
template <>
struct Access<16> {
    using type = uint4;
};
template <>
struct Access<4> {
    using type = uint32_t;
};
template <>
struct Access<2> {
    using type = uint16_t;
};
template <typename T, int P>
__device__ __forceinline__ uint4 load_pieces(const T *row, int first, int step, int F) {
    using A = typename Access<P * (int)sizeof(T)>::type;
    uint4 u = make_uint4(0, 0, 0, 0);
    A *piece = reinterpret_cast<A *>(&u);
#pragma unroll
    for (int q = 0; q < Vec<T>::N / P; ++q)
        if (first + q * step < F) piece[q] = __ldcs(reinterpret_cast<const A *>(row + first + q * step));
    return u;
}
template <typename T, int P>
__device__ __forceinline__ void store_pieces(T *row, int first, int step, int F, const uint4 &u) {
    using A = typename Access<P * (int)sizeof(T)>::type;
    const A *piece = reinterpret_cast<const A *>(&u);
#pragma unroll
    for (int q = 0; q < Vec<T>::N / P; ++q)
        if (first + q * step < F) __stcs(reinterpret_cast<A *>(row + first + q * step), piece[q]);
}

// out[c] = sum of partial[b][c] over the blocks, in a fixed order: 16 threads take every 16th block of a column.
template <typename T>
__global__ void __launch_bounds__(512) column_sum_kernel(const float *__restrict__ partial, int64_t blocks, int64_t F, T *out) {
    __shared__ float red[16][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < F) {
#pragma unroll 8
        for (int64_t b = threadIdx.y; b < blocks; b += 16) s += partial[b * F + c];
    }
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < F) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
        out[c] = from_f32<T>(s);
    }
}

}  // namespace gnnagg
