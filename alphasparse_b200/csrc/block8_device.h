// Device side of the 8-bit types of asp_b200_block8.h: scales, rounding, loads and stores of the caller's types.
#ifndef ASP_BLOCK8_DEVICE_H
#define ASP_BLOCK8_DEVICE_H
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

namespace asp
{
namespace block8
{
// |v| where it is finite, else 0
__device__ __forceinline__ float finite_size(float v)
{
    v = fabsf(v);
    return v < __int_as_float(0x7f800000) ? v : 0.f;
}

// Exponent + 127 of the scale: the smallest k >= -126 with most <= 448 * 2^k. 448 = 1.75 * 2^8, so k is most's own exponent less 8, and one
// more where its fraction is above 0.75. (Subnormal `most`: exponent field 0, far below the smallest k.)
__device__ __forceinline__ unsigned scale_of(float most)
{
    const unsigned bits = __float_as_uint(most);
    const int k = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)max(k, 1);
}
__device__ __forceinline__ float power(unsigned scale) { return __uint_as_float(scale << 23); }            // 2^k
__device__ __forceinline__ float inverse(unsigned scale) { return __uint_as_float((254u - scale) << 23); } // 2^-k; scale is 1 to 247

// Two elements to e4m3, `a` in the low byte; NaN stays NaN. The conversion saturates: where an element may be infinite it is made NaN first
// (v - v is NaN then, else 0).
template <bool infinite> __device__ __forceinline__ unsigned pack2(float a, float b, float inv)
{
    unsigned short r;
    a = infinite ? __fmaf_rn(a, inv, a - a) : a * inv;
    b = infinite ? __fmaf_rn(b, inv, b - b) : b * inv;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
template <bool infinite> __device__ __forceinline__ unsigned pack4(const float *v, float inv) { return pack2<infinite>(v[0], v[1], inv) | pack2<infinite>(v[2], v[3], inv) << 16; }

// two e4m3 (exact in fp16, NaN included)
__device__ __forceinline__ __half2 unpack2(unsigned two)
{
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)two));
    return *reinterpret_cast<__half2 *>(&h);
}
__device__ __forceinline__ void unpack4(unsigned four, float *v)
{
    const float2 a = __half22float2(unpack2(four & 0xffffu)), b = __half22float2(unpack2(four >> 16));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The 16 elements that lane `lane8` of 8 has of a row's block of 128 columns, and what becomes of them. vec: the row begins on a 16-byte
// boundary and has the whole block; the lane then has pieces of 16 bytes, every eighth one, and otherwise every eighth element, so that the lanes read and
// write side by side either way.
template <class T> __device__ __forceinline__ unsigned column_in_block(int i, unsigned lane8, bool vec)
{
    constexpr int per = 16 / sizeof(T);
    return vec ? i / per * 8 * per + lane8 * per + i % per : 8 * i + lane8;
}
// as they lie in memory, zeros behind the row's end
template <class T> struct Raw
{
    uint4 w[sizeof(T)];
    __device__ __forceinline__ void load(const T *row, unsigned col0, unsigned n_cols, unsigned lane8, bool vec)
    {
        constexpr int per = 16 / sizeof(T);
        if (vec)
#pragma unroll
            for (int i = 0; i < 16 / per; i++) w[i] = *reinterpret_cast<const uint4 *>(row + col0 + column_in_block<T>(i * per, lane8, true));
        else
        {
            T e[16];
#pragma unroll
            for (int i = 0; i < 16; i++)
            {
                const unsigned c = col0 + 8 * i + lane8;
                e[i] = c < n_cols ? row[c] : from_float<T>(0.f);
            }
            memcpy(w, e, sizeof(w));
        }
    }
    __device__ __forceinline__ void floats(float *v) const
    {
        T e[16];
        memcpy(e, w, sizeof(w));
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = to_float(e[i]);
    }
};
// The scale of what the eight lanes of a block have, and whether something infinite is among it. All lanes of the warp take part. (fmaxf passes NaN over;
// only what is infinite takes a second look.)
__device__ __forceinline__ unsigned scale_of_8(const float *v, bool &infinite)
{
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) most = fmaxf(most, fabsf(v[i]));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    infinite = __any_sync(~0u, isinf(most));
    if (infinite)
    {
        most = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) most = fmaxf(most, finite_size(v[i]));
#pragma unroll
        for (int d = 1; d < 8; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    }
    return scale_of(most);
}
// to 8 bits, four to a word, in the order of `v`
__device__ __forceinline__ void pack16(const float *v, unsigned scale, bool infinite, unsigned *q)
{
    const float inv = inverse(scale);
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = infinite ? pack4<true>(v + 4 * i, inv) : pack4<false>(v + 4 * i, inv);
}
// and to where they belong; `to` is the block's first byte
template <class T> __device__ __forceinline__ void store_block(const unsigned *q, bool vec, unsigned lane8, uint8_t *to)
{
    constexpr int per = 16 / sizeof(T);
    if (vec)
#pragma unroll
        for (int i = 0; i < 16; i += per)
        {
            uint8_t *at = to + column_in_block<T>(i, lane8, true);
            if constexpr (per == 4) *reinterpret_cast<unsigned *>(at) = q[i / 4];
            else *reinterpret_cast<uint2 *>(at) = make_uint2(q[i / 4], q[i / 4 + 1]);
        }
    else
#pragma unroll
        for (int i = 0; i < 16; i++) to[8 * i + lane8] = (uint8_t)(q[i / 4] >> 8 * (i % 4));
}
// the other way: a block in 8 bits to the caller's type
template <class T> __device__ __forceinline__ void restore_block(const uint8_t *from, float scale, T *row, unsigned col0, unsigned n_cols, unsigned lane8, bool vec)
{
    constexpr int per = 16 / sizeof(T);
    if (vec)
#pragma unroll
        for (int i = 0; i < 16; i += per)
        {
            const unsigned c = column_in_block<T>(i, lane8, true);
            float v[per];
#pragma unroll
            for (int k = 0; k < per; k += 4) unpack4(*reinterpret_cast<const unsigned *>(from + c + k), v + k);
            uint4 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int k = 0; k < per; k++) e[k] = from_float<T>(v[k] * scale);
            *reinterpret_cast<uint4 *>(row + col0 + c) = w;
        }
    else
#pragma unroll
        for (int i = 0; i < 16; i++)
        {
            const unsigned c = 8 * i + lane8;
            if (col0 + c < n_cols) row[col0 + c] = from_float<T>(__low2float(unpack2(from[c])) * scale);
        }
}
} // namespace block8
} // namespace asp
#endif
