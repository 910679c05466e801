// Device side of the 8-bit types of asp_b200_block8.h: scales, rounding, loads and stores of the caller's types.
#ifndef ASP_BLOCK8_DEVICE_H
#define ASP_BLOCK8_DEVICE_H
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include "block8.h"

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
// (v - v is NaN then, else 0, taken with a minus so that -0 stays -0 wherever it stands).
template <bool infinite> __device__ __forceinline__ unsigned pack2(float a, float b, float inv)
{
    unsigned short r;
    a = infinite ? __fmaf_rn(a, inv, -(a - a)) : a * inv;
    b = infinite ? __fmaf_rn(b, inv, -(b - b)) : b * inv;
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

// ---- copies to shared memory of 16 bytes, by the thread that will read them ----
__device__ __forceinline__ void copy16(void *to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_are_one_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n> __device__ __forceinline__ void wait_for_all_groups_but() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

// ---- rows that begin anywhere ----
// A row's elements are taken 16 bytes at a time whether it begins on a 16-byte boundary or not: a lane loads the aligned piece in which its own begins,
// gets the next one from the lane beside it and shifts the two. (Loads and stores element by element took 2.4 and 3 times as long for rows of
// 4001 bf16.) A piece that is not all inside the caller's matrix is put together from the elements that are.

// bytes [o, o + 16) of `a` and `b` side by side; o = 4 * words + bits / 8
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, unsigned words, unsigned bits)
{
    unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 7; i++) w[i] = words & 1 ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 shuffled(uint4 v, unsigned from)
{
    return make_uint4(__shfl_sync(~0u, v.x, from), __shfl_sync(~0u, v.y, from), __shfl_sync(~0u, v.z, from), __shfl_sync(~0u, v.w, from));
}
// the 16 bytes at p (on a 16-byte boundary), those of them that are in [lo, hi); T: what lies there
template <class T> __device__ __forceinline__ uint4 load_piece(uintptr_t p, uintptr_t lo, uintptr_t hi)
{
    if (p >= lo && p + 16 <= hi) return *reinterpret_cast<const uint4 *>(p);
    uint4 r = make_uint4(0, 0, 0, 0);
    if (p + 16 <= lo || p >= hi) return r;
    T e[16 / sizeof(T)];
#pragma unroll
    for (unsigned i = 0; i < 16 / sizeof(T); i++)
    {
        const uintptr_t at = p + i * sizeof(T);
        e[i] = at >= lo && at < hi ? *reinterpret_cast<const T *>(at) : from_float<T>(0.f);
    }
    memcpy(&r, e, 16);
    return r;
}

// The 16 elements that lane `lane8` of 8 has of a row's block of 128 columns: pieces of 16 bytes, every eighth one.
template <class T> __device__ __forceinline__ unsigned column_in_block(int i, unsigned lane8)
{
    constexpr int per = 16 / sizeof(T);
    return i / per * 8 * per + lane8 * per + i % per;
}
// as they come from memory, from where a block begins (`first`) and with what is inside [lo, hi)
template <class T> struct Raw
{
    static constexpr int per = 16 / sizeof(T), pieces = 16 / per;
    uint4 w[pieces], more; // more: the piece behind the block's last, of its last lane
    unsigned words, bits;
    __device__ __forceinline__ void load(const T *first, const T *lo, const T *hi, unsigned lane8)
    {
        const uintptr_t o = (uintptr_t)first & 15, at = (uintptr_t)first - o + 16 * lane8;
        words = (unsigned)o / 4, bits = (unsigned)o % 4 * 8;
#pragma unroll
        for (int i = 0; i < pieces; i++) w[i] = load_piece<T>(at + 128 * i, (uintptr_t)lo, (uintptr_t)hi);
        if (o && lane8 == 7) more = load_piece<T>(at + 128 * (pieces - 1) + 16, (uintptr_t)lo, (uintptr_t)hi);
    }
    // the lane's elements; all lanes of the warp take part; `columns` of the block are in the row, zeros behind them
    __device__ __forceinline__ void elements(uint4 *u, unsigned lane8, unsigned columns) const
    {
        const unsigned lane = threadIdx.x % 32, beside = lane8 < 7 ? lane + 1 : lane - 7;
        if (__any_sync(~0u, words | bits))
        {
#pragma unroll
            for (int i = 0; i < pieces; i++)
            {
                // the first lane of a block is asked for its next piece, by the last one
                uint4 next = shuffled(lane8 == 0 && i + 1 < pieces ? w[i + 1 < pieces ? i + 1 : i] : w[i], beside);
                if (i + 1 == pieces && lane8 == 7) next = more;
                u[i] = shifted(w[i], next, words, bits);
            }
        }
        else
#pragma unroll
            for (int i = 0; i < pieces; i++) u[i] = w[i];
        if (columns < 128)
        {
            T e[16];
            memcpy(e, u, sizeof(e));
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (column_in_block<T>(i, lane8) >= columns) e[i] = from_float<T>(0.f);
            memcpy(u, e, sizeof(e));
        }
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
template <class T> __device__ __forceinline__ unsigned floats_to_eight(const uint4 *u, unsigned *q)
{
    T e[16];
    memcpy(e, u, sizeof(e));
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = to_float(e[i]);
    bool infinite;
    const unsigned scale = scale_of_8(v, infinite);
    pack16(v, scale, infinite, q);
    return scale;
}
// Both at once: what the eight lanes of a block have (Raw::elements) to 8 bits, and the scale. All lanes of the warp take part.
template <class T> __device__ __forceinline__ unsigned to_eight(const uint4 *u, unsigned *q) { return floats_to_eight<T>(u, q); }
// 16-bit types two elements at a time: the largest, and the division, which is exact, or leaves something that is zero in 8 bits. What is infinite,
// and numbers near fp16's smallest, whose scales it does not have, go by 32 bits.
template <class Two> __device__ __forceinline__ float largest_of_8(const Two *e)
{
    Two most = __habs2(e[0]); // (the larger of a number and NaN is the number)
#pragma unroll
    for (int i = 1; i < 8; i++) most = __hmax2(most, __habs2(e[i]));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) most = __hmax2(most, __shfl_xor_sync(~0u, most, d));
    return fmaxf(fmaxf(to_float(most.x), to_float(most.y)), 0.f);
}
template <> __device__ __forceinline__ unsigned to_eight<__nv_bfloat16>(const uint4 *u, unsigned *q)
{
    __nv_bfloat162 e[8];
    memcpy(e, u, sizeof(e));
    const float most = largest_of_8(e);
    if (__any_sync(~0u, isinf(most))) return floats_to_eight<__nv_bfloat16>(u, q);
    const unsigned scale = scale_of(most);
    const __nv_bfloat162 inv = __float2bfloat162_rn(inverse(scale));
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        const float2 v = __bfloat1622float2(__hmul2(e[i], inv));
        unsigned short two;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(v.y), "f"(v.x));
        q[i / 2] = i % 2 ? q[i / 2] | (unsigned)two << 16 : two;
    }
    return scale;
}
template <> __device__ __forceinline__ unsigned to_eight<__half>(const uint4 *u, unsigned *q)
{
    __half2 e[8];
    memcpy(e, u, sizeof(e));
    const float most = largest_of_8(e);
    if (__any_sync(~0u, isinf(most) || (most > 0.f && most < 0x1p-21f))) return floats_to_eight<__half>(u, q);
    const unsigned scale = scale_of(most);
    const int up = most > 0.f ? 127 - (int)scale : 0, first = min(up, 15); // -8 to 30
    const __half2 f1 = __float2half2_rn(power((unsigned)(127 + first))), f2 = __float2half2_rn(power((unsigned)(127 + up - first)));
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        const __half2 v = __hmul2(__hmul2(e[i], f1), f2);
        unsigned short two;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(two) : "r"(*reinterpret_cast<const unsigned *>(&v)));
        q[i / 2] = i % 2 ? q[i / 2] | (unsigned)two << 16 : two;
    }
    return scale;
}
// Rows X of a product: as the caller has them (of type X), or in 8 bits already (Held)
struct Held
{
};
struct XRows
{
    const void *p;
    uint64_t ld;
    unsigned n, n_cols;
    Rows8Dev held;
};
// What lane `lane8` of 8 has of a row's block on its way
template <class X> struct Fetched
{
    Raw<X> raw;
    unsigned columns; // of the block that are in the row
    __device__ __forceinline__ void ask(const XRows &rows, unsigned row, unsigned kb, unsigned lane8)
    {
        const X *x = reinterpret_cast<const X *>(rows.p);
        columns = rows.n_cols - kb * 128;
        raw.load(x + row * rows.ld + kb * 128, x, x + (rows.n - 1) * rows.ld + rows.n_cols, lane8);
    }
    // 16 elements in 8 bits, element i that of column column(i, lane8), and their scale. All lanes of the warp take part.
    __device__ __forceinline__ unsigned eight(unsigned *q, unsigned lane8) const
    {
        uint4 u[Raw<X>::pieces];
        raw.elements(u, lane8, columns);
        return to_eight<X>(u, q);
    }
    static constexpr int per = 16 / sizeof(X); // elements side by side
    static __device__ __forceinline__ unsigned column(int i, unsigned lane8) { return column_in_block<X>(i, lane8); }
};
template <> struct Fetched<Held>
{
    uint4 v;
    unsigned scale;
    __device__ __forceinline__ void ask(const XRows &rows, unsigned row, unsigned kb, unsigned lane8)
    {
        v = *reinterpret_cast<const uint4 *>(rows.held.values + row * rows.held.ld + kb * 128 + 16 * lane8);
        scale = rows.held.scales[scale_at(rows.held, row, kb)];
    }
    __device__ __forceinline__ unsigned eight(unsigned *q, unsigned) const
    {
        q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
        return scale;
    }
    static constexpr int per = 16;
    static __device__ __forceinline__ unsigned column(int i, unsigned lane8) { return 16 * lane8 + i; }
};
// and to where they belong; `to` is the block's first byte
template <class T> __device__ __forceinline__ void store_block(const unsigned *q, unsigned lane8, uint8_t *to)
{
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += per)
    {
        uint8_t *at = to + column_in_block<T>(i, lane8);
        if constexpr (per == 4) *reinterpret_cast<unsigned *>(at) = q[i / 4];
        else *reinterpret_cast<uint2 *>(at) = make_uint2(q[i / 4], q[i / 4 + 1]);
    }
}
// The other way, for a warp's four blocks: `from` is the block's first byte, `first` where it goes to, `end` where the row ends. Pieces of 16 bytes that are not all
// the warp's are stored element by element. All lanes of the warp take part.
template <class T> __device__ __forceinline__ void restore_block(const uint8_t *from, float scale, T *first, T *end, unsigned lane8)
{
    constexpr int per = 16 / sizeof(T), pieces = 16 / per;
    const unsigned lane = threadIdx.x % 32;
    uint4 u[pieces];
#pragma unroll
    for (int i = 0; i < pieces; i++)
    {
        const unsigned c = column_in_block<T>(i * per, lane8);
        float v[per];
#pragma unroll
        for (int k = 0; k < per; k += 4) unpack4(*reinterpret_cast<const unsigned *>(from + c + k), v + k);
        T e[per];
#pragma unroll
        for (int k = 0; k < per; k++) e[k] = from_float<T>(v[k] * scale);
        memcpy(&u[i], e, 16);
    }
    const uintptr_t o = (uintptr_t)first & 15, lo = (uintptr_t)(first - lane / 8 * 128), hi = min((uintptr_t)end, lo + 512 * sizeof(T)); // of the warp's elements
    const auto put = [&](uintptr_t at, uint4 w) {
        if (at >= lo && at + 16 <= hi) *reinterpret_cast<uint4 *>(at) = w;
        else
        {
            T e[per];
            memcpy(e, &w, 16);
#pragma unroll
            for (int k = 0; k < per; k++)
                if (at + k * sizeof(T) >= lo && at + k * sizeof(T) < hi) *reinterpret_cast<T *>(at + k * sizeof(T)) = e[k];
        }
    };
    uintptr_t at = (uintptr_t)first - o + 16 * lane8;
    if (o == 0) // (of a row: the same for all of the warp)
    {
#pragma unroll
        for (int i = 0; i < pieces; i++) put(at + 128 * i, u[i]);
        return;
    }
    // the last o bytes of the piece before, and the first of one's own
    const unsigned words = (16 - (unsigned)o) / 4, bits = (16 - (unsigned)o) % 4 * 8;
#pragma unroll
    for (int i = 0; i < pieces; i++)
    {
        const uint4 beside = shuffled(u[i], lane - 1 & 31), far = shuffled(u[i > 0 ? i - 1 : pieces - 1], i > 0 ? lane + 7 & 31 : lane - 1 & 31);
        put(at + 128 * i, shifted(lane8 ? beside : far, u[i], words, bits));
    }
    // behind the warp's last piece
    if (lane == 31) put(at + 128 * (pieces - 1) + 16, shifted(u[pieces - 1], make_uint4(0, 0, 0, 0), words, bits));
}
} // namespace block8
} // namespace asp
#endif
