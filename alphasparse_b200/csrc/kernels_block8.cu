// Block-sparse 8-bit matrices (asp_b200_block8.h): conversions to and from 8 bits, products with a few rows.
#include "../../include/asp_b200.h"
#include "block8.h"
#include "block8_device.h"
#include "host/block8_plan.hpp"
#include "launch.h"

#include <cooperative_groups.h>


namespace asp
{
namespace
{
using namespace block8;

template <class F> cudaError_t by_type(int dtype, F f)
{
    if (dtype == ASP_F32) return f(float());
    if (dtype == ASP_F16) return f(__half());
    return f(__nv_bfloat16());
}

// ---- rows ----------------------------------------------------------------------------------------------------------

// A row's four blocks to a warp, 8 lanes and 16 elements a lane each, so that an element is read once, its block's largest is known after
// three exchanges, and the four scales leave as a word. Bounded by memory: 8192 x 8192 bf16 in 32.8 us, 202 MB at 6.2 TB/s. Eight rows to a CTA: no
// warp waits for another. Rows that begin anywhere cost the shifts: 4096 x 4001 bf16 in 11.8 us (8.7 for 4096 x 4096).
template <class T> __global__ void __launch_bounds__(256) k_rows8_quantize(const T *x, uint64_t ld, unsigned n, Rows8Dev out)
{
    const unsigned lane = threadIdx.x % 32, lane8 = lane % 8, n_blocks = (out.n_cols + 127) / 128, fours = (n_blocks + 3) / 4;
    const unsigned blk0 = blockIdx.x % fours * 4, blk = blk0 + lane / 8, row = blockIdx.x / fours * 8 + threadIdx.x / 32;
    grid_wait();
    grid_release();
    if (row >= n) return;
    Raw<T> raw;
    raw.load(x + (uint64_t)row * ld + blk * 128, x, x + (uint64_t)(n - 1) * ld + out.n_cols, lane8);
    uint4 u[Raw<T>::pieces];
    raw.elements(u, lane8, out.n_cols - min(out.n_cols, blk * 128)); // (zeros behind the last column, and behind the last block)
    unsigned q[4];
    const unsigned scale = to_eight<T>(u, q);
    if (blk < n_blocks) store_block<T>(q, lane8, out.values + (uint64_t)row * out.ld + blk * 128);
    unsigned four = scale << lane / 8 * 8;
    four |= __shfl_xor_sync(~0u, four, 8);
    four |= __shfl_xor_sync(~0u, four, 16);
    if (lane == 0) *reinterpret_cast<unsigned *>(out.scales + scale_at(out, row, blk0)) = four; // (those behind the last block are not used)
}

// The same the other way: 8192 x 4096 to bf16 in 17 us, 101 MB at 5.9 TB/s; 4096 x 4001 in 15.6, as the ends of a warp's part
// of a row are stored element by element. Registers are held down so that 48 (32 bits) or 64 (16 bits) warps fit an SM.
template <class T> __global__ void __launch_bounds__(256, sizeof(T) == 2 ? 8 : 6) k_rows8_restore(Rows8Dev x, T *out, uint64_t ld)
{
    const unsigned lane = threadIdx.x % 32, lane8 = lane % 8, n_blocks = (x.n_cols + 127) / 128, fours = (n_blocks + 3) / 4;
    const unsigned blk = blockIdx.x % fours * 4 + lane / 8, row = blockIdx.x / fours * 8 + threadIdx.x / 32;
    grid_wait();
    grid_release();
    if (row >= x.n) return;
    T *to = out + (uint64_t)row * ld;
    const unsigned b = min(blk, n_blocks - 1); // (lanes without a block read the last one's, and store nothing)
    restore_block(x.values + (uint64_t)row * x.ld + b * 128, power(x.scales[scale_at(x, row, b)]), to + blk * 128, to + x.n_cols, lane8);
}

// ---- the matrix's values --------------------------------------------------------------------------------------------

// A block to a CTA, its 64 elements a thread in registers between the search for the largest and the conversion. Thread t has rows
// 16 i + t / 16 (i = 0..7), columns 8 (t % 16) on. The transposed copy goes through shared memory, so that both are written in whole lines. Bounded by memory: 1024
// blocks of 32 bits with their transposed copies in 14.2 us, 102 MB at 7.2 TB/s (what is written stays in L2).
__device__ __forceinline__ void put_scale(const Block8Set &to, unsigned block, unsigned scale)
{
    if (threadIdx.x == 0) to.scales[block] = (uint8_t)scale;
    if (threadIdx.x < 128) reinterpret_cast<unsigned *>(to.scale_rows)[(uint64_t)block * 128 + threadIdx.x] = scale * 0x01010101u;
}
template <class T>
__global__ void __launch_bounds__(256) k_block8_set(const T *from, const unsigned *row, const unsigned *col, const unsigned *place, Block8Set a, Block8Set t, unsigned first, unsigned n_rows,
                                                    unsigned n_cols)
{
    __shared__ float largest[8];
    __shared__ __align__(16) uint8_t tile[128][132];
    const unsigned b = first + blockIdx.x, r0 = threadIdx.x / 16, c0 = 8 * (threadIdx.x % 16);
    const T *src = from + (uint64_t)blockIdx.x * 16384 + r0 * 128 + c0;
    const unsigned rows = min(128u, n_rows - row[b] * 128), cols = min(128u, n_cols - col[b] * 128); // inside the matrix
    float v[8][8];
    float most = 0.f;
    grid_wait();
    grid_release();
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        constexpr int per = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8; j += per)
        {
            const uint4 w = *reinterpret_cast<const uint4 *>(src + i * 16 * 128 + j);
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int k = 0; k < per; k++)
            {
                v[i][j + k] = r0 + 16 * i < rows && c0 + j + k < cols ? to_float(e[k]) : 0.f;
                most = fmaxf(most, finite_size(v[i][j + k]));
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    if (threadIdx.x % 32 == 0) largest[threadIdx.x / 32] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) most = fmaxf(most, largest[i]);
    const unsigned scale = scale_of(most);
    const float inv = inverse(scale);
    uint8_t *to = a.values + (uint64_t)b * 16384 + r0 * 128 + c0;
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        const uint2 q = make_uint2(pack4<true>(v[i], inv), pack4<true>(v[i] + 4, inv));
        *reinterpret_cast<uint2 *>(to + i * 16 * 128) = q;
        if (t.values)
        {
            unsigned *s = reinterpret_cast<unsigned *>(&tile[r0 + 16 * i][c0]);
            s[0] = q.x, s[1] = q.y;
        }
    }
    put_scale(a, b, scale);
    if (!t.values) return;
    const unsigned bt = place[b];
    put_scale(t, bt, scale);
    __syncthreads();
    // row c of the transposed block: the elements of column c
    for (unsigned i = threadIdx.x; i < 128 * 32; i += 256)
    {
        const unsigned c = i % 128, r = i / 128 * 4; // (consecutive threads, consecutive columns: no conflicts)
        const unsigned w = tile[r][c] | tile[r + 1][c] << 8 | tile[r + 2][c] << 16 | (unsigned)tile[r + 3][c] << 24;
        *reinterpret_cast<unsigned *>(t.values + (uint64_t)bt * 16384 + c * 128 + r) = w;
    }
}

// Four elements and 16 bytes a thread, four times. Bounded by what it writes: 1024 blocks in 10.6 us, 84 MB at 7.9 TB/s (in part to L2).
__global__ void __launch_bounds__(256) k_block8_get(const uint8_t *values, const uint8_t *scales, float *out)
{
    const uint64_t at = (uint64_t)blockIdx.x * 4096 + threadIdx.x * 4;
    grid_wait();
    grid_release();
    const float scale = power(scales[blockIdx.x / 4]);
    unsigned q[4];
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = *reinterpret_cast<const unsigned *>(values + at + i * 1024);
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        float v[4];
        unpack4(q[i], v);
        *reinterpret_cast<float4 *>(out + at + i * 1024) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
    }
}

// ---- products with a few rows ----------------------------------------------------------------------------------------

// n <= 32 rows, a few blocks a CTA (block8_batch). Y[t][128 R + r] = sum over the blocks j of block row R of 2^(kA + kX) sum over c of A_j[r][c] X_j[t][c].
//
// The matrix is read once and nothing else counts: 16 KB a block, four or five blocks ahead, as the A operand of m16n8k16 with a warp to 16 rows (a
// thread copies what it will itself read: no warp waits for another's); X in shared memory is the B operand, 8 rows of it a tile. Both as fp16, which has every e4m3 number: the form for e4m3 converts
// both operands anew in each product (556 instructions a block and warp for 32 rows instead of 190). The order of the 128 columns in a sum is free, so a lane
// takes 16 bytes of a row at once (columns 64 h + 16 q on) and its words serve four products. A block's sum is in the products' own units; it is
// scaled by both powers of two in 32 bits, in two halves, since the product of the two may not be a number although the result is one.
//
// A block row is shared by a cluster of CTAs, a contiguous piece of its blocks each, so that all SMs read; the cluster adds up the pieces in
// order in one another's shared memory: no atomics, no room, the same bits every time.
//
// A form for each 8 rows: 19 rows, 60 % of 4001 x 2047, 7.5 us, 7.9 by the one for 32.
//
// X is converted for 4 / NT blocks at a time, which is a row's block to each eight lanes, and asked for while the stage before the one before is
// multiplied: a stage's X is in shared memory, the next one's in registers.
//
// One row of bf16, half of 1024 x 1024: 3.1 us, of which the blocks are the least: a launch, X on its way and converted, the products, the cluster's sum. 4096 x 4096, all
// of it: 6.0 us, 2.8 TB/s, where the matrix is in L2, 7.7 where it is not.
constexpr int kFewPitch = 272; // bytes a row and block: 16-byte reads of 8 lanes in 2 rows meet no conflict
template <int NT> constexpr int kFewAhead = NT >= 3 ? 4 : 5; // blocks on their way: two CTAs' 128 or 160 KB an SM, with room for X
template <int NT> struct FewShared
{
    uint4 a[kFewAhead<NT>][4][256];
    static constexpr unsigned per = 4 / NT; // blocks a stage
    uint8_t x[2][per][8 * NT][kFewPitch];
    float2 factor[2][per][8 * NT];
    float part[8 * NT][132];
};

struct FewArgs
{
    Block8Dev a;
    XRows x;
    void *y;
    uint64_t ldy;
    unsigned n_split;
};

__device__ __forceinline__ void mma_f16(float *c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 elements as eight words of two
__device__ __forceinline__ void unpack16(uint4 q, unsigned *h)
{
    const unsigned in[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        const __half2 v = unpack2(in[i / 2] >> 16 * (i % 2) & 0xffffu);
        h[i] = *reinterpret_cast<const unsigned *>(&v);
    }
}

// eight lanes' part of a row's block to shared memory, as fp16 in the products' units
template <class X> __device__ __forceinline__ unsigned put(const Fetched<X> &got, uint8_t *to, unsigned lane8, bool there) // (`there` or not, for the exchanges)
{
    unsigned q[4], h[8];
    const unsigned scale = got.eight(q, lane8);
    if (!there) return scale;
    unpack16(make_uint4(q[0], q[1], q[2], q[3]), h);
#pragma unroll
    for (int i = 0; i < 16; i += Fetched<X>::per)
    {
        uint8_t *at = to + 2 * Fetched<X>::column(i, lane8);
        if constexpr (Fetched<X>::per == 4) *reinterpret_cast<uint2 *>(at) = make_uint2(h[i / 2], h[i / 2 + 1]);
        else
#pragma unroll
            for (int k = 0; k < Fetched<X>::per / 2; k += 4) *reinterpret_cast<uint4 *>(at + 4 * k) = make_uint4(h[i / 2 + k], h[i / 2 + k + 1], h[i / 2 + k + 2], h[i / 2 + k + 3]);
    }
    return scale;
}

template <int NT, class X, class Y> __global__ void __launch_bounds__(256, 2) k_block8_few(const FewArgs args)
{
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) unsigned char raw[];
    FewShared<NT> &sh = *reinterpret_cast<FewShared<NT> *>(raw);
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned split = args.n_split, piece = blockIdx.x % split;
    const uint4 mine_of = args.a.rows[blockIdx.x / split];
    const unsigned tokens = args.x.n, br = mine_of.x, lo = mine_of.y, len = mine_of.z;
    const unsigned j0 = lo + (unsigned)((uint64_t)len * piece / split), j1 = lo + (unsigned)((uint64_t)len * (piece + 1) / split);
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q = lane % 4;

    constexpr unsigned per = FewShared<NT>::per;
    const uint8_t *mine = args.a.values + (warp * 16 + g) * 128 + 16 * q;
    const auto load = [&](unsigned j) { // (a group of copies for each block, empty ones behind the last)
        if (j < j1)
        {
            const uint8_t *p = mine + (uint64_t)j * 16384;
            uint4(*to)[256] = sh.a[(j - j0) % kFewAhead<NT>];
            copy16(&to[0][threadIdx.x], p), copy16(&to[1][threadIdx.x], p + 8 * 128), copy16(&to[2][threadIdx.x], p + 64), copy16(&to[3][threadIdx.x], p + 64 + 8 * 128);
        }
        copies_are_one_group();
    };
    float acc[NT][4] = {};
    const auto add = [&](unsigned j) {
        const uint4(*w)[256] = sh.a[(j - j0) % kFewAhead<NT>];
        const unsigned at = (j - j0) / per % 2, slot = (j - j0) % per;
        float c[NT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            unsigned lo[8], hi[8]; // of rows g and g + 8
            unpack16(w[2 * h][threadIdx.x], lo);
            unpack16(w[2 * h + 1][threadIdx.x], hi);
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                {
                    const uint4 b = *reinterpret_cast<const uint4 *>(&sh.x[at][slot][8 * nt + g][128 * h + 32 * q + 16 * m]);
                    mma_f16(c[nt], lo[4 * m], hi[4 * m], lo[4 * m + 1], hi[4 * m + 1], b.x, b.y);
                    mma_f16(c[nt], lo[4 * m + 2], hi[4 * m + 2], lo[4 * m + 3], hi[4 * m + 3], b.z, b.w);
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
        {
            const float4 f = *reinterpret_cast<const float4 *>(&sh.factor[at][slot][8 * nt + 2 * q]);
            acc[nt][0] = __fmaf_rn(c[nt][0] * f.x, f.y, acc[nt][0]);
            acc[nt][1] = __fmaf_rn(c[nt][1] * f.z, f.w, acc[nt][1]);
            acc[nt][2] = __fmaf_rn(c[nt][2] * f.x, f.y, acc[nt][2]);
            acc[nt][3] = __fmaf_rn(c[nt][3] * f.z, f.w, acc[nt][3]);
        }
    };
    // Until the kernels before this one are done the matrix may still be written: it is brought to L2, which is never behind, and read afterwards.
    if (threadIdx.x == 0 && j0 < j1)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(args.a.values + (uint64_t)j0 * 16384), "r"(min(j1 - j0, 8u) * 16384) : "memory");
    for (unsigned i = threadIdx.x; i < sizeof(sh.x) / 16; i += 256) reinterpret_cast<uint4 *>(sh.x)[i] = make_uint4(0, 0, 0, 0);
    for (unsigned i = threadIdx.x; i < 2 * per * 8 * NT; i += 256) (&sh.factor[0][0][0])[i] = make_float2(1.f, 1.f);
    grid_wait();
    grid_release();
#pragma unroll
    for (int k = 0; k < kFewAhead<NT>; k++) load(j0 + k);
    const unsigned lane8 = lane % 8, task = threadIdx.x / 8, t = task % (8 * NT), slot = task / (8 * NT); // the row and the stage's block that these eight lanes convert
    Fetched<X> got = {};
    unsigned block_scale = 127;
    const auto ask = [&](unsigned j) { // of the stage that begins with block j
        if (j + slot >= j1 || slot >= per || t >= tokens) return; // (24 rows leave 8 tasks over)
        got.ask(args.x, t, args.a.col[j + slot], lane8);
        block_scale = args.a.scales[j + slot];
    };
    const auto convert = [&](unsigned j) {
        const unsigned at = (j - j0) / per % 2;
        const bool there = j + slot < j1 && slot < per && t < tokens;
        const unsigned both = put(got, sh.x[at][slot % per][t], lane8, there) + block_scale, half = both / 2; // exponents + 127 each
        if (there && lane8 == 0) sh.factor[at][slot][t] = make_float2(power(half), power(both - half));
    };
    ask(j0);
    __syncthreads(); // (zeros everywhere)
    convert(j0);
    ask(j0 + per);
    for (unsigned j = j0; j < j1; j += per)
    {
        __syncthreads();
        if (j + per < j1) // (the same for all of the CTA)
        {
            convert(j + per);
            ask(j + 2 * per);
        }
        for (unsigned k = j; k < min(j + per, j1); k++)
        {
            wait_for_all_groups_but<kFewAhead<NT> - 1>();
            add(k);
            load(k + kFewAhead<NT>);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            sh.part[8 * nt + 2 * q + i][warp * 16 + g] = acc[nt][i];
            sh.part[8 * nt + 2 * q + i][warp * 16 + g + 8] = acc[nt][2 + i];
        }
    cluster.sync();
    Y *y = reinterpret_cast<Y *>(args.y);
    for (unsigned i = threadIdx.x + 256 * piece; i < tokens * 128; i += 256 * split)
    {
        const unsigned t = i / 128, r = i % 128;
        float v[8], sum = 0.f; // all on their way before the first is needed
#pragma unroll
        for (unsigned s = 0; s < 8; s++) v[s] = s < split ? *cluster.map_shared_rank(&sh.part[t][r], s) : 0.f;
#pragma unroll
        for (unsigned s = 0; s < 8; s++) sum += v[s]; // (in order; zeros behind the last change nothing)
        if (br * 128 + r < args.a.n_rows) y[(uint64_t)t * args.ldy + br * 128 + r] = from_float<Y>(sum);
    }
    cluster.sync(); // (its shared memory is read until here)
}

template <int NT, class X, class Y> cudaError_t few(FewArgs &args, cudaStream_t st)
{
    auto *kernel = k_block8_few<NT, X, Y>;
    const size_t smem = sizeof(FewShared<NT>);
    static SharedAllowance allowance;
    static ClusterRoom room;
    unsigned fit[9];
    cudaError_t e = allowance.need((const void *)kernel, (int)smem);
    if (e == cudaSuccess) e = room.most((const void *)kernel, 256, smem, fit);
    if (e != cudaSuccess) return e;
    args.n_split = host::block8_few_split(args.a.n_block_rows, args.a.longest, FewShared<NT>::per, fit);
    return launch_pdl_cluster(kernel, args.n_split, dim3(args.a.n_block_rows * args.n_split), dim3(256), smem, st, args);
}
template <class X, class Y> cudaError_t few_by_rows(FewArgs &args, cudaStream_t st)
{
    if (args.x.n <= 8) return few<1, X, Y>(args, st);
    if (args.x.n <= 16) return few<2, X, Y>(args, st);
    if (args.x.n <= 24) return few<3, X, Y>(args, st);
    return few<4, X, Y>(args, st);
}
} // namespace

cudaError_t launch_rows8_quantize(const Dense &x, unsigned n, const Rows8Dev &out, cudaStream_t st)
{
    if (n == 0) return cudaSuccess;
    return by_type(x.dtype, [&](auto t) {
        using T = decltype(t);
        const unsigned grid = (out.n_cols + 511) / 512 * ((n + 7) / 8);
        return launch_pdl(k_rows8_quantize<T>, dim3(grid), dim3(256), 0, st, (const T *)x.p, x.ld, n, out);
    });
}

cudaError_t launch_rows8_restore(const Rows8Dev &x, const Dense &out, cudaStream_t st)
{
    if (x.n == 0) return cudaSuccess;
    return by_type(out.dtype, [&](auto t) {
        using T = decltype(t);
        const unsigned grid = (x.n_cols + 511) / 512 * ((x.n + 7) / 8);
        return launch_pdl(k_rows8_restore<T>, dim3(grid), dim3(256), 0, st, x, (T *)out.p, out.ld);
    });
}

cudaError_t launch_block8_set(const Block8Dev &a, const unsigned *row, const unsigned *place, const Block8Set to[2], const void *from, int dtype, unsigned first, unsigned end, cudaStream_t st)
{
    if (first >= end) return cudaSuccess;
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_pdl(k_block8_set<T>, dim3(end - first), dim3(256), 0, st, (const T *)from, row, a.col, place, to[0], to[1], first, a.n_rows, a.n_cols);
    });
}

cudaError_t launch_block8_get(const Block8Dev &a, float *out, cudaStream_t st)
{
    if (a.n_blocks == 0) return cudaSuccess;
    return launch_pdl(k_block8_get, dim3(a.n_blocks * 4), dim3(256), 0, st, a.values, a.scales, out);
}

cudaError_t launch_block8_few(const Block8Dev &a, const Dense *x, const Rows8Dev *held, unsigned n, const Dense &y, int sm_count, unsigned *fault, cudaStream_t st)
{
    if (n == 0) return cudaSuccess;
    unsigned fit[9];
    const cudaError_t e = block8_batch_room(fit);
    if (e != cudaSuccess) return e;
    if (host::block8_batch(a.n_block_rows, a.longest, n, y.dtype == ASP_F32, sm_count, fit)) return launch_block8_batch(a, x, held, n, y, sm_count, fit, fault, st);
    FewArgs args = {};
    args.a = a;
    args.x.n = n, args.x.n_cols = a.n_cols;
    args.y = y.p;
    args.ldy = y.ld;
    return by_type(y.dtype, [&](auto ty) {
        using Y = decltype(ty);
        if (held)
        {
            args.x.held = *held;
            return few_by_rows<Held, Y>(args, st);
        }
        args.x.p = x->p, args.x.ld = x->ld;
        return by_type(x->dtype, [&](auto tx) {
            using X = decltype(tx);
            return few_by_rows<X, Y>(args, st);
        });
    });
}
} // namespace asp
