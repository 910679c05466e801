// The gradient by the stored blocks (asp_block8_gradient).
#include <algorithm>

#include "../../include/asp_b200.h"
#include "block8.h"
#include "block8_device.h"
#include "host/block8_plan.hpp"
#include "launch.h"
#include "tcgen05.h"
#include "tensor_map.h"

#include <cooperative_groups.h>

namespace asp
{
namespace
{
using namespace block8;

// dA_b[r][c] = sum over t of dy[t][128 R + r] x[t][128 C + c], for the stored blocks b = (R, C) only.
//
// The sum runs over the rows t, in which the scales of x differ from row to row, so they cannot be the products' scales: x is unfolded to the
// 16-bit type of dy, exactly, and multiplied in that type. Both factors lie in memory with r and c side by side, which
// tcgen05.mma takes as it is (columns of k). D's lanes are c, so that a warp stores 128 bytes in a row of a block.
//
// What bounds it is shared memory, 128 bytes a clock and SM: for 64 rows t, x of a block column passes it four times (8 KB in, 8 out, unfolded 16 in and
// with each product 16 out), dy of a block row twice and more. Two blocks of a column share x: 56 KB a block instead of 80 for one alone, 448 clocks
// where the products take 256. (Four would be 384, but leave no room for a second D: measured the same, with the rows below in one sum.) A quarter of
// 4096 x 4096 by 4096 rows in bf16: 42.6 us, 806 TFLOP/s; of 8192 x 4096 by 8192: 164 us, 838 TFLOP/s, and 187 in a training step, at the power limit.
//
// Tensor cores cut off what they add up to, which over 8192 rows in one sum showed as 6.5e-6 of the result, where sums that are rounded have 6e-7. So D takes
// 1280 rows in bf16 (8e-7), 768 in fp16, whose products have more bits (8e-7; 1.4e-6 with 1280), then another one the next, while the first is added,
// rounded, to the sum of those before: in tensor memory where a group is one block, by L2 where it is two (12 % of the time for 8192
// rows). A CTA per SM goes through the groups. Where there are few of them a cluster shares the
// rows of one; its CTAs then add to the result one after the other, each beginning with another part of it: the same order, and bits, every time.
//
// 8 bits round up: the largest numbers of either 16-bit type become 256 times the largest scale, 2^16 or 2^128, which the type does not have. Rows with that scale
// are unfolded to half of what they are, and a CTA that has met some adds the other half when it is done with its groups (add_halves). (A second pass of such steps through
// the tensor cores has the issuing warp look at each step whether there are any, between two waits: 48.1 us instead of 45.4 for 243 blocks of 4096 x 4096 and 4096 rows, without any.)
//
// Warp 0 copies, warp 1 issues products, warps 4 to 11 add up and store, warps 12 to 19 and 20 to 27 unfold x, every second step each.
constexpr unsigned kRows = host::kBlock8GradientRows; // t a step
constexpr unsigned kTile = kRows * 128; // bytes of 64 columns of a step's rows in 16 bits, of 128 in 8
constexpr unsigned kRoom = 8, kBlockBytes = 2 * kTile;        // dy: blocks of a step's rows, as many steps as fit
constexpr unsigned kHeld = 4, kHeldBytes = kTile + 1024;      // x in 8 bits, and its scales
// A place for x belongs to one of the two groups that unfold it. Were it to change hands, the group that is two steps ahead might look for the second of two
// copies to a place before the first has arrived (they may overtake one another), and take the one before both, of the same parity, for it.
static_assert(kHeld % 2 == 0, "places for x are shared out between two groups of warps");
constexpr unsigned kUnfolded = 3, kUnfoldedBytes = 2 * kTile; // x in 16 bits: 64 columns after 64 columns, a row t 128 bytes
constexpr unsigned kThreads = 896;
constexpr size_t kSharedBytes = kRoom * kBlockBytes + kUnfolded * kUnfoldedBytes + kHeld * kHeldBytes + 1024;
// Rows of dy that are not all on 16-byte boundaries cannot be copied by tiles. The warps that unfold x bring them, one of their steps ahead, in the aligned
// pieces of 16 bytes that they lie in, and shift them to where they belong: 4001 rows, a quarter of 4001 x 4003, take 125 us (450 element by
// element) where 4096 rows of 4096 x 4096 take 43 by tiles. They then take a part of dy's room, and groups are single blocks.
constexpr unsigned kPitch = 272, kRawBytes = kRows * kPitch, kShiftedStages = 3; // 17 pieces a row
static_assert(kShiftedStages * kBlockBytes + 4 * kRawBytes <= kRoom * kBlockBytes, "two steps of each group of warps beside the stages");

struct GradientArgs
{
    Rows8Dev x;
    const Block8Group *list;
    unsigned n_groups, most;
    const void *dy;
    uint64_t ld;
    float *out;
    unsigned n_rows, n_cols;
    unsigned split;  // CTAs that share the rows of a group
    unsigned stages; // of dy
    bool direct; // dy can be copied by tiles
    bool accumulate;
    unsigned *fault;
};

struct Shared
{
    uint64_t full[kRoom], empty[kRoom], held[kHeld], read[kHeld], unfolded[kUnfolded], used[kUnfolded], done[2], taken[2];
    unsigned tensor, gave_up;
    unsigned halved; // some rows were unfolded to half of what they are
};

// 16 elements in 8 bits times a row's power of two: eight words of two elements.
struct Unfold16 // to fp16: in two factors, since the power may be below what fp16 has (the product is not, as x was fp16)
{
    static constexpr bool bf16 = false;
    using Type = __half;
    static constexpr unsigned round = 768 / kRows; // steps a sum
    static constexpr unsigned largest = 127 + 8;   // scale of what exceeds 57344: 256 times it is 2^16
    static __device__ __forceinline__ void words(uint4 q, unsigned scale, unsigned *out)
    {
        scale = min(scale, largest - 1);
        const int k1 = max((int)scale, 127 - 14);
        const __half2 f1 = __float2half2_rn(power((unsigned)k1)), f2 = __float2half2_rn(power((unsigned)((int)scale - k1 + 127)));
        const unsigned in[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 8; i++)
        {
            const __half2 v = __hmul2(__hmul2(unpack2(in[i / 2] >> 16 * (i % 2) & 0xffffu), f1), f2);
            out[i] = *reinterpret_cast<const unsigned *>(&v);
        }
    }
};
// To bf16, whose exponent has 8 bits where e4m3 has 4: with exponent and fraction put where bf16 has them a number is 2^-120 of what it was (subnormal
// ones included), and one product sets that right together with the scale. Integer instructions, of which an SM does half as many a clock, bound this:
// 5 for four elements, since the even and the odd bytes stay together as they lie in the word (elements 0, 2 and 1, 3 of four: D's
// lanes are told apart when they are stored). NaN, which e4m3 writes as its largest number, is lost that way and put back.
struct UnfoldB16
{
    static constexpr bool bf16 = true;
    using Type = __nv_bfloat16;
    static constexpr unsigned round = 1280 / kRows;
    static constexpr unsigned largest = 127 + 120;
    static __device__ __forceinline__ void words(uint4 q, unsigned scale, unsigned *out)
    {
        const unsigned in[4] = {q.x, q.y, q.z, q.w};
        const unsigned f = (min(scale + 120, 254u) << 7) * 0x10001u; // 2^(scale - 127 + 120); what is missing of scales above 2^7 follows
        unsigned nan = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            const unsigned w = in[i];
            nan |= (w & 0x7f7f7f7fu) + 0x01010101u;
            out[2 * i] = product((w << 4 & 0x07f007f0u) | (w << 8 & 0x80008000u), f);
            out[2 * i + 1] = product((w >> 4 & 0x07f007f0u) | (w & 0x80008000u), f);
        }
        if (scale + 120 > 254)
#pragma unroll
            for (int i = 0; i < 8; i++) out[i] = product(out[i], ((min(scale, largest - 1) + 120 - 254 + 127) << 7) * 0x10001u);
        if (nan & 0x80808080u)
#pragma unroll
            for (int i = 0; i < 16; i++)
                if ((in[i / 4] >> 8 * (i % 4) & 0x7f) == 0x7f) out[i / 4 * 2 + i % 2] |= 0x7fffu << 16 * (i % 4 / 2);
    }
    static __device__ __forceinline__ unsigned product(unsigned a, unsigned b)
    {
        unsigned r;
        asm("mul.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
// the column of a block that D's lane has
template <class Unfold> __device__ __forceinline__ unsigned column_of(unsigned lane) { return Unfold::bf16 && (lane % 4 == 1 || lane % 4 == 2) ? lane ^ 3 : lane; }

// Where a lane's part of a group's blocks goes
struct Places
{
    float *to[2];     // element (0, c) of each block
    unsigned rows[2]; // of them inside the matrix; 0: the column is not
};
template <class Unfold> __device__ __forceinline__ Places places(const GradientArgs &p, const Block8Group &group, unsigned quarter, unsigned lane)
{
    const unsigned c = quarter * 32 + column_of<Unfold>(lane);
    Places at = {};
#pragma unroll
    for (unsigned k = 0; k < 2; k++)
        if (k < group.n)
        {
            at.to[k] = p.out + (uint64_t)group.block[k] * 16384 + c;
            at.rows[k] = group.col * 128 + c < p.n_cols ? min(128u, p.n_rows - group.row[k] * 128) : 0;
        }
    return at;
}
// 16 columns of D (r, block after block) from c on, a quarter of its lanes
__device__ __forceinline__ void store_columns(const Places &at, const float *v, unsigned c, bool add)
{
    const unsigned r0 = c % 128, rows = c < 128 ? at.rows[0] : at.rows[1];
    float *to = (c < 128 ? at.to[0] : at.to[1]) + r0 * 128;
    if (add)
    {
        // By L2, without waiting; one thread's additions to a place stay in order. L2 takes numbers below 2^-126 for zero; read, added and written here they would
        // stay, and 243 blocks of 4096 x 4096 and 4096 rows would take 51.6 us instead of 45.4, 300 rows added to 1024 blocks 43 instead of 24.
#pragma unroll
        for (unsigned k = 0; k < 16; k++)
            if (r0 + k < rows) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(to + k * 128), "f"(v[k]) : "memory");
    }
    else
    {
#pragma unroll
        for (unsigned k = 0; k < 16; k++) __stcg(to + k * 128, r0 + k < rows ? v[k] : 0.f); // zero outside the matrix
    }
}

// The other half of the rows with the largest scale, to the result of a group, by the whole CTA: 32 such rows at a time come to shared memory as 32-bit numbers, and a
// thread multiplies and adds for 4 columns of every 28th row of a block, in the order of the rows: the same bits every time.
// 243 blocks of 4096 x 4096 and 4096 rows: 45.4 us without such rows (44.2 without the test for them and the votes of waits), 65 with one, 89 with 64 in one block column, 1640 where all are in one.
constexpr unsigned kWarps = kThreads / 32, kHalvesAtOnce = 32;
struct Halves
{
    unsigned found[kWarps][4]; // 128 rows of x each: those with the largest scale, a bit each
    unsigned rows[kWarps * 128];
    float x[kHalvesAtOnce][128], dy[kHalvesAtOnce][128];
};
static_assert(sizeof(Halves) <= kRoom * kBlockBytes, "where dy was");
template <class Unfold> __device__ __noinline__ void add_halves(const GradientArgs &p, unsigned u, unsigned t0, unsigned t1, Halves &sh)
{
    constexpr unsigned per = (128 + kWarps - 1) / kWarps;
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const typename Unfold::Type *dy = reinterpret_cast<const typename Unfold::Type *>(p.dy);
    const unsigned col = p.list[u].col, n = p.list[u].n;
    for (unsigned k = 0; k < n; k++)
    {
        const unsigned r0 = p.list[u].row[k] * 128, inside = min(128u, p.n_rows - r0);
        float sum[per][4] = {};
        bool some = false;
        for (unsigned part = t0 / 128 * 128; part < t1; part += kWarps * 128)
        {
            // a warp's scales: row 32 i + lane in word i (scale_at)
            const unsigned t = part + warp * 128;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (t < t1) w = *reinterpret_cast<const uint4 *>(p.x.scales + scale_at(p.x, t + lane, col / 4 * 4));
            const unsigned words[4] = {w.x, w.y, w.z, w.w};
            unsigned mine[4];
#pragma unroll
            for (unsigned i = 0; i < 4; i++)
            {
                const unsigned at = t + 32 * i + lane;
                mine[i] = __ballot_sync(~0u, at >= t0 && at < t1 && (words[i] >> col % 4 * 8 & 0xff) == Unfold::largest);
                if (lane == i) sh.found[warp][i] = mine[i];
            }
            __syncthreads();
            unsigned before = 0, all = 0;
            if (lane < kWarps)
                for (unsigned i = 0; i < 4; i++) all += __popc(sh.found[lane][i]);
            before = __reduce_add_sync(~0u, lane < warp ? all : 0);
            all = __reduce_add_sync(~0u, all);
            if (all == 0) // (the same for all of the CTA)
            {
                __syncthreads();
                continue;
            }
            some = true;
#pragma unroll
            for (unsigned i = 0; i < 4; i++)
            {
                if (mine[i] >> lane & 1) sh.rows[before + __popc(mine[i] & ((1u << lane) - 1))] = t + 32 * i + lane;
                before += __popc(mine[i]);
            }
            __syncthreads();
            for (unsigned first = 0; first < all; first += kHalvesAtOnce)
            {
                const unsigned rows = min(kHalvesAtOnce, all - first);
                for (unsigned i = threadIdx.x; i < rows * 32; i += kThreads)
                {
                    float v[4];
                    unpack4(*reinterpret_cast<const unsigned *>(p.x.values + sh.rows[first + i / 32] * p.x.ld + col * 128 + i % 32 * 4), v);
                    const float scale = power(Unfold::largest - 1);
                    *reinterpret_cast<float4 *>(&sh.x[i / 32][i % 32 * 4]) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
                }
                for (unsigned i = threadIdx.x; i < rows * 128; i += kThreads)
                    sh.dy[i / 128][i % 128] = i % 128 < inside ? to_float(dy[sh.rows[first + i / 128] * p.ld + r0 + i % 128]) : 0.f;
                __syncthreads();
                for (unsigned i = 0; i < rows; i++)
                {
                    const float4 x = *reinterpret_cast<const float4 *>(&sh.x[i][4 * lane]);
#pragma unroll
                    for (unsigned j = 0; j < per; j++)
                    {
                        const float v = sh.dy[i][min(warp + j * kWarps, 127u)];
                        sum[j][0] = __fmaf_rn(v, x.x, sum[j][0]), sum[j][1] = __fmaf_rn(v, x.y, sum[j][1]);
                        sum[j][2] = __fmaf_rn(v, x.z, sum[j][2]), sum[j][3] = __fmaf_rn(v, x.w, sum[j][3]);
                    }
                }
                __syncthreads();
            }
        }
        if (!some) continue;
#pragma unroll
        for (unsigned j = 0; j < per; j++)
        {
            const unsigned r = warp + j * kWarps;
            float *to = p.out + (uint64_t)p.list[u].block[k] * 16384 + r * 128 + 4 * lane;
#pragma unroll
            for (unsigned i = 0; i < 4; i++)
                if (r < inside && col * 128 + 4 * lane + i < p.n_cols) __stcg(to + i, __ldcg(to + i) + sum[j][i]);
        }
    }
}

template <class Unfold>
__global__ void __launch_bounds__(kThreads, 1) k_block8_gradient(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ GradientArgs p)
{
    namespace cg = cooperative_groups;
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char *dys = raw + (1024 - tc::shared_address(raw) % 1024) % 1024;
    unsigned char *halves = dys + kRoom * kBlockBytes, *bytes = halves + kUnfolded * kUnfoldedBytes;
    const unsigned warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned piece = blockIdx.x % p.split, u0 = blockIdx.x / p.split, stride = gridDim.x / p.split;
    const unsigned steps = (p.x.n + kRows - 1) / kRows, step0 = (unsigned)((uint64_t)steps * piece / p.split), step1 = (unsigned)((uint64_t)steps * (piece + 1) / p.split);
    const unsigned width_d = p.most * 128; // two Ds, and the sum of a single block behind them
    if (threadIdx.x == 32)
    {
        tc::prefetch_map(&map_x);
        if (p.direct) tc::prefetch_map(&map_dy);
    }
    if (threadIdx.x == 0)
    {
        for (unsigned i = 0; i < p.stages; i++) tc::barrier_init(&sh.full[i], 1), tc::barrier_init(&sh.empty[i], 1);
        for (unsigned i = 0; i < kHeld; i++) tc::barrier_init(&sh.held[i], 1), tc::barrier_init(&sh.read[i], 8);
        for (unsigned i = 0; i < kUnfolded; i++) tc::barrier_init(&sh.unfolded[i], 8), tc::barrier_init(&sh.used[i], 1);
        for (unsigned i = 0; i < 2; i++) tc::barrier_init(&sh.done[i], 1), tc::barrier_init(&sh.taken[i], 8);
        sh.gave_up = sh.halved = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) tc::tensor_alloc(&sh.tensor, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tensor = sh.tensor;
    const Block8Group first = p.list[u0];
    grid_wait();
    grid_release();

    if (warp == 0)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0, x = 0, x_phase = 0;
            for (unsigned u = u0; u < p.n_groups; u += stride)
            {
                const Block8Group group = u == u0 ? first : p.list[u];
                const unsigned blocks = group.n, col = group.col;
                for (unsigned i = step0; i < step1; i++)
                {
                    const int t = (int)(i * kRows);
                    if (!tc::barrier_wait(&sh.read[x], x_phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = bytes + x * kHeldBytes;
                    tc::barrier_expect(&sh.held[x], kTile + 512);
                    tc::copy_tile(to, &map_x, (int)(col * 128), t, &sh.held[x]);
                    tc::copy_bytes(to + kTile, p.x.scales + ((uint64_t)(col / 4) * p.x.pieces + t / 128) * 512, 512, &sh.held[x]);
                    if (++x == kHeld) x = 0, x_phase ^= 1;
                    if (!p.direct) continue;
                    if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                    tc::barrier_expect(&sh.full[s], blocks * kBlockBytes);
                    to = dys + s * p.most * kBlockBytes;
#pragma unroll
                    for (unsigned k = 0; k < 2; k++)
                        if (k < blocks)
                        {
                            tc::copy_tile(to + k * kBlockBytes, &map_dy, (int)group.row[k] * 128, t, &sh.full[s]);
                            tc::copy_tile(to + k * kBlockBytes + kTile, &map_dy, (int)group.row[k] * 128 + 64, t, &sh.full[s]);
                        }
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
            }
        }
    }
    else if (warp == 1)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0, h = 0, h_phase = 0, d = 0, d_phase = 0;
            for (unsigned u = u0; u < p.n_groups; u += stride)
            {
                const unsigned shape = tc::halves(128 * (u == u0 ? first.n : p.list[u].n), Unfold::bf16);
                for (unsigned i = step0, left = 0; i < step1; i++)
                {
                    const bool fresh = left == 0;
                    if (fresh)
                    {
                        if (!tc::barrier_wait(&sh.taken[d], d_phase ^ 1, &sh.gave_up)) goto end;
                        left = Unfold::round;
                    }
                    if (p.direct && !tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) goto end;
                    if (!tc::barrier_wait(&sh.unfolded[h], h_phase, &sh.gave_up)) goto end;
                    tc::fence_after();
                    const unsigned x = tc::shared_address(halves + h * kUnfoldedBytes), dy = tc::shared_address(dys + s * p.most * kBlockBytes);
#pragma unroll
                    for (unsigned k = 0; k < kRows / 16; k++) // 16 rows of 128 bytes on
                        tc::mma_halves(tensor + d * width_d, tc::columns_of_k(x + 2048 * k, kTile), tc::columns_of_k(dy + 2048 * k, kTile), shape, !fresh || k > 0);
                    tc::commit(&sh.empty[s]);
                    tc::commit(&sh.used[h]);
                    if (++s == p.stages) s = 0, phase ^= 1;
                    if (++h == kUnfolded) h = 0, h_phase ^= 1;
                    if (--left == 0 || i + 1 == step1)
                    {
                        tc::commit(&sh.done[d]);
                        left = 0;
                        d ^= 1;
                        if (d == 0) d_phase ^= 1;
                    }
                }
            }
        }
    }
    else if (warp >= 12)
    {
        // 8 lanes and 16 columns a lane to a row t: 4 rows a warp at once, warp w rows 4 w on, then 32 rows further
        const unsigned lane8 = lane % 8, w = (warp - 12) % 8, row0 = w * 4 + lane / 8, mine = (warp - 12) / 8;
        unsigned s = 0, phase = 0, x = 0, x_phase = 0, h = 0, h_phase = 0, turn = 0, parity = 0;
        // Rows of dy that begin anywhere: a thread has piece j of rows 2 w + lane / 16 + 16 k of a step, which all lie the same number of bytes behind a boundary,
        // in all steps.
        const unsigned j = lane % 16, row_dy = 2 * w + lane / 16;
        unsigned char *raws = dys + kShiftedStages * kBlockBytes + mine * 2 * kRawBytes + row_dy * kPitch + 16 * j;
        const uintptr_t lo = (uintptr_t)p.dy, hi = lo + ((uint64_t)(p.x.n - 1) * p.ld + p.n_rows) * 2; // dy
        const unsigned offset = (unsigned)(lo + row_dy * p.ld * 2) & 15u; // (128 r more elements change nothing)
        const auto settle = [&](unsigned &u, unsigned &i) { // step i of the rows, or as much further on in the groups after this one
            while (u < p.n_groups && i >= step1) i -= step1 - step0, u += stride;
        };
        const auto ask = [&](unsigned u, unsigned i, unsigned to) {
            if (u < p.n_groups)
            {
                const unsigned r0 = p.list[u].row[0] * 128;
                const uintptr_t at = lo + (((uint64_t)i * kRows + row_dy) * p.ld + r0) * 2 - offset + 16 * j, far = 32 * p.ld;
                unsigned char *piece = raws + to * kRawBytes;
                if (i > 0 && lo + (((uint64_t)i * kRows + kRows - 1) * p.ld + r0) * 2 + kPitch <= hi) // all of the step's pieces are in dy
                {
#pragma unroll
                    for (unsigned k = 0; k < 4; k++)
                    {
                        copy16(piece + k * 16 * kPitch, reinterpret_cast<const void *>(at + k * far));
                        if (j == 15) copy16(piece + k * 16 * kPitch + 16, reinterpret_cast<const void *>(at + k * far + 16));
                    }
                }
                else
                    for (unsigned k = 0; k < 4; k++)
                        for (unsigned e = 0; e < (j == 15 ? 2 : 1); e++)
                            *reinterpret_cast<uint4 *>(piece + k * 16 * kPitch + e * 16) =
                                i * kRows + row_dy + 16 * k < p.x.n ? load_piece<__half>(at + k * far + e * 16, lo, hi) : make_uint4(0, 0, 0, 0);
            }
            copies_are_one_group();
        };
        if (!p.direct)
        {
            unsigned first_u = u0, first_i = step0 + mine;
            settle(first_u, first_i);
            ask(first_u, first_i, 0);
        }
        for (unsigned u = u0; u < p.n_groups; u += stride)
        {
            const unsigned byte = (u == u0 ? first.col : p.list[u].col) % 4, row = u == u0 ? first.row[0] : p.list[u].row[0];
            for (unsigned i = step0; i < step1; i++)
            {
                if (turn == mine)
                {
                    if (!tc::warp_wait(&sh.held[x], x_phase, &sh.gave_up)) goto end;
                    const unsigned char *from = bytes + x * kHeldBytes;
                    uint4 q[2];
                    unsigned scale[2];
#pragma unroll
                    for (unsigned n = 0; n < 2; n++)
                    {
                        const unsigned t = row0 + 32 * n, at = i * kRows + t;
                        q[n] = *reinterpret_cast<const uint4 *>(from + t * 128 + 16 * lane8);
                        scale[n] = at < p.x.n ? from[kTile + row0 * 16 + at / 32 % 4 * 4 + byte] : 127; // (rows behind the last one are zeros, with any scale)
                    }
                    // The next copy may come while these are unfolded. Reads and copies are of different proxies: without the fence a copy overtook reads that
                    // other kernels' warps held up.
                    tc::fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tc::barrier_arrive(&sh.read[x]);
                    unsigned v[2][8]; // (in front of the wait, which votes)
#pragma unroll
                    for (unsigned n = 0; n < 2; n++) Unfold::words(q[n], scale[n], v[n]);
                    if (!tc::warp_wait(&sh.used[h], h_phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = halves + h * kUnfoldedBytes + lane8 / 4 * kTile;
#pragma unroll
                    for (unsigned n = 0; n < 2; n++)
                    {
                        const unsigned t = row0 + 32 * n;
                        // 16-byte pieces 2 l and 2 l + 1 of the row's 128 bytes, swapped in the second half so that eight lanes meet no conflict
                        unsigned char *line = to + t * 128;
                        const unsigned at = lane8 % 4 * 2, second = lane8 / 4;
                        const uint4 lo = make_uint4(v[n][0], v[n][1], v[n][2], v[n][3]), hi = make_uint4(v[n][4], v[n][5], v[n][6], v[n][7]);
                        *reinterpret_cast<uint4 *>(line + (((at + second) ^ (t % 8)) * 16)) = second ? hi : lo;
                        *reinterpret_cast<uint4 *>(line + (((at + 1 - second) ^ (t % 8)) * 16)) = second ? lo : hi;
                    }
                    if (!p.direct)
                    {
                        unsigned next_u = u, next_i = i + 2;
                        settle(next_u, next_i);
                        __syncwarp(); // (the lanes beside have read what is copied to)
                        ask(next_u, next_i, parity ^ 1);
                        wait_for_all_groups_but<1>();
                        __syncwarp();
                        if (!tc::warp_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                        const int columns = (int)(p.n_rows - row * 128) - (int)(8 * j); // of the piece, that are in the matrix
#pragma unroll
                        for (unsigned k = 0; k < 4; k++)
                        {
                            const unsigned t = row_dy + 16 * k;
                            const uint4 *piece = reinterpret_cast<const uint4 *>(raws + parity * kRawBytes + k * 16 * kPitch);
                            uint4 v = shifted(piece[0], piece[1], offset / 4, offset % 4 * 8);
                            if (columns < 8)
                            {
                                const auto keep = [&](unsigned word, int e) { return columns > e + 1 ? word : columns > e ? word & 0xffffu : 0u; };
                                v = make_uint4(keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6));
                            }
                            *reinterpret_cast<uint4 *>(dys + s * kBlockBytes + j / 8 * kTile + t * 128 + ((j % 8) ^ (t % 8)) * 16) = v;
                        }
                        parity ^= 1;
                    }
                    tc::fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tc::barrier_arrive(&sh.unfolded[h]);
                    if (max(scale[0], scale[1]) == Unfold::largest) sh.halved = 1;
                }
                turn ^= 1;
                if (++s == p.stages) s = 0, phase ^= 1;
                if (++x == kHeld) x = 0, x_phase ^= 1;
                if (++h == kUnfolded) h = 0, h_phase ^= 1;
            }
        }
    }
    else if (warp >= 4)
    {
        // two warps to a quarter of D's lanes, every second 16 columns each
        unsigned d = 0, d_phase = 0;
        const unsigned quarter = warp % 4, mine = (warp - 4) / 4 * 16;
        for (unsigned u = u0; u < p.n_groups; u += stride)
        {
            const Block8Group group = u == u0 ? first : p.list[u];
            const unsigned blocks = group.n;
            const Places at = places<Unfold>(p, group, quarter, lane);
            for (unsigned i = step0; i < step1; i += Unfold::round)
            {
                if (!tc::warp_wait<64>(&sh.done[d], d_phase, &sh.gave_up)) goto end;
                tc::fence_after();
                const bool last = i + Unfold::round >= step1 && p.split == 1;
                for (unsigned c = mine; c < blocks * 128; c += 32)
                {
                    float v[16];
                    tc::tensor_load16(tensor + d * width_d + c + (quarter * 32 << 16), v);
                    if (p.most == 2) store_columns(at, v, c, p.accumulate || i > step0);
                    else
                    {
                        const unsigned sum = tensor + 256 + c + (quarter * 32 << 16);
                        if (i > step0)
                        {
                            float o[16];
                            tc::tensor_load16(sum, o);
#pragma unroll
                            for (int k = 0; k < 16; k++) v[k] += o[k];
                        }
                        if (last) store_columns(at, v, c, p.accumulate);
                        else tc::tensor_store16(sum, v);
                    }
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::barrier_arrive(&sh.taken[d]);
                d ^= 1;
                if (d == 0) d_phase ^= 1;
            }
        }
    }
end:
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    // A cluster (and a block each): the sum's columns in `split` parts of 16 to 64; a CTA begins with its own. (All CTAs of the cluster go through this
    // together, whatever became of their waits.)
    unsigned some = sh.halved;
    if (p.split > 1)
    {
        const Places at = places<Unfold>(p, first, warp % 4, lane);
        const unsigned width = 128 / p.split;
        for (unsigned turn = 0; turn < p.split; turn++)
        {
            const unsigned part = (piece + turn) % p.split, c = part * width + (warp - 4) / 4 * 16;
            if (warp >= 4 && c < (part + 1) * width && !sh.gave_up)
            {
                float v[16];
                tc::tensor_load16(tensor + 256 + c + (warp % 4 * 32 << 16), v);
                store_columns(at, v, c, p.accumulate || turn > 0);
            }
            cg::this_cluster().sync();
            if (turn == 0 && lane < p.split) some |= *cg::this_cluster().map_shared_rank(&sh.halved, lane); // (there is another turn: its shared memory stays)
        }
    }
    const bool any = __any_sync(~0u, some != 0); // (the same for all CTAs of a cluster)
    for (unsigned turn = 0; turn < p.split && any; turn++)
    {
        if (turn == piece && !sh.gave_up)
            for (unsigned u = u0; u < p.n_groups; u += stride) add_halves<Unfold>(p, u, step0 * kRows, min(step1 * kRows, p.x.n), *reinterpret_cast<Halves *>(dys));
        if (p.split > 1) cg::this_cluster().sync();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (sh.gave_up)
    {
        // copies and products in flight end by themselves; their memory is kept until then
        const uint64_t since = tc::now_ns();
        while (tc::now_ns() - since < 10000000ull) __nanosleep(1000);
        if (threadIdx.x == 0 && p.fault) *reinterpret_cast<volatile unsigned *>(p.fault) = 1;
    }
    if (warp == 1) tc::tensor_free(tensor, 512);
}

template <class Unfold> cudaError_t gradient(const CUtensorMap &map_dy, const CUtensorMap &map_x, const GradientArgs &p, int sm_count, cudaStream_t st)
{
    static SharedAllowance allowance;
    const cudaError_t e = allowance.need((const void *)k_block8_gradient<Unfold>, (int)kSharedBytes);
    if (e != cudaSuccess) return e;
    const unsigned grid = p.split > 1 ? p.n_groups * p.split : std::min<unsigned>(p.n_groups, (unsigned)sm_count);
    return launch_pdl_cluster(k_block8_gradient<Unfold>, p.split, dim3(grid), dim3(kThreads), kSharedBytes, st, map_dy, map_x, p);
}

} // namespace

cudaError_t launch_block8_gradient(const Block8Dev &a, const Block8Groups &groups, const Rows8Dev &x, const Dense &dy, float *out, bool accumulate, int sm_count, unsigned *fault, cudaStream_t st)
{
    if (a.n_blocks == 0) return cudaSuccess;
    if (x.n == 0) return accumulate ? cudaSuccess : cudaMemsetAsync(out, 0, (size_t)a.n_blocks * 16384 * sizeof(float), st);
    GradientArgs p = {};
    const bool direct = ((uintptr_t)dy.p & 15) == 0 && dy.ld % 8 == 0 && dy.ld < 1ull << 38; // (a tile map's distances are below 2^40 bytes)
    static SharedAllowance allowance;
    static ClusterRoom room;
    unsigned fit[9];
    const void *any = (const void *)k_block8_gradient<UnfoldB16>; // (of both types, one CTA fits an SM)
    cudaError_t e = allowance.need(any, (int)kSharedBytes);
    if (e == cudaSuccess) e = room.most(any, kThreads, kSharedBytes, fit);
    if (e != cudaSuccess) return e;
    const host::Block8GradientPlan plan = host::block8_gradient_plan(a.n_blocks, direct ? groups.twos : 0, x.n, sm_count, fit);
    p.most = plan.most, p.split = plan.split;
    p.x = x, p.list = groups.groups[p.most - 1], p.n_groups = groups.count[p.most - 1];
    p.dy = dy.p, p.ld = dy.ld, p.out = out, p.accumulate = accumulate, p.fault = fault;
    p.n_rows = a.n_rows, p.n_cols = a.n_cols;
    p.stages = direct ? kRoom / p.most : kShiftedStages;
    p.direct = direct;
    CUtensorMap map_dy, map_x;
    e = byte_map(&map_x, x.values, x.ld, x.n, x.ld, kRows, false); // as it lies, without swizzle
    if (e == cudaSuccess && p.direct)
        e = tensor_map(&map_dy, dy.dtype == ASP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dy.p, a.n_rows, x.n, dy.ld * 2, 64, kRows);
    else map_dy = map_x; // (not used)
    if (e != cudaSuccess) return e;
    if (dy.dtype == ASP_BF16) return gradient<UnfoldB16>(map_dy, map_x, p, sm_count, st);
    return gradient<Unfold16>(map_dy, map_x, p, sm_count, st);
}
} // namespace asp
