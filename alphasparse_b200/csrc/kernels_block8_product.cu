// Products of block-sparse 8-bit matrices with many rows in 8 bits (asp_block8_product).
#include <math.h>

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

// Y[t][128 R + r] = sum over the blocks j of block row R of 2^(kA_j) sum over c of A_j[r][c] * 2^(kX_{t, c_j}) X_{t, c_j}[c].
//
// A tile is 128 rows of A by up to 192 rows of X: D[128][192] in tensor memory, a block of A (16 KB) and the same 128 columns of X (24 KB) a
// step, four tcgen05.mma of 32 columns each. The powers of two go into the products as their scales (a byte per row of the block and per row of X), so sums
// over blocks of different scales stay in tensor memory, in 32 bits. A's rows are the
// rows of D because a block is 128 rows of A whatever the pattern, while X can be cut anywhere; 192 since two tiles' sums (384
// columns) and the scales (24) then share the 512 columns, so that a tile is stored under the next one's products, and whole 64s since the
// scales of X begin at every second column.
//
// Where there are fewer tiles than SMs, a cluster shares the blocks of a tile; its CTAs put their sums into shared memory and add them up in order,
// some columns each.
//
// What bounds it is shared memory, 128 bytes a clock and SM: a step writes 40 KB to it and the products read 40 KB, 640 clocks where the products alone
// take 384. Rows, columns and rows of X, share of blocks stored: 8192, 8192, 8192, half: 256 us, 2.15 PFLOP/s in a burst; called over and over the chip comes to its
// power limit and 1.28 GHz, and it takes 293. 4096, 4096, 2048, a quarter: 15.6 us, 1.10 PFLOP/s (352 tiles of unequal length over 148 SMs: 16,000 clocks of steps in
// the longest CTA, 12,200 on average, and each CTA's first copies and last stores).
//
// A CTA per SM goes through tiles: warp 0 copies blocks, rows and their scales, warp 1 issues products, warps 2 to 17 store.
constexpr unsigned kMostRows = host::kBlock8ProductRows;
constexpr unsigned kStages = 8; // at most
// Tensor cores cut off what they add up to: 64 blocks (8192 columns) in one sum were 3.0e-6 off, 16 are 6e-7, where sums rounded in 32 bits are 4e-7. Results in
// 32 bits therefore take sums of 16 blocks, in one D and the other, added up, rounded, in the registers of the warps that store (2048 rows by 4096 x 8192: 70.4 us instead
// of 68.3; added up by L2 where the result is: 83). In 16 bits, which lose 2^-9 or 2^-12 at the end, a hundredth of that is enough.
template <class Y> constexpr unsigned kRound = sizeof(Y) == 4 ? host::kBlock8Sum : 256;
constexpr unsigned kScaleBytes = 512 + 1024;
constexpr unsigned kRoom = 221 * 1024; // of shared memory for stages
constexpr unsigned kThreads = 576;

struct ProductArgs
{
    Block8Dev a;
    Rows8Dev x;
    void *y;
    uint64_t ldy;
    unsigned tile;   // rows of X a tile, a multiple of 64
    unsigned tiles_x, wide;
    unsigned n_tiles;
    unsigned split;  // CTAs that share a tile's blocks; then a CTA has one tile
    unsigned stages, stage_bytes;
    bool pairs;      // two 16-bit elements of y at a time
    unsigned *fault;
};

struct Shared
{
    uint64_t full[kStages], empty[kStages], done[2], taken[2];
    unsigned tensor, gave_up;
};

// The steps of a CTA, in order: the blocks of its tiles. Tiles are in the order of their block rows, longest first, and handed out to the CTAs forwards and backwards in
// turn, so that who has a long one gets a short one next (a quarter of 4096 x 4096 by 2048 rows, where eight warps stored: 17.8 us, 19.1 with block rows side by side and always
// forwards). What a CTA has to know of a tile is asked for a tile ahead (17.8 to 17.0 us).
// Where X is larger than a part of L2 it is gone through in parts of `wide` tiles, each with all block rows.
struct Steps
{
    const ProductArgs &p;
    bool valid;
    unsigned j, end, row, t0;
    __device__ __forceinline__ explicit Steps(const ProductArgs &args) : p(args), tile(blockIdx.x / args.split)
    {
        ask();
        next_tile();
    }
    __device__ __forceinline__ void next_tile()
    {
        valid = tile < p.n_tiles;
        if (!valid) return;
        row = next.x, t0 = next_t0;
        const unsigned piece = blockIdx.x % p.split;
        j = next.y + next.z * piece / p.split, end = next.y + next.z * (piece + 1) / p.split; // (less than 2^24 blocks, 8 pieces at most)
        turn++;
        if (turn > p.n_tiles / gridDim.x || p.split > 1) tile = p.n_tiles; // (a cluster has one tile only)
        else tile = turn * gridDim.x + (turn % 2 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        ask();
    }

  private:
    unsigned tile, turn = 0; // of the tile after this one, whose block row is on its way
    uint4 next;
    unsigned next_t0;
    __device__ __forceinline__ void ask()
    {
        if (tile >= p.n_tiles) return;
        const unsigned per = p.wide * p.a.n_block_rows, part = tile / per, in = tile % per, columns = min(p.wide, p.tiles_x - part * p.wide);
        next = p.a.rows[in / columns];
        next_t0 = (part * p.wide + in % columns) * p.tile;
    }
};

// 16 columns of D (rows of Y), 32 of its lanes
template <class Y> __device__ __forceinline__ void store_columns(const float *v, const ProductArgs &p, unsigned row0, unsigned lane, unsigned t0, unsigned limit)
{
    Y *y = reinterpret_cast<Y *>(p.y);
    const unsigned row = row0 + lane;
    if constexpr (sizeof(Y) == 2)
    {
        if (p.pairs)
        {
            // lanes 2 i and 2 i + 1 exchange, so that each has two rows of one column: 4 bytes
            const bool odd = lane & 1;
            Y *to = y + (uint64_t)(t0 + odd) * p.ldy + (row & ~1u);
            const bool both = (row & ~1u) + 1 < p.a.n_rows, one = (row & ~1u) < p.a.n_rows;
#pragma unroll
            for (int c = 0; c < 16; c += 2)
            {
                const float got = __shfl_xor_sync(~0u, odd ? v[c] : v[c + 1], 1);
                const Y lo = from_float<Y>(odd ? got : v[c]), hi = from_float<Y>(odd ? v[c + 1] : got);
                if (t0 + c + odd < limit)
                {
                    if (both)
                    {
                        Y two[2] = {lo, hi};
                        *reinterpret_cast<unsigned *>(to) = *reinterpret_cast<unsigned *>(two);
                    }
                    else if (one) *to = lo;
                }
                to += 2 * p.ldy;
            }
            return;
        }
    }
    if (row >= p.a.n_rows) return;
#pragma unroll
    for (int c = 0; c < 16; c++)
        if (t0 + c < limit) y[(uint64_t)(t0 + c) * p.ldy + row] = from_float<Y>(v[c]);
}

template <class Y>
__global__ void __launch_bounds__(kThreads, 1) k_block8_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ ProductArgs p)
{
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char *stages = raw + (1024 - tc::shared_address(raw) % 1024) % 1024;
    const unsigned warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 32) tc::prefetch_map(&map_a), tc::prefetch_map(&map_x);
    if (threadIdx.x == 0)
    {
        for (unsigned i = 0; i < p.stages; i++)
        {
            tc::barrier_init(&sh.full[i], 1);
            tc::barrier_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; i++)
        {
            tc::barrier_init(&sh.done[i], 1);
            tc::barrier_init(&sh.taken[i], 16);
        }
        sh.gave_up = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) tc::tensor_alloc(&sh.tensor, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tensor = sh.tensor;
    Steps at(p);
    grid_wait();
    grid_release();
    const unsigned x_bytes = p.tile * 128;

    if (warp == 0)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0;
            for (; at.valid; at.next_tile())
                for (; at.j < at.end; at.j++)
                {
                    const unsigned col = p.a.col[at.j];
                    if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = stages + s * p.stage_bytes;
                    // scales of X: the pieces of 128 rows that have rows of the tile
                    const unsigned piece = at.t0 / 128, pieces = (min(at.t0 + p.tile, p.x.n) + 127) / 128 - piece;
                    tc::barrier_expect(&sh.full[s], 16384 + x_bytes + 512 + pieces * 512);
                    tc::copy_tile(to, &map_a, 0, (int)(at.j * 128), &sh.full[s]);
                    tc::copy_tile(to + 16384, &map_x, (int)(col * 128), (int)at.t0, &sh.full[s]);
                    tc::copy_bytes(to + 16384 + x_bytes, p.a.scale_rows + (uint64_t)at.j * 512, 512, &sh.full[s]);
                    tc::copy_bytes(to + 16384 + x_bytes + 512, p.x.scales + ((uint64_t)(col / 4) * p.x.pieces + piece) * 512, pieces * 512, &sh.full[s]);
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
        }
    }
    else if (warp == 1)
    {
        if (tc::one_lane())
        {
            // A step's copies are waited for under the products of the step before: a look at a barrier takes a hundred clocks and more, and the tensor cores
            // have no more than two or three products waiting.
            unsigned s = 0, phase = 0, b = 0, b_phase = 0, turn = 0;
            bool ready = false;
            for (; at.valid; at.next_tile())
            {
                const unsigned shift = at.t0 % 128 / 32; // (of the first row among its piece's columns)
                while (at.j < at.end)
                {
                    if (!tc::barrier_wait(&sh.taken[b], b_phase ^ 1, &sh.gave_up)) goto end;
                    const unsigned d = tensor + b * kMostRows, last = min(at.end, at.j + kRound<Y>);
                    bool add = false;
                    for (; at.j < last; at.j++)
                    {
                        const unsigned shape = tc::scaled_e4m3(p.tile, p.a.col[at.j] % 4);
                        if (!ready && !tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) goto end;
                        tc::fence_after();
                        const unsigned a = tc::shared_address(stages + s * p.stage_bytes), x = a + 16384, scales = x + x_bytes;
                        const unsigned sa = tensor + 2 * kMostRows + turn * 4, sx = tensor + 2 * kMostRows + 8 + turn * 8;
                        uint64_t *const empty = &sh.empty[s];
                        if (++s == p.stages) s = 0, phase ^= 1;
                        tc::copy_scales(sa, tc::scale_rows(scales));
                        tc::copy_scales(sx, tc::scale_rows(scales + 512));
                        if (shift + p.tile / 32 > 4) tc::copy_scales(sx + 4, tc::scale_rows(scales + 1024));
#pragma unroll
                        for (int k = 0; k < 4; k++)
                        {
                            if (k == 1)
                            {
                                ready = at.j + 1 < at.end;
                                if (ready && !tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) goto end;
                            }
                            tc::mma_scaled(d, tc::rows_k_major(a + 32 * k), tc::rows_k_major(x + 32 * k), shape, sa, sx + shift, add);
                            add = true;
                        }
                        tc::commit(empty);
                        turn ^= 1;
                    }
                    tc::commit(&sh.done[b]);
                    b ^= 1;
                    if (b == 0) b_phase ^= 1;
                }
            }
        }
    }
    else
    {
        unsigned b = 0, b_phase = 0;
        const unsigned quarter = warp % 4, first = (warp - 2) / 4 * 16; // four warps to a quarter of D's lanes, every fourth 16 columns each
        constexpr unsigned most = kMostRows / 64;
        for (; at.valid; at.next_tile())
        {
            const unsigned row0 = at.row * 128 + quarter * 32, limit = min(p.x.n, at.t0 + p.tile);
            float sum[most][16];
#pragma unroll
            for (unsigned k = 0; k < most; k++)
#pragma unroll
                for (int i = 0; i < 16; i++) sum[k][i] = 0.f;
            bool all = true;
            while (at.j < at.end)
            {
                all = tc::warp_wait<64>(&sh.done[b], b_phase, &sh.gave_up);
                if (!all) break;
                tc::fence_after();
#pragma unroll
                for (unsigned k = 0; k < most; k++)
                    if (first + 64 * k < p.tile)
                    {
                        float v[16];
                        tc::tensor_load16(tensor + b * kMostRows + first + 64 * k + (quarter * 32 << 16), v);
#pragma unroll
                        for (int i = 0; i < 16; i++) sum[k][i] += v[i];
                    }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::barrier_arrive(&sh.taken[b]);
                b ^= 1;
                if (b == 0) b_phase ^= 1;
                at.j += min(at.end - at.j, kRound<Y>);
            }
            if (!all) break;
            // a cluster's part goes to shared memory: all blocks have been copied and multiplied, the stages are free
#pragma unroll
            for (unsigned k = 0; k < most; k++)
            {
                const unsigned c = first + 64 * k;
                if (c >= p.tile) break;
                if (p.split == 1) store_columns<Y>(sum[k], p, row0, lane, at.t0 + c, limit);
                else
#pragma unroll
                    for (int i = 0; i < 16; i++) reinterpret_cast<float *>(stages)[(c + i) * 128 + quarter * 32 + lane] = sum[k][i];
            }
        }
    }
end:
    __syncwarp();
    if (p.split > 1) // (all CTAs of the cluster come here, whatever became of their waits)
    {
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        const float *part = reinterpret_cast<const float *>(stages);
        cluster.sync();
        const Steps at(p); // (those that copy and multiply have gone on)
        Y *y = reinterpret_cast<Y *>(p.y);
        const unsigned rows = min(128u, p.a.n_rows - at.row * 128), columns = min(p.tile, p.x.n - at.t0);
        for (unsigned i = threadIdx.x + kThreads * (blockIdx.x % p.split); i < columns * 32; i += kThreads * p.split)
        {
            float4 v[8]; // all on their way before the first is needed
#pragma unroll
            for (unsigned s = 0; s < 8; s++)
                if (s < p.split) v[s] = *cluster.map_shared_rank(reinterpret_cast<const float4 *>(part) + i, s);
            float sum[4] = {};
#pragma unroll
            for (unsigned s = 0; s < 8; s++)
                if (s < p.split) sum[0] += v[s].x, sum[1] += v[s].y, sum[2] += v[s].z, sum[3] += v[s].w;
            const unsigned r = i % 32 * 4;
            Y *to = y + (uint64_t)(at.t0 + i / 32) * p.ldy + at.row * 128 + r;
            if (p.pairs && sizeof(Y) == 2 && r + 4 <= rows)
            {
                Y four[4] = {from_float<Y>(sum[0]), from_float<Y>(sum[1]), from_float<Y>(sum[2]), from_float<Y>(sum[3])};
                reinterpret_cast<unsigned *>(to)[0] = reinterpret_cast<const unsigned *>(four)[0], reinterpret_cast<unsigned *>(to)[1] = reinterpret_cast<const unsigned *>(four)[1];
            }
            else
#pragma unroll
                for (unsigned k = 0; k < 4; k++)
                    if (r + k < rows) to[k] = from_float<Y>(sum[k]);
        }
        cluster.sync(); // (its shared memory is read until here)
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

template <class Y> cudaError_t product(const CUtensorMap &map_a, const CUtensorMap &map_x, const ProductArgs &p, int sm_count, cudaStream_t st)
{
    const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
    static SharedAllowance allowance;
    const cudaError_t e = allowance.need((const void *)k_block8_product<Y>, kRoom + 1024);
    if (e != cudaSuccess) return e;
    const unsigned grid = p.split > 1 ? p.n_tiles * p.split : std::min<unsigned>(p.n_tiles, (unsigned)sm_count);
    return launch_pdl_cluster(k_block8_product<Y>, p.split, dim3(grid), dim3(kThreads), smem, st, map_a, map_x, p);
}
} // namespace

cudaError_t launch_block8_product(const Block8Dev &a, const Rows8Dev &x, const Dense &y, int sm_count, unsigned *fault, cudaStream_t st)
{
    if (x.n == 0) return cudaSuccess;
    ProductArgs p = {};
    p.a = a, p.x = x, p.y = y.p, p.ldy = y.ld, p.fault = fault;
    static SharedAllowance allowance;
    static ClusterRoom room;
    unsigned fit[9];
    const void *any = (const void *)k_block8_product<float>; // (of all types, one CTA fits an SM)
    cudaError_t e = allowance.need(any, kRoom + 1024);
    if (e == cudaSuccess) e = room.most(any, kThreads, kRoom + 1024, fit);
    if (e != cudaSuccess) return e;
    const host::Block8ProductPlan plan = host::block8_product_plan(a.n_block_rows, a.n_blocks, a.longest, x.n, sm_count, fit);
    p.tile = plan.tile, p.split = plan.split;
    p.tiles_x = (x.n + p.tile - 1) / p.tile;
    const uint64_t tiles = (uint64_t)a.n_block_rows * p.tiles_x;
    if (tiles > 0xf0000000u) return cudaErrorInvalidValue; // (2^38 rows of blocks' results and more)
    p.n_tiles = (unsigned)tiles;
    // Tiles of X that are gone through together: all where X stays near in L2, else so many that the tiles that run at the same time have as many bytes of A as of X.
    p.wide = p.tiles_x;
    if (x.n * x.ld > 40ull << 20) // 8192 rows of 8192: 4096 of them, a quarter, 76.3 us in parts and 81.5 without; 8192 rows of 4096 (34 MB) 89 and 88
    {
        const double side = 16384.0 * a.n_blocks / a.n_block_rows / (p.tile * x.ld);
        const unsigned most = std::max(1u, (unsigned)(sqrt(sm_count * side) + 0.5)), parts = (p.tiles_x + most - 1) / most;
        p.wide = (p.tiles_x + parts - 1) / parts;
    }
    p.stage_bytes = (16384 + p.tile * 128 + kScaleBytes + 1023) / 1024 * 1024;
    p.stages = std::min(kStages, kRoom / p.stage_bytes);
    p.pairs = y.dtype != ASP_F32 && ((uintptr_t)y.p & 3) == 0 && y.ld % 2 == 0;
    CUtensorMap map_a, map_x;
    // (a matrix without blocks has nothing to copy: any map does)
    e = byte_map(&map_a, a.values, 128, (uint64_t)std::max(1u, a.n_blocks) * 128, 128, 128);
    if (e == cudaSuccess) e = byte_map(&map_x, x.values, x.ld, x.n, x.ld, p.tile);
    if (e != cudaSuccess) return e;
    if (y.dtype == ASP_F32) return product<float>(map_a, map_x, p, sm_count, st);
    if (y.dtype == ASP_F16) return product<__half>(map_a, map_x, p, sm_count, st);
    return product<__nv_bfloat16>(map_a, map_x, p, sm_count, st);
}
} // namespace asp
