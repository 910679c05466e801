// Products of block-sparse 8-bit matrices with a batch of rows (asp_block8_apply, asp_block8_product).
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

// n <= 32 rows, many blocks a CTA (block8_batch). Y[t][128 R + r] as for many rows (k_block8_product): D[128][32] in tensor memory, the powers of two as the products'
// scales, so that nothing is done to a block but to copy it, 16 KB in the products' layout, up to five ahead, and to multiply it.
//
// What is left beside the memory is X, which comes as the caller has it: every CTA converts the columns of its blocks, 32 rows of 128 a block, and that bounds it
// where there are more than 16 rows. Eight warps do, as two or four teams that take the blocks in turn, each with its next block's X on its way.
//
// A block row is shared by a cluster of CTAs, a contiguous piece of its blocks each; the cluster adds up the pieces in order in one another's shared memory.
//
// 8192 x 8192, all of it, bf16: 1 row 10.0 us (6.9 TB/s, much of it from L2), 16 rows 13.0, 32 rows 17.7; X in 8 bits already: 9.9, 11.3, 12.9. With products by mma.sync, which
// then bound it, 13.6, 20.2 and 31.2. Three matrices in turn, so that all comes from memory: 14.5 (4.8 TB/s; 10.3 for the bytes, the rest first copies, the cluster's
// sum and the next launch), 17.2, 20.2; by mma.sync 15.4, 22.1, 32.7.
constexpr unsigned kRows = 32;
constexpr unsigned kStages = 5;
constexpr unsigned kX = 16384, kScalesA = kX + kRows * 128, kScalesX = kScalesA + 512, kStageBytes = kScalesX + 512;
static_assert(kStageBytes % 1024 == 0, "blocks on 1024-byte boundaries");
constexpr unsigned kThreads = 320;
constexpr size_t kSharedBytes = kStages * kStageBytes + 1024;
// A team that comes to a stage has waited for the step that is a round of teams and a round of stages behind it. With more teams than stages that would say nothing of
// the stage's last step but one, and the wait for the last one, which is for a parity, could take one for the other.
constexpr unsigned kTeams = 4;
static_assert(kTeams < kStages, "a wait for a stage is for one of two steps");
constexpr unsigned kScalesAt = 32, kColumns = 64; // of tensor memory: D, then two places for a step's scales

struct BatchArgs
{
    Block8Dev a;
    XRows x;
    void *y;
    uint64_t ldy;
    unsigned n_split;
    unsigned teams; // of converting warps: 4 for up to 8 rows, else 2
    unsigned *fault;
};

struct Shared
{
    uint64_t full[kStages], converted[kStages], empty[kStages], done;
    unsigned tensor, gave_up;
};

template <class X, class Y> __global__ void __launch_bounds__(kThreads, 2) k_block8_batch(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ BatchArgs p)
{
    namespace cg = cooperative_groups;
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char *stages = raw + (1024 - tc::shared_address(raw) % 1024) % 1024;
    const unsigned warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned split = p.n_split, piece = blockIdx.x % split;
    const uint4 of = p.a.rows[blockIdx.x / split];
    const unsigned j0 = of.y + of.z * piece / split, j1 = of.y + of.z * (piece + 1) / split; // (less than 2^24 blocks, 8 pieces at most)
    if (threadIdx.x == 0)
    {
        tc::prefetch_map(&map_a);
        // Until the kernels before this one are done the matrix may still be written: it is brought to L2, which is never behind, and read afterwards.
        if (j0 < j1) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.a.values + (uint64_t)j0 * 16384), "r"(min(j1 - j0, 8u) * 16384) : "memory");
        for (unsigned i = 0; i < kStages; i++) tc::barrier_init(&sh.full[i], 1), tc::barrier_init(&sh.converted[i], 8 / p.teams), tc::barrier_init(&sh.empty[i], 1);
        tc::barrier_init(&sh.done, 1);
        sh.gave_up = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) tc::tensor_alloc(&sh.tensor, kColumns);
    // rows that are not there: zeros, times one
    for (unsigned s = 0; s < min(kStages, j1 - j0) && p.x.n < kRows; s++)
    {
        for (unsigned i = threadIdx.x; i < kRows * 8; i += kThreads) reinterpret_cast<uint4 *>(stages + s * kStageBytes + kX)[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x < 32) *reinterpret_cast<unsigned *>(stages + s * kStageBytes + kScalesX + threadIdx.x * 16) = 0x7f7f7f7fu;
    }
    tc::fence_async_shared();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tensor = sh.tensor;
    grid_wait();
    grid_release();
    float *part = reinterpret_cast<float *>(stages);

    if (warp == 0)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0;
            for (unsigned j = j0; j < j1; j++)
            {
                if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) break;
                unsigned char *to = stages + s * kStageBytes;
                tc::barrier_expect(&sh.full[s], 16384 + 512);
                tc::copy_tile(to, &map_a, 0, (int)(j * 128), &sh.full[s]);
                tc::copy_bytes(to + kScalesA, p.a.scale_rows + (uint64_t)j * 512, 512, &sh.full[s]);
                if (++s == kStages) s = 0, phase ^= 1;
            }
        }
    }
    else if (warp == 1)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0;
            bool all = true;
            for (unsigned j = j0; j < j1; j++)
            {
                all = tc::barrier_wait(&sh.full[s], phase, &sh.gave_up) && tc::barrier_wait(&sh.converted[s], phase, &sh.gave_up);
                if (!all) break;
                tc::fence_after();
                const unsigned a = tc::shared_address(stages + s * kStageBytes);
                const unsigned sa = tensor + kScalesAt + j % 2 * 8, sx = sa + 4;
                tc::copy_scales(sa, tc::scale_rows(a + kScalesA));
                tc::copy_scales(sx, tc::scale_rows(a + kScalesX));
#pragma unroll
                for (unsigned k = 0; k < 4; k++) tc::mma_scaled(tensor, tc::rows_k_major(a + 32 * k), tc::rows_k_major(a + kX + 32 * k), tc::scaled_e4m3(kRows, 0), sa, sx, j > j0 || k > 0);
                tc::commit(&sh.empty[s]);
                if (++s == kStages) s = 0, phase ^= 1;
            }
            if (all) tc::commit(&sh.done);
        }
    }
    else
    {
        // A row's block to each eight lanes, and the block 16 rows further where there are so many; `teams` of warps take the blocks in turn
        const unsigned lane8 = lane % 8, per_team = 8 / p.teams, t = (warp - 2) % per_team * 4 + lane / 8, team = (warp - 2) / per_team;
        unsigned s = team, phase = 0;
        Fetched<X> got[2] = {};
        unsigned col = 0;
        const auto ask = [&](unsigned j) {
#pragma unroll
            for (unsigned r = 0; r < 2; r++)
                if (t + 16 * r < p.x.n && j < j1) got[r].ask(p.x, t + 16 * r, col, lane8);
            if (j + p.teams < j1) col = p.a.col[j + p.teams];
        };
        if (j0 + team < j1) col = p.a.col[j0 + team];
        ask(j0 + team);
        bool all = true;
        for (unsigned j = j0 + team; j < j1; j += p.teams)
        {
            unsigned q[2][4], scale[2];
#pragma unroll
            for (unsigned r = 0; r < 2; r++)
                if (t - lane / 8 + 16 * r < p.x.n) scale[r] = got[r].eight(q[r], lane8); // (any row of the warp's)
            ask(j + p.teams);
            all = tc::warp_wait(&sh.empty[s], phase ^ 1, &sh.gave_up);
            if (!all) break;
            unsigned char *to = stages + s * kStageBytes;
#pragma unroll
            for (unsigned r = 0; r < 2; r++)
                if (t + 16 * r < p.x.n)
                {
#pragma unroll
                    for (int i = 0; i < 16; i += Fetched<X>::per)
                    {
                        const unsigned c = Fetched<X>::column(i, lane8);
                        unsigned char *at = to + kX + (t + 16 * r) * 128 + (c / 16 ^ t % 8) * 16 + c % 16; // (the copies' 128-byte swizzle)
                        if constexpr (Fetched<X>::per == 4) *reinterpret_cast<unsigned *>(at) = q[r][i / 4];
                        else if constexpr (Fetched<X>::per == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(q[r][i / 4], q[r][i / 4 + 1]);
                        else *reinterpret_cast<uint4 *>(at) = make_uint4(q[r][0], q[r][1], q[r][2], q[r][3]);
                    }
                    if (lane8 == 0) *reinterpret_cast<unsigned *>(to + kScalesX + (t + 16 * r) * 16) = scale[r] * 0x01010101u;
                }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::barrier_arrive(&sh.converted[s]);
            s += p.teams;
            if (s >= kStages) s -= kStages, phase ^= 1;
        }
        // the sums to shared memory: all blocks have been copied and multiplied, the stages are free
        const unsigned quarter = warp % 4, first = (warp - 2) / 4 * 16;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = 0.f;
        if (j0 < j1 && all && tc::warp_wait(&sh.done, 0, &sh.gave_up))
        {
            tc::fence_after();
            tc::tensor_load16(tensor + first + (quarter * 32 << 16), v);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) part[(first + i) * 128 + quarter * 32 + lane] = v[i];
    }
    __syncwarp();
    tc::fence_before();
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync(); // (all CTAs of the cluster come here, whatever became of their waits)
    tc::fence_after();
    Y *y = reinterpret_cast<Y *>(p.y);
    const unsigned inside = min(128u, p.a.n_rows - of.x * 128);
    for (unsigned i = threadIdx.x + kThreads * piece; i < p.x.n * 32; i += kThreads * split)
    {
        float4 v[8]; // all on their way before the first is needed
#pragma unroll
        for (unsigned s = 0; s < 8; s++)
            if (s < split) v[s] = *cluster.map_shared_rank(reinterpret_cast<const float4 *>(part) + i, s);
        float sum[4] = {};
#pragma unroll
        for (unsigned s = 0; s < 8; s++) // (in order)
            if (s < split) sum[0] += v[s].x, sum[1] += v[s].y, sum[2] += v[s].z, sum[3] += v[s].w;
        const unsigned r = i % 32 * 4;
        Y *to = y + (uint64_t)(i / 32) * p.ldy + of.x * 128 + r;
#pragma unroll
        for (unsigned k = 0; k < 4; k++)
            if (r + k < inside) to[k] = from_float<Y>(sum[k]);
    }
    cluster.sync(); // (its shared memory is read until here)
    if (sh.gave_up)
    {
        // copies and products in flight end by themselves; their memory is kept until then
        const uint64_t since = tc::now_ns();
        while (tc::now_ns() - since < 10000000ull) __nanosleep(1000);
        if (threadIdx.x == 0 && p.fault) *reinterpret_cast<volatile unsigned *>(p.fault) = 1;
    }
    if (warp == 1) tc::tensor_free(tensor, kColumns);
}

// Two CTAs share an SM, and its tensor memory. The driver, when asked, counts one for kernels that take any, so it is asked about this one, which is never launched.
__global__ void __launch_bounds__(kThreads, 2) k_without_tensor_memory() {}

template <class X, class Y> cudaError_t batch(const CUtensorMap &map_a, const BatchArgs &p, cudaStream_t st)
{
    auto *kernel = k_block8_batch<X, Y>;
    static SharedAllowance allowance;
    const cudaError_t e = allowance.need((const void *)kernel, (int)kSharedBytes);
    if (e != cudaSuccess) return e;
    return launch_pdl_cluster(kernel, p.n_split, dim3(p.a.n_block_rows * p.n_split), dim3(kThreads), kSharedBytes, st, map_a, p);
}
template <class Y> cudaError_t batch_of(int dtype, const CUtensorMap &map_a, const BatchArgs &p, cudaStream_t st)
{
    if (dtype < 0) return batch<Held, Y>(map_a, p, st);
    if (dtype == ASP_F32) return batch<float, Y>(map_a, p, st);
    if (dtype == ASP_F16) return batch<__half, Y>(map_a, p, st);
    return batch<__nv_bfloat16, Y>(map_a, p, st);
}
} // namespace

cudaError_t block8_batch_room(unsigned fit[9])
{
    static SharedAllowance allowance;
    static ClusterRoom room;
    const void *kernel = (const void *)k_without_tensor_memory;
    const cudaError_t e = allowance.need(kernel, (int)kSharedBytes);
    return e == cudaSuccess ? room.most(kernel, kThreads, kSharedBytes, fit) : e;
}

cudaError_t launch_block8_batch(const Block8Dev &a, const Dense *x, const Rows8Dev *held, unsigned n, const Dense &y, int sm_count, const unsigned *fit, unsigned *fault, cudaStream_t st)
{
    BatchArgs p = {};
    p.a = a, p.y = y.p, p.ldy = y.ld, p.fault = fault;
    p.x.n = n, p.x.n_cols = a.n_cols;
    if (held) p.x.held = *held;
    else p.x.p = x->p, p.x.ld = x->ld;
    p.teams = n <= 8 ? 4 : 2;
    p.n_split = host::block8_batch_split(a.n_block_rows, a.longest, sm_count, fit);
    CUtensorMap map_a;
    const cudaError_t e = byte_map(&map_a, a.values, 128, (uint64_t)(a.n_blocks ? a.n_blocks : 1) * 128, 128, 128);
    if (e != cudaSuccess) return e;
    const int from = held ? -1 : x->dtype;
    if (y.dtype == ASP_F32) return batch_of<float>(from, map_a, p, st);
    if (y.dtype == ASP_F16) return batch_of<__half>(from, map_a, p, st);
    return batch_of<__nv_bfloat16>(from, map_a, p, st);
}
} // namespace asp
