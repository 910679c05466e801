// The gradient by the stored blocks (asp_block8_gradient).
#include <algorithm>

#include "../../include/asp_b200.h"
#include "block8.h"
#include "block8_device.h"
#include "tcgen05.h"
#include "tensor_map.h"

namespace asp
{
namespace
{
using namespace block8;

// dA_b[r][c] = sum over t of dy[t][128 R + r] x[t][128 C + c], for the stored blocks b = (R, C) only.
//
// The sum runs over the rows t, in which the scales of x differ from row to row, so they cannot be the products' scales: x is unfolded to the
// 16-bit type of dy, exactly, and multiplied in that type. Both factors lie in memory with r and c side by side, which
// tcgen05.mma takes as it is (columns of k). Two blocks of a block row share the copies of dy: D[128][256] in tensor
// memory, twice, so that a pair's 128 KB leave under the next one's products. A step is 64 rows t: 16 KB of dy, 8 KB of x a block.
//
// A CTA per SM goes through pairs: warp 0 copies, warp 1 issues products, warps 4 to 7 store, warps 8 to 15 unfold x.
constexpr unsigned kRows = 64;              // t a step
constexpr unsigned kStages = 4, kUnfolded = 2;
constexpr unsigned kTile = kRows * 128;     // elements of a step's factor
constexpr unsigned kStageBytes = 2 * kTile + 2 * kTile + 1024; // dy, x of two blocks, their scales
constexpr unsigned kThreads = 512;

struct GradientArgs
{
    Block8Dev a;
    Rows8Dev x;
    const unsigned *row, *pairs; // first block, and whether a second one of the same row follows (bit 31)
    const void *dy;
    uint64_t ld;
    float *out;
    unsigned n_pairs;
    bool direct; // dy can be copied by tiles
    bool accumulate;
    unsigned *fault;
};

struct Shared
{
    uint64_t full[kStages], empty[kStages], unfolded[kUnfolded], used[kUnfolded], done[2], taken[2];
    unsigned tensor, gave_up;
};

// 4 elements in 8 bits times a row's power of two
struct Unfold16 // to fp16: in two factors, since the power may be below what fp16 has (the product is not, as x was fp16)
{
    __half2 f1, f2;
    __device__ __forceinline__ Unfold16(unsigned scale)
    {
        const int k1 = max((int)scale, 127 - 14);
        f1 = __float2half2_rn(power((unsigned)k1)), f2 = __float2half2_rn(power((unsigned)((int)scale - k1 + 127)));
    }
    __device__ __forceinline__ uint2 operator()(unsigned four) const
    {
        const __half2 a = __hmul2(__hmul2(unpack2(four & 0xffffu), f1), f2), b = __hmul2(__hmul2(unpack2(four >> 16), f1), f2);
        return make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
    static constexpr bool bf16 = false;
};
struct UnfoldB16
{
    float f;
    __device__ __forceinline__ UnfoldB16(unsigned scale) : f(power(scale)) {}
    __device__ __forceinline__ uint2 operator()(unsigned four) const
    {
        float v[4];
        unpack4(four, v);
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0] * f, v[1] * f), b = __floats2bfloat162_rn(v[2] * f, v[3] * f);
        return make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
    static constexpr bool bf16 = true;
};

template <class Unfold>
__global__ void __launch_bounds__(kThreads, 1) k_block8_gradient(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ GradientArgs p)
{
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char *stages = raw + (1024 - tc::shared_address(raw) % 1024) % 1024;
    unsigned char *halves = stages + kStages * kStageBytes; // unfolded x: two blocks, 64 columns after 64 columns, a row t 128 bytes
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const unsigned steps = (p.x.n + kRows - 1) / kRows;
    if (threadIdx.x == 0)
    {
        for (unsigned i = 0; i < kStages; i++) tc::barrier_init(&sh.full[i], 1), tc::barrier_init(&sh.empty[i], 1);
        for (unsigned i = 0; i < kUnfolded; i++) tc::barrier_init(&sh.unfolded[i], 8), tc::barrier_init(&sh.used[i], 1);
        for (unsigned i = 0; i < 2; i++) tc::barrier_init(&sh.done[i], 1), tc::barrier_init(&sh.taken[i], 4);
        sh.gave_up = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) tc::tensor_alloc(&sh.tensor, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tensor = sh.tensor;

    if (warp == 0)
    {
        if (lane == 0)
        {
            unsigned s = 0, phase = 0;
            for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
            {
                const unsigned b = p.pairs[u] & 0x7fffffffu, blocks = 1 + (p.pairs[u] >> 31), r = p.row[b] * 128;
                unsigned col[2] = {p.a.col[b], blocks > 1 ? p.a.col[b + 1] : 0};
                for (unsigned i = 0; i < steps; i++)
                {
                    if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = stages + s * kStageBytes;
                    const int t = (int)(i * kRows);
                    tc::barrier_expect(&sh.full[s], (p.direct ? 2 * kTile : 0) + blocks * (kTile + 512));
                    if (p.direct)
                    {
                        tc::copy_tile(to, &map_dy, (int)r, t, &sh.full[s]);
                        tc::copy_tile(to + kTile, &map_dy, (int)r + 64, t, &sh.full[s]);
                    }
                    for (unsigned k = 0; k < blocks; k++)
                    {
                        tc::copy_tile(to + (2 + k) * kTile, &map_x, (int)(col[k] * 128), t, &sh.full[s]);
                        tc::copy_bytes(to + 4 * kTile + k * 512, p.x.scales + ((uint64_t)(col[k] / 4) * p.x.pieces + t / 128) * 512, 512, &sh.full[s]);
                    }
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    }
    else if (warp == 1)
    {
        if (lane == 0)
        {
            unsigned s = 0, phase = 0, h = 0, h_phase = 0, d = 0, d_phase = 0;
            for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
            {
                const unsigned shape = tc::halves(128 + 128 * (p.pairs[u] >> 31), Unfold::bf16);
                if (!tc::barrier_wait(&sh.taken[d], d_phase ^ 1, &sh.gave_up)) goto end;
                tc::fence_after();
                for (unsigned i = 0; i < steps; i++)
                {
                    if (!tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) goto end;
                    if (!tc::barrier_wait(&sh.unfolded[h], h_phase, &sh.gave_up)) goto end;
                    tc::fence_after();
                    const unsigned dy = tc::shared_address(stages + s * kStageBytes), x = tc::shared_address(halves + h * 4 * kTile);
#pragma unroll
                    for (unsigned k = 0; k < kRows / 16; k++) // 16 rows of 128 bytes on
                        tc::mma_halves(tensor + d * 256, tc::columns_of_k(dy + 2048 * k, kTile), tc::columns_of_k(x + 2048 * k, kTile), shape, i > 0 || k > 0);
                    tc::commit(&sh.empty[s]);
                    tc::commit(&sh.used[h]);
                    if (++s == kStages) s = 0, phase ^= 1;
                    if (++h == kUnfolded) h = 0, h_phase ^= 1;
                }
                tc::commit(&sh.done[d]);
                d ^= 1;
                if (d == 0) d_phase ^= 1;
            }
        }
    }
    else if (warp >= 8)
    {
        // 8 lanes and 16 columns a lane to a row t: 4 rows a warp at once, warp w rows 4 w on, then 32 rows further
        const unsigned lane8 = lane % 8, first = (warp - 8) * 4 + lane / 8;
        unsigned s = 0, phase = 0, h = 0, h_phase = 0;
        for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
        {
            const unsigned b = p.pairs[u] & 0x7fffffffu, blocks = 1 + (p.pairs[u] >> 31), r0 = p.row[b] * 128;
            const unsigned byte[2] = {p.a.col[b] % 4, blocks > 1 ? p.a.col[b + 1] % 4 : 0};
            for (unsigned i = 0; i < steps; i++)
            {
                if (!tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) goto end;
                if (!tc::barrier_wait(&sh.used[h], h_phase ^ 1, &sh.gave_up)) goto end;
                unsigned char *from = stages + s * kStageBytes, *to = halves + h * 4 * kTile;
                for (unsigned k = 0; k < blocks; k++)
#pragma unroll
                    for (unsigned j = 0; j < kRows / 32; j++)
                    {
                        const unsigned t = first + 32 * j, row = i * kRows + t;
                        const uint4 q = *reinterpret_cast<const uint4 *>(from + (2 + k) * kTile + t * 128 + 16 * lane8);
                        // (rows behind the last one: zeros, whose scales may be anything)
                        const unsigned scale = row < p.x.n ? from[4 * kTile + k * 512 + row % 32 * 16 + row / 32 % 4 * 4 + byte[k]] : 127;
                        const Unfold f(scale);
                        const uint2 a = f(q.x), b2 = f(q.y), c = f(q.z), e = f(q.w);
                        // 16-byte pieces 2 l and 2 l + 1 of the row's 128 bytes, swapped in the second half so that eight lanes meet no conflict
                        unsigned char *line = to + (2 * k + lane8 / 4) * kTile + t * 128;
                        const unsigned piece = lane8 % 4 * 2, second = lane8 / 4;
                        const uint4 lo = make_uint4(a.x, a.y, b2.x, b2.y), hi = make_uint4(c.x, c.y, e.x, e.y);
                        *reinterpret_cast<uint4 *>(line + (((piece + second) ^ (t % 8)) * 16)) = second ? hi : lo;
                        *reinterpret_cast<uint4 *>(line + (((piece + 1 - second) ^ (t % 8)) * 16)) = second ? lo : hi;
                    }
                if (!p.direct) // dy element by element, into the same swizzle
                {
                    const unsigned short *dy = reinterpret_cast<const unsigned short *>(p.dy);
                    for (unsigned e = threadIdx.x - 256; e < kRows * 128; e += 256)
                    {
                        const unsigned t = e / 128, r = e % 128;
                        const unsigned short v = i * kRows + t < p.x.n && r0 + r < p.a.n_rows ? dy[(uint64_t)(i * kRows + t) * p.ld + r0 + r] : 0;
                        *reinterpret_cast<unsigned short *>(from + r / 64 * kTile + t * 128 + ((r % 64 / 8) ^ (t % 8)) * 16 + r % 8 * 2) = v;
                    }
                }
                tc::fence_async_shared();
                __syncwarp();
                if (lane == 0) tc::barrier_arrive(&sh.unfolded[h]);
                if (++s == kStages) s = 0, phase ^= 1;
                if (++h == kUnfolded) h = 0, h_phase ^= 1;
            }
        }
    }
    else if (warp >= 4)
    {
        unsigned d = 0, d_phase = 0;
        const unsigned quarter = warp % 4, r = quarter * 32 + lane;
        for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
        {
            const unsigned b = p.pairs[u] & 0x7fffffffu, blocks = 1 + (p.pairs[u] >> 31);
            const bool row_in = p.row[b] * 128 + r < p.a.n_rows;
            if (!tc::barrier_wait(&sh.done[d], d_phase, &sh.gave_up)) goto end;
            tc::fence_after();
            for (unsigned c = 0; c < blocks * 128; c += 32)
            {
                float v[32];
                tc::tensor_load32(tensor + d * 256 + c + (quarter * 32 << 16), v);
                const unsigned block = b + c / 128, col0 = p.a.col[block] * 128 + c % 128;
                float4 *to = reinterpret_cast<float4 *>(p.out + (uint64_t)block * 16384 + r * 128 + c % 128);
#pragma unroll
                for (unsigned k = 0; k < 32; k++)
                    if (!row_in || col0 + k >= p.a.n_cols) v[k] = 0.f; // outside the matrix
#pragma unroll
                for (int k = 0; k < 8; k++)
                {
                    float4 w = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                    if (p.accumulate)
                    {
                        const float4 o = to[k];
                        w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
                    }
                    to[k] = w;
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::barrier_arrive(&sh.taken[d]);
            d ^= 1;
            if (d == 0) d_phase ^= 1;
        }
    }
end:
    __syncwarp();
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
    const size_t smem = kStages * kStageBytes + kUnfolded * 4 * kTile + 1024;
    const cudaError_t e = cudaFuncSetAttribute(k_block8_gradient<Unfold>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    k_block8_gradient<Unfold><<<std::min<unsigned>(p.n_pairs, (unsigned)sm_count), kThreads, smem, st>>>(map_dy, map_x, p);
    return cudaGetLastError();
}
} // namespace

cudaError_t launch_block8_gradient(const Block8Dev &a, const unsigned *row, const unsigned *pairs, unsigned n_pairs, const Rows8Dev &x, const Dense &dy, float *out, bool accumulate, int sm_count,
                                   unsigned *fault, cudaStream_t st)
{
    if (a.n_blocks == 0) return cudaSuccess;
    if (x.n == 0) return accumulate ? cudaSuccess : cudaMemsetAsync(out, 0, (size_t)a.n_blocks * 16384 * sizeof(float), st);
    GradientArgs p = {};
    p.a = a, p.x = x, p.row = row, p.pairs = pairs, p.n_pairs = n_pairs;
    p.dy = dy.p, p.ld = dy.ld, p.out = out, p.accumulate = accumulate, p.fault = fault;
    p.direct = ((uintptr_t)dy.p & 15) == 0 && dy.ld % 8 == 0;
    CUtensorMap map_dy, map_x;
    cudaError_t e = byte_map(&map_x, x.values, x.ld, x.n, x.ld, kRows, false);
    if (e == cudaSuccess && p.direct)
        e = tensor_map(&map_dy, dy.dtype == ASP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dy.p, a.n_rows, x.n, dy.ld * 2, 64, kRows);
    else map_dy = map_x; // (not used)
    if (e != cudaSuccess) return e;
    if (dy.dtype == ASP_BF16) return gradient<UnfoldB16>(map_dy, map_x, p, sm_count, st);
    return gradient<Unfold16>(map_dy, map_x, p, sm_count, st);
}
} // namespace asp
