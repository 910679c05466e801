// The gradient by the stored blocks (asp_block8_gradient).
#include <algorithm>

#include "../../include/asp_b200.h"
#include "block8.h"
#include "block8_device.h"
#include "launch.h"
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
// A CTA per SM goes through pairs: warp 0 copies, warp 1 issues products, warps 4 to 7 store, warps 8 to 15 and 16 to 23 unfold x, every second
// step each.
constexpr unsigned kRows = 64;          // t a step
constexpr unsigned kTile = kRows * 128; // bytes of 64 columns of a step's rows in 16 bits, of 128 in 8
constexpr unsigned kStages = 4, kStageBytes = 2 * kTile;      // dy
constexpr unsigned kHeld = 3, kHeldBytes = 2 * kTile + 1024;  // x of two blocks, and its scales
constexpr unsigned kUnfolded = 3, kUnfoldedBytes = 4 * kTile; // x of two blocks in 16 bits: 64 columns after 64 columns, a row t 128 bytes
constexpr unsigned kThreads = 768;

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
    uint64_t full[kStages], empty[kStages], held[kHeld], read[kHeld], unfolded[kUnfolded], used[kUnfolded], done[2], taken[2];
    unsigned tensor, gave_up;
};

// 16 elements in 8 bits times a row's power of two: eight words of two elements.
struct Unfold16 // to fp16: in two factors, since the power may be below what fp16 has (the product is not, as x was fp16)
{
    static constexpr bool bf16 = false;
    static __device__ __forceinline__ void words(uint4 q, unsigned scale, unsigned *out)
    {
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
// columns are told apart when they are stored). NaN, which e4m3 writes as its largest number, is lost that way and put back.
struct UnfoldB16
{
    static constexpr bool bf16 = true;
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
            for (int i = 0; i < 8; i++) out[i] = product(out[i], ((scale + 120 - 254 + 127) << 7) * 0x10001u);
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
// D's column of column c of a block
template <class Unfold> __device__ __forceinline__ constexpr unsigned column_of(unsigned c) { return Unfold::bf16 && (c % 4 == 1 || c % 4 == 2) ? c ^ 3 : c; }

template <class Unfold>
__global__ void __launch_bounds__(kThreads, 1) k_block8_gradient(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ GradientArgs p)
{
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char *stages = raw + (1024 - tc::shared_address(raw) % 1024) % 1024;
    unsigned char *halves = stages + kStages * kStageBytes, *bytes = halves + kUnfolded * kUnfoldedBytes;
    const unsigned warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned steps = (p.x.n + kRows - 1) / kRows;
    if (threadIdx.x == 32)
    {
        tc::prefetch_map(&map_x);
        if (p.direct) tc::prefetch_map(&map_dy);
    }
    if (threadIdx.x == 0)
    {
        for (unsigned i = 0; i < kStages; i++) tc::barrier_init(&sh.full[i], 1), tc::barrier_init(&sh.empty[i], 1);
        for (unsigned i = 0; i < kHeld; i++) tc::barrier_init(&sh.held[i], 1), tc::barrier_init(&sh.read[i], 8);
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
    grid_wait();
    grid_release();

    if (warp == 0)
    {
        if (tc::one_lane())
        {
            unsigned s = 0, phase = 0, x = 0, x_phase = 0;
            for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
            {
                const unsigned b = p.pairs[u] & 0x7fffffffu, blocks = 1 + (p.pairs[u] >> 31), r = p.row[b] * 128;
                const unsigned col[2] = {p.a.col[b], blocks > 1 ? p.a.col[b + 1] : 0};
                for (unsigned i = 0; i < steps; i++)
                {
                    const int t = (int)(i * kRows);
                    if (!tc::barrier_wait(&sh.read[x], x_phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = bytes + x * kHeldBytes;
                    tc::barrier_expect(&sh.held[x], blocks * (kTile + 512));
#pragma unroll
                    for (unsigned k = 0; k < 2; k++)
                        if (k < blocks)
                        {
                            tc::copy_tile(to + k * kTile, &map_x, (int)(col[k] * 128), t, &sh.held[x]);
                            tc::copy_bytes(to + 2 * kTile + k * 512, p.x.scales + ((uint64_t)(col[k] / 4) * p.x.pieces + t / 128) * 512, 512, &sh.held[x]);
                        }
                    if (++x == kHeld) x = 0, x_phase ^= 1;
                    if (!p.direct) continue;
                    if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                    tc::barrier_expect(&sh.full[s], kStageBytes);
                    tc::copy_tile(stages + s * kStageBytes, &map_dy, (int)r, t, &sh.full[s]);
                    tc::copy_tile(stages + s * kStageBytes + kTile, &map_dy, (int)r + 64, t, &sh.full[s]);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    }
    else if (warp == 1)
    {
        if (tc::one_lane())
        {
            // A step's factors are waited for under the products of the step before, of which the tensor cores have no more than two or three waiting:
            // a look at a barrier takes 130 clocks, a step's products 512.
            unsigned s = 0, phase = 0, h = 0, h_phase = 0, d = 0, d_phase = 0;
            const auto ready = [&] { return (!p.direct || tc::barrier_wait(&sh.full[s], phase, &sh.gave_up)) && tc::barrier_wait(&sh.unfolded[h], h_phase, &sh.gave_up); };
            if (!ready()) goto end;
            for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
            {
                const unsigned shape = tc::halves(128 + 128 * (p.pairs[u] >> 31), Unfold::bf16);
                const bool last = u + gridDim.x >= p.n_pairs;
                if (!tc::barrier_wait(&sh.taken[d], d_phase ^ 1, &sh.gave_up)) goto end;
                for (unsigned i = 0; i < steps; i++)
                {
                    tc::fence_after();
                    const unsigned dy = tc::shared_address(stages + s * kStageBytes), x = tc::shared_address(halves + h * kUnfoldedBytes);
                    uint64_t *const empty = &sh.empty[s], *const used = &sh.used[h];
                    if (++s == kStages) s = 0, phase ^= 1;
                    if (++h == kUnfolded) h = 0, h_phase ^= 1;
#pragma unroll
                    for (unsigned k = 0; k < kRows / 16; k++) // 16 rows of 128 bytes on
                    {
                        if (k == 1 && !(last && i + 1 == steps) && !ready()) goto end;
                        tc::mma_halves(tensor + d * 256, tc::columns_of_k(dy + 2048 * k, kTile), tc::columns_of_k(x + 2048 * k, kTile), shape, i > 0 || k > 0);
                    }
                    tc::commit(empty);
                    tc::commit(used);
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
        const unsigned lane8 = lane % 8, first = warp % 8 * 4 + lane / 8, mine = warp / 16;
        unsigned s = 0, phase = 0, x = 0, x_phase = 0, h = 0, h_phase = 0, turn = 0;
        for (unsigned u = blockIdx.x; u < p.n_pairs; u += gridDim.x)
        {
            const unsigned b = p.pairs[u] & 0x7fffffffu, blocks = 1 + (p.pairs[u] >> 31), r0 = p.row[b] * 128;
            const unsigned byte[2] = {p.a.col[b] % 4, blocks > 1 ? p.a.col[b + 1] % 4 : 0};
            for (unsigned i = 0; i < steps; i++)
            {
                if (turn == mine)
                {
                    if (!tc::barrier_wait(&sh.held[x], x_phase, &sh.gave_up)) goto end;
                    const unsigned char *from = bytes + x * kHeldBytes;
                    uint4 q[2][2];
                    unsigned scale[2][2];
#pragma unroll
                    for (unsigned k = 0; k < 2; k++)
#pragma unroll
                        for (unsigned j = 0; j < 2; j++)
                        {
                            const unsigned t = first + 32 * j, row = i * kRows + t;
                            scale[k][j] = 127; // (of rows behind the last one, which are zeros)
                            if (k >= blocks) continue;
                            q[k][j] = *reinterpret_cast<const uint4 *>(from + k * kTile + t * 128 + 16 * lane8);
                            if (row < p.x.n) scale[k][j] = from[2 * kTile + k * 512 + first * 16 + row / 32 % 4 * 4 + byte[k]];
                        }
                    __syncwarp();
                    if (lane == 0) tc::barrier_arrive(&sh.read[x]); // the next copy may come while these are unfolded
                    if (!tc::barrier_wait(&sh.used[h], h_phase ^ 1, &sh.gave_up)) goto end;
                    unsigned char *to = halves + h * kUnfoldedBytes;
#pragma unroll
                    for (unsigned k = 0; k < 2; k++)
#pragma unroll
                        for (unsigned j = 0; j < 2; j++)
                        {
                            if (k >= blocks) continue;
                            const unsigned t = first + 32 * j;
                            unsigned v[8];
                            Unfold::words(q[k][j], scale[k][j], v);
                            // 16-byte pieces 2 l and 2 l + 1 of the row's 128 bytes, swapped in the second half so that eight lanes meet no conflict
                            unsigned char *line = to + (2 * k + lane8 / 4) * kTile + t * 128;
                            const unsigned piece = lane8 % 4 * 2, second = lane8 / 4;
                            const uint4 lo = make_uint4(v[0], v[1], v[2], v[3]), hi = make_uint4(v[4], v[5], v[6], v[7]);
                            *reinterpret_cast<uint4 *>(line + (((piece + second) ^ (t % 8)) * 16)) = second ? hi : lo;
                            *reinterpret_cast<uint4 *>(line + (((piece + 1 - second) ^ (t % 8)) * 16)) = second ? lo : hi;
                        }
                    if (!p.direct) // dy element by element, into the same swizzle
                    {
                        if (!tc::barrier_wait(&sh.empty[s], phase ^ 1, &sh.gave_up)) goto end;
                        const unsigned short *dy = reinterpret_cast<const unsigned short *>(p.dy);
                        for (unsigned e = threadIdx.x % 256; e < kRows * 128; e += 256)
                        {
                            const unsigned t = e / 128, r = e % 128;
                            const unsigned short v = i * kRows + t < p.x.n && r0 + r < p.a.n_rows ? dy[(uint64_t)(i * kRows + t) * p.ld + r0 + r] : 0;
                            *reinterpret_cast<unsigned short *>(stages + s * kStageBytes + r / 64 * kTile + t * 128 + ((r % 64 / 8) ^ (t % 8)) * 16 + r % 8 * 2) = v;
                        }
                    }
                    tc::fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tc::barrier_arrive(&sh.unfolded[h]);
                }
                turn ^= 1;
                if (++s == kStages) s = 0, phase ^= 1;
                if (++x == kHeld) x = 0, x_phase ^= 1;
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
            if (!tc::barrier_wait<64>(&sh.done[d], d_phase, &sh.gave_up)) goto end;
            tc::fence_after();
            for (unsigned c = 0; c < blocks * 128; c += 32)
            {
                float d32[32], v[32];
                tc::tensor_load32(tensor + d * 256 + c + (quarter * 32 << 16), d32);
                const unsigned block = b + c / 128, col0 = p.a.col[block] * 128 + c % 128;
                float4 *to = reinterpret_cast<float4 *>(p.out + (uint64_t)block * 16384 + r * 128 + c % 128);
#pragma unroll
                for (unsigned k = 0; k < 32; k++) v[k] = row_in && col0 + k < p.a.n_cols ? d32[column_of<Unfold>(k)] : 0.f; // zero outside the matrix
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
    const size_t smem = kStages * kStageBytes + kUnfolded * kUnfoldedBytes + kHeld * kHeldBytes + 1024;
    static SharedAllowance allowance;
    const cudaError_t e = allowance.need((const void *)k_block8_gradient<Unfold>, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_block8_gradient<Unfold>, dim3(std::min<unsigned>(p.n_pairs, (unsigned)sm_count)), dim3(kThreads), smem, st, map_dy, map_x, p);
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
    cudaError_t e = byte_map(&map_x, x.values, x.ld, x.n, x.ld, kRows, false); // as it lies, without swizzle
    if (e == cudaSuccess && p.direct)
        e = tensor_map(&map_dy, dy.dtype == ASP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dy.p, a.n_rows, x.n, dy.ld * 2, 64, kRows);
    else map_dy = map_x; // (not used)
    if (e != cudaSuccess) return e;
    if (dy.dtype == ASP_BF16) return gradient<UnfoldB16>(map_dy, map_x, p, sm_count, st);
    return gradient<Unfold16>(map_dy, map_x, p, sm_count, st);
}
} // namespace asp
