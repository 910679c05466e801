// The gradient by the stored blocks (asp_block8_gradient).
#include "../../include/asp_b200.h"
#include "block8.h"
#include "block8_device.h"

namespace asp
{
namespace
{
using namespace block8;

// dA_b[r][c] = sum over t of dy[t][128 R + r] x[t][128 C + c]: a block to a CTA, 8 x 8 elements a thread, 16 rows of dy and x at a time
// in shared memory, in 32 bits.
constexpr int kRows = 16;
template <class T>
__global__ void __launch_bounds__(256) k_block8_gradient(Block8Dev a, const unsigned *row, Rows8Dev x, const T *dy, uint64_t ld, float *out, bool accumulate)
{
    __shared__ float sy[kRows][128], sx[kRows][128];
    const unsigned b = blockIdx.x, r0 = row[b] * 128, cb = a.col[b], ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    float acc[8][8] = {};
    for (unsigned t0 = 0; t0 < x.n; t0 += kRows)
    {
        for (unsigned i = threadIdx.x; i < kRows * 128; i += 256)
        {
            const unsigned t = t0 + i / 128, r = r0 + i % 128;
            sy[i / 128][i % 128] = t < x.n && r < a.n_rows ? to_float(dy[(uint64_t)t * ld + r]) : 0.f;
        }
        for (unsigned i = threadIdx.x; i < kRows * 32; i += 256)
        {
            const unsigned t = t0 + i / 32, c = i % 32 * 4;
            float v[4] = {};
            if (t < x.n)
            {
                unpack4(*reinterpret_cast<const unsigned *>(x.values + t * x.ld + cb * 128 + c), v);
                const float scale = power(x.scales[scale_at(x, t, cb)]);
                for (int k = 0; k < 4; k++) v[k] *= scale;
            }
            for (int k = 0; k < 4; k++) sx[i / 32][c + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kRows; t++)
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[i][j] = __fmaf_rn(sy[t][ty + 16 * i], sx[t][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 8; j++)
        {
            float *to = out + (uint64_t)b * 16384 + (ty + 16 * i) * 128 + tx + 16 * j;
            *to = accumulate ? *to + acc[i][j] : acc[i][j];
        }
}
} // namespace

cudaError_t launch_block8_gradient(const Block8Dev &a, const unsigned *row, const Rows8Dev &x, const Dense &dy, float *out, bool accumulate, int sm_count, cudaStream_t st)
{
    if (a.n_blocks == 0) return cudaSuccess;
    if (dy.dtype == ASP_F16) k_block8_gradient<<<a.n_blocks, 256, 0, st>>>(a, row, x, reinterpret_cast<const __half *>(dy.p), dy.ld, out, accumulate);
    else k_block8_gradient<<<a.n_blocks, 256, 0, st>>>(a, row, x, reinterpret_cast<const __nv_bfloat16 *>(dy.p), dy.ld, out, accumulate);
    return cudaGetLastError();
}
} // namespace asp
