// The parts of sm_100a's asynchronous machinery that the kernels of block-sparse matrices use: barriers with bounded waits, tiled copies,
// tensor memory, and the two kinds of tcgen05.mma.
#ifndef ASP_TCGEN05_H
#define ASP_TCGEN05_H
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace asp
{
#ifdef __CUDACC__
namespace tc
{
__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

// One lane of the warp, which is here as a whole. The compiler knows that what follows runs in one lane and issues copies and products as they
// are; behind a test of the lane's number it goes through the lanes for each of them (measured: 490 clocks for what takes 50).
__device__ __forceinline__ bool one_lane()
{
    unsigned one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// ---- barriers ----
__device__ __forceinline__ void barrier_init(uint64_t *b, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint64_t *b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(b)) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint64_t *b, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint64_t *b, unsigned parity)
{
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(shared_address(b)), "r"(parity) : "memory");
    return done != 0;
}
// A wait that ends: after about two seconds, or as soon as another wait of the CTA has given up, it returns false, and so do all that come
// after it. What is waited for takes microseconds.
__device__ __forceinline__ uint64_t now_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// idle_ns: what a warp that waits for long sleeps between two looks, so that it does not take issue slots from those that work
template <unsigned idle_ns = 0> __device__ __forceinline__ bool barrier_wait(uint64_t *b, unsigned parity, volatile unsigned *gave_up)
{
    if (barrier_test(b, parity)) return true;
    uint64_t since = 0;
    for (unsigned i = 1;; i++)
    {
        if (idle_ns) __nanosleep(idle_ns);
        if (barrier_test(b, parity)) return true;
        if (i % 256) continue;
        if (*gave_up) return false;
        const uint64_t t = now_ns();
        if (since == 0) since = t;
        else if (t - since > 2000000000ull)
        {
            *gave_up = 1;
            return false;
        }
    }
}
// For a warp that goes on as a whole: its lanes look one by one, and one may give up where another finds that it need not. True where all of them may go on.
template <unsigned idle_ns = 0> __device__ __forceinline__ bool warp_wait(uint64_t *b, unsigned parity, volatile unsigned *gave_up)
{
    return __all_sync(~0u, barrier_wait<idle_ns>(b, parity, gave_up));
}
__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tiled copies ---- (x: the contiguous coordinate, a multiple of 16 bytes)
__device__ __forceinline__ void prefetch_map(const CUtensorMap *m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ void copy_tile(void *to, const CUtensorMap *m, int x, int y, uint64_t *b)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(shared_address(to)), "l"(m), "r"(x), "r"(y),
                 "r"(shared_address(b))
                 : "memory");
}

// bytes as they lie (whole 16s, both addresses on 16-byte boundaries)
__device__ __forceinline__ void copy_bytes(void *to, const void *from, unsigned bytes, uint64_t *b)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(to)), "l"(from), "r"(bytes), "r"(shared_address(b)) : "memory");
}

// ---- tensor memory ---- (alloc and free: one whole warp; the address of the first column goes to *where)
__device__ __forceinline__ void tensor_alloc(unsigned *where, unsigned columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(where)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tensor_free(unsigned at, unsigned columns) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 columns of the 32 lanes that belong to the warp (number of the warp modulo 4). The registers are written while the program goes on: they go
// through the wait, so that nothing that is computed from them can come before it.
__device__ __forceinline__ void tensor_load16(unsigned at, float *v)
{
    unsigned r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tensor_store16(unsigned at, const float *v)
{
    unsigned r[16];
#pragma unroll
    for (int i = 0; i < 16; i++) r[i] = __float_as_uint(v[i]);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                 "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
                 : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---- products ---- (one thread issues them; they run in order)
__device__ __forceinline__ void commit(uint64_t *b)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(b)) : "memory");
}
// Rows of 128 bytes of k, in the copies' 128-byte swizzle: groups of 8 rows are 1024 bytes apart. Begins on a 1024-byte boundary, or 32, 64, 96
// bytes of k behind one.
__device__ __forceinline__ uint64_t rows_k_major(unsigned address) { return (uint64_t)(address >> 4 & 0x3fff) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61; }
// Columns of k of 16-bit elements, 64 side by side (128 bytes) a row of k in the copies' 128-byte swizzle: groups of 8 k are 1024 bytes apart, the next 64
// elements `next` bytes. Begins on a 1024-byte boundary.
__device__ __forceinline__ uint64_t columns_of_k(unsigned address, unsigned next) { return (uint64_t)(address >> 4 & 0x3fff) | (uint64_t)(next >> 4) << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61; }
// D[128][N] (+)= A B^T over 16 k, 16-bit elements of one type (bf16 or fp16), both in columns of k
__device__ __forceinline__ constexpr unsigned halves(unsigned n, bool bf16) { return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | 1u << 15 | 1u << 16 | (n >> 3) << 17 | (128u >> 4) << 24; }
__device__ __forceinline__ void mma_halves(unsigned d, uint64_t a, uint64_t b, unsigned shape, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((unsigned)add)
                 : "memory");
}
// 32 scales of 16 bytes, without swizzle: groups of 8 are 128 bytes apart
__device__ __forceinline__ uint64_t scale_rows(unsigned address) { return (uint64_t)(address >> 4 & 0x3fff) | 8ull << 16 | 8ull << 32 | 1ull << 46; }
// 512 bytes to 4 columns: lane l of each quarter gets bytes 16 l to 16 l + 15
__device__ __forceinline__ void copy_scales(unsigned to, uint64_t from) { asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from) : "memory"); }
// D[128][N] (+)= A B^T over 32 bytes of k, e4m3, both k-major, each row's products times a power of two of A's row and of B's: byte 0 of A's words that
// copy_scales put there and byte `b_byte` of B's, row 32 c + l in lane l of column c.
__device__ __forceinline__ constexpr unsigned scaled_e4m3(unsigned n, unsigned b_byte) { return b_byte << 4 | 1u << 23 | (n >> 3) << 17 | (128u >> 4) << 24; }
__device__ __forceinline__ void mma_scaled(unsigned d, uint64_t a, uint64_t b, unsigned shape, unsigned a_scale, unsigned b_scale, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(shape), "r"(a_scale), "r"(b_scale), "r"((unsigned)add)
                 : "memory");
}
} // namespace tc
#endif
} // namespace asp
#endif
