// What the kernels of block-sparse 8-bit matrices (asp_b200_block8.h) are given, and their launches (kernels_block8*.cu).
#ifndef ASP_BLOCK8_H
#define ASP_BLOCK8_H
#include <cuda_runtime.h>
#include <stdint.h>

namespace asp
{
// one direction: blocks of A or, transposed, of A^T
struct Block8Dev
{
    const uint8_t *values;  // [blocks][128][128], row by row
    const uint8_t *scales;  // [blocks]: exponent + 127
    const uint8_t *scale_rows; // [blocks][512]: the same byte, once for each row of the block and each word, as tensor memory takes it
    const unsigned *col;    // [blocks]
    const uint4 *rows;      // block rows, longest first: {which one, its first block, number of its blocks, 0}
    unsigned n_block_rows, n_blocks, longest;
    unsigned n_rows, n_cols; // of the matrix: lengths of a row of Y and of X
};

struct Rows8Dev
{
    uint8_t *values; // [room][ld], ld a multiple of 128
    uint8_t *scales; // exponent + 127, in pieces of 512 bytes for 128 rows and 4 blocks of 128 columns, [n_cols / 512][pieces][512]; see scale_at
    uint64_t ld;
    unsigned pieces; // room / 128
    unsigned n_cols;
    unsigned n; // rows held
};
// Where the scale of a row and a block of 128 columns is. Inside a piece as tensor memory takes it: row 32 c + l in word c of lane l's 16 bytes, a
// byte for each of the 4 blocks.
#ifdef __CUDACC__
__host__ __device__
#endif
inline uint64_t scale_at(const Rows8Dev &x, uint64_t row, unsigned block)
{
    return ((uint64_t)(block / 4) * x.pieces + row / 128) * 512 + row % 32 * 16 + row / 32 % 4 * 4 + block % 4;
}

// a matrix in the caller's memory
struct Dense
{
    void *p;
    int dtype; // asp_dtype: f32, f16, bf16
    uint64_t ld;
};

cudaError_t launch_rows8_quantize(const Dense &x, unsigned n, const Rows8Dev &out, cudaStream_t st);
cudaError_t launch_rows8_restore(const Rows8Dev &x, const Dense &out, cudaStream_t st);
// where the values of A and of A^T go; those of A^T may be NULL
struct Block8Set
{
    uint8_t *values, *scales, *scale_rows;
};
// blocks [first, end) (from: the values of block `first` on); row: block row of each block; place: where it lies among the blocks of A^T
cudaError_t launch_block8_set(const Block8Dev &a, const unsigned *row, const unsigned *place, const Block8Set to[2], const void *from, int dtype, unsigned first, unsigned end, cudaStream_t st);
cudaError_t launch_block8_get(const Block8Dev &a, float *out, cudaStream_t st);
// a few rows, up to 32: X as it is (held == NULL) or in 8 bits. fault: a word that a kernel sets when it gives up a wait
cudaError_t launch_block8_few(const Block8Dev &a, const Dense *x, const Rows8Dev *held, unsigned n, const Dense &y, int sm_count, unsigned *fault, cudaStream_t st);
// fit: of block8_batch_room, the clusters of its kernel that run at once
cudaError_t block8_batch_room(unsigned fit[9]);
cudaError_t launch_block8_batch(const Block8Dev &a, const Dense *x, const Rows8Dev *held, unsigned n, const Dense &y, int sm_count, const unsigned *fit, unsigned *fault, cudaStream_t st);
// many rows in 8 bits
cudaError_t launch_block8_product(const Block8Dev &a, const Rows8Dev &x, const Dense &y, int sm_count, unsigned *fault, cudaStream_t st);
// The blocks by block column, in groups (Block8Pattern): everything about a group in one place, since each look-up waits for the one before
struct alignas(16) Block8Group
{
    unsigned block[2], row[2], col, n; // blocks of A, their block rows, their block column, how many
};
struct Block8Groups
{
    const Block8Group *groups[2];
    unsigned count[2], twos;
};
cudaError_t launch_block8_gradient(const Block8Dev &a, const Block8Groups &groups, const Rows8Dev &x, const Dense &dy, float *out, bool accumulate, int sm_count, unsigned *fault, cudaStream_t st);
} // namespace asp
#endif
