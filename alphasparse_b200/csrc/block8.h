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
    const unsigned *ptr;    // [block rows + 1]
    const unsigned *col;    // [blocks]
    const unsigned *order;  // block rows, longest first
    unsigned n_block_rows, n_blocks, longest;
    unsigned n_rows, n_cols; // of the matrix: lengths of a row of Y and of X
};

struct Rows8Dev
{
    uint8_t *values; // [room][ld], ld a multiple of 128
    uint8_t *scales; // [blocks of 128 columns][ld_scales]: exponent + 127
    uint64_t ld, ld_scales;
    unsigned n_cols;
    unsigned n; // rows held
};

// a matrix in the caller's memory
struct Dense
{
    void *p;
    int dtype; // asp_dtype: f32, f16, bf16
    uint64_t ld;
};

cudaError_t launch_rows8_quantize(const Dense &x, unsigned n, const Rows8Dev &out, cudaStream_t st);
cudaError_t launch_rows8_restore(const Rows8Dev &x, const Dense &out, cudaStream_t st);
// blocks [first, end) of `values` (values of block `first` at its start); row: block row of each block; place: where it lies among the
// blocks of A^T, whose values and scales may be NULL
cudaError_t launch_block8_set(const Block8Dev &a, const unsigned *row, const unsigned *place, uint8_t *values, uint8_t *scales, uint8_t *values_t, uint8_t *scales_t, const void *from,
                              int dtype, unsigned first, unsigned end, cudaStream_t st);
cudaError_t launch_block8_get(const Block8Dev &a, float *out, cudaStream_t st);
// a few rows: X as it is (held == NULL) or in 8 bits
cudaError_t launch_block8_few(const Block8Dev &a, const Dense *x, const Rows8Dev *held, unsigned n, const Dense &y, int sm_count, cudaStream_t st);
// row: block row of each block
cudaError_t launch_block8_gradient(const Block8Dev &a, const unsigned *row, const Rows8Dev &x, const Dense &dy, float *out, bool accumulate, int sm_count, cudaStream_t st);
} // namespace asp
#endif
