/*
 * asp_b200_block8.h -- products with block-sparse matrices in 8 bits, and their gradients.
 *
 * The reference multiplies one vector by a matrix of 32- or 64-bit values (code_builder.cc:1534-1550) and stores single
 * non-zeros; this part has no counterpart in it. It is for matrices that are sparse by blocks and multiplied by many rows at
 * once: the pruned weights of a network, in training and in serving.
 *
 * asp_block8: an n_rows x n_cols matrix A of which 128 x 128 blocks are stored, at multiples of 128 (the last ones may stick out; what
 * sticks out counts as zero). A block holds 8-bit floating-point values (e4m3: 4 exponent bits, 3 mantissa bits, largest 448) and
 * one scale.
 * asp_rows8: rows X (activations, gradients), e4m3 with one scale for each row and 128 columns.
 *
 * A scale is a power of two: the smallest 2^k, k >= -126, for which no finite magnitude of its block is above 448 * 2^k. Elements are
 * divided by it (exactly) and rounded to the nearest e4m3, ties to even; what is infinite or NaN becomes NaN and has no say in
 * the scale. What 8 bits stand for, q * 2^k, is thus within 2^-4 of the element, or 2^(k - 10) where that is more, and converting
 * it again gives it back (as long as the type has it: the largest 32-bit numbers round to 2^128). Powers of two are what the
 * tensor cores of sm_100a apply by themselves, and they keep q * 2^k exact in 16-bit types.
 *
 * Sums are in 32 bits and rounded to the result's type once, when they are stored. (Tensor cores cut off, by less than 2^-23 of the sum, whenever they add 32
 * columns to it; where the result has 32 bits they do so over 2048 columns at most, and what is more is added up rounded.
 * What is cut off goes by the factors' exponents: of the 16-bit types' subnormal numbers, in a gradient, that of the smallest normal one.) All entry points: device pointers aligned to their element type
 * unless said otherwise; ld = distance of two rows in elements, 0 = their length (what lies between two rows may be read, and is not written); asynchronous on the context's stream; the context
 * is of the device that the handle was created on. A handle's calls may be captured into a graph, which then needs the context and the handles for as
 * long as it is replayed; those that create and destroy may not. How many rows an asp_rows8 holds, and from which type, is as the calls were made or
 * captured; a replay does not change it. Calls of several contexts are in no order unless the caller gives them one.
 * n == 0 is allowed and touches no row. Results have the same bits every time.
 * Kernels that wait for their own copies and products give up after about two seconds (of work that takes microseconds). asp_synchronize alone says so (ASP_ERR_TIMEOUT): a
 * program that waits by its own stream, event or graph calls it, too, before it relies on what it waited for.
 */
#ifndef ASP_B200_BLOCK8_H
#define ASP_B200_BLOCK8_H

#include "asp_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ASP_BLOCK8_SIZE 128u
#define ASP_BLOCK8_APPLY_ROWS 32u /* most rows of one asp_block8_apply */

typedef struct asp_block8 asp_block8;
typedef struct asp_rows8 asp_rows8;

/* ---- rows in 8 bits ---- */

/* Room for up to max_rows rows of n_cols columns (a byte each, and a byte for each row and 128 columns; rows in whole 128s, columns in whole 512s at most). */
asp_status asp_rows8_create(asp_ctx *ctx, uint64_t max_rows, uint64_t n_cols, asp_rows8 **out);
void asp_rows8_destroy(asp_rows8 *rows);
/* X (n rows, ASP_F32 | ASP_F16 | ASP_BF16) to 8 bits; the handle then holds n rows. Rows behind them are left as they were. */
asp_status asp_rows8_quantize(asp_ctx *ctx, asp_rows8 *rows, const void *d_x, int dtype, uint64_t n, uint64_t ld);
/* What the rows held stand for, in any of the three types (rounded to nearest where the type cannot hold it: fp16 of 63488 and more has become 65536 in 8 bits, which
 * is infinite in fp16). */
asp_status asp_rows8_restore(asp_ctx *ctx, const asp_rows8 *rows, void *d_out, int dtype, uint64_t ld);
/* rows held */
uint64_t asp_rows8_count(const asp_rows8 *rows);

/* ---- the matrix ---- */

/* Stored blocks by block row: block_ptr has ceil(n_rows / 128) + 1 entries, block_col the block columns, ascending in each row
 * (ASP_ERR_BOUNDS otherwise). transposed != 0: the blocks are also kept transposed (a second byte per element), which products with
 * A^T need. All values are zero until asp_block8_set_values. */
asp_status asp_block8_create(asp_ctx *ctx, uint64_t n_rows, uint64_t n_cols, const int64_t *block_ptr, const uint32_t *block_col, int transposed, asp_block8 **out);
/* From an asp_matrix (asp_b200_host.h) before any dense-view node: the blocks with at least one of its entries, and its values, taken
 * as 32-bit ones. Returns when the values are on the device. */
asp_status asp_block8_from_matrix(asp_ctx *ctx, const void *matrix, int transposed, asp_block8 **out);
void asp_block8_destroy(asp_block8 *m);
uint64_t asp_block8_blocks(const asp_block8 *m);
/* the pattern: block_ptr and block_col as asp_block8_create takes them */
asp_status asp_block8_pattern(const asp_block8 *m, int64_t *block_ptr, uint32_t *block_col);
/* bytes of device memory */
uint64_t asp_block8_bytes(const asp_block8 *m);
/* New values for all stored blocks: 128 x 128 row-major each, one after the other in the order of block_col, ASP_F32 | ASP_F16 |
 * ASP_BF16, d_values 16-byte aligned. What sticks out of the matrix is taken as zero. */
asp_status asp_block8_set_values(asp_ctx *ctx, asp_block8 *m, const void *d_values, int dtype);
/* What the stored blocks stand for, 32 bits, in the same order; d_values 16-byte aligned. */
asp_status asp_block8_get_values(asp_ctx *ctx, const asp_block8 *m, float *d_values);

/* ---- products ---- */

/* y = A x for each of the n <= 32 rows x of X (ASP_F32 | ASP_F16 | ASP_BF16), converted to 8 bits on the way as asp_rows8_quantize does: serving.
 * One kernel, no room. (From 17 rows on every CTA converts more than it multiplies: by a full matrix of 4096 x 4096 and more asp_rows8_quantize and asp_block8_product
 * together take 3 to 7 % less, by smaller or sparser ones up to a quarter more.) transposed: y = A^T x, rows of n_rows in, of n_cols out. Y in any of the three types; it must not overlap X. */
asp_status asp_block8_apply(asp_ctx *ctx, const asp_block8 *m, int transposed, const void *d_x, int x_dtype, uint64_t n, uint64_t ldx, void *d_y, int y_dtype, uint64_t ldy);
/* y = A x (transposed: A^T x) for each of the rows held. Rows of y whose block row of A (or A^T) has no stored block are zero. */
asp_status asp_block8_product(asp_ctx *ctx, const asp_block8 *m, int transposed, const asp_rows8 *x, void *d_y, int y_dtype, uint64_t ldy);
/* The gradient of a loss by the stored blocks, from the gradient dY by the rows of y = A x and the rows x kept in 8 bits:
 * dA[block (i, j)] = sum over the rows of dy[128 i + .] x[128 j + .]^T, 32 bits, in the order of asp_block8_set_values; zero outside the
 * matrix. dY: ASP_F16 | ASP_BF16, the type that x was converted from (ASP_ERR_UNSUPPORTED otherwise), so that the products' factors
 * are exact; as many rows as x holds. What 8 bits have made of the type's largest numbers, 2^16 or 2^128, counts as that, although the type does not have it: rows
 * with numbers above 57344 (fp16) or 1.75 * 2^127 (bf16) take some forty times as long as others. Rows of dY on 16-byte boundaries (d_dy, and ld a multiple of 8) are copied by tiles, others take up to three times as
 * long. accumulate != 0: added to d_out. d_out 16-byte aligned. Sums of at most 1280 rows are added up, rounded, in one order; numbers below
 * 2^-126, in d_out or among these sums, may count as zero where something is added (L2 adds them up). */
asp_status asp_block8_gradient(asp_ctx *ctx, const asp_block8 *m, const asp_rows8 *x, const void *d_dy, int dtype, uint64_t ld, float *d_out, int accumulate);

#ifdef __cplusplus
}
#endif
#endif /* ASP_B200_BLOCK8_H */
