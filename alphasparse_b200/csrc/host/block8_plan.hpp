// How the kernels of block-sparse 8-bit matrices are cut up: rules on sizes, without a device.
#ifndef ASP_HOST_BLOCK8_PLAN_HPP
#define ASP_HOST_BLOCK8_PLAN_HPP

namespace asp
{
namespace host
{
// CTAs that share work are a cluster of 1 to 8; fit[s]: how many clusters of s CTAs run at once, two CTAs an SM or one, as the kernel takes (ClusterRoom).
// Those that do not fit would run after the others: 5000 x 5000, one row, 7 CTAs a block row, take 13.1 us, 6, which fit, 8.3.

// Blocks in one sum of a tensor core, where the result has 32 bits
constexpr unsigned kBlock8Sum = 16;

// Products with up to 32 rows: by the kernel for few rows or for a batch (k_block8_few, k_block8_batch)?
bool block8_batch(unsigned n_block_rows, unsigned longest, unsigned n, bool wide, int sm_count, const unsigned *fit);
// and CTAs that share the blocks of a block row
unsigned block8_few_split(unsigned n_block_rows, unsigned longest, unsigned per, const unsigned *fit); // per: blocks whose rows of X are converted at once
unsigned block8_batch_split(unsigned n_block_rows, unsigned longest, int sm_count, const unsigned *fit);

// Products with many rows (k_block8_product): rows of X a tile (64, 128, 192), and CTAs that share the blocks of a tile (1 to 8).
struct Block8ProductPlan
{
    unsigned tile, split;
};
constexpr unsigned kBlock8ProductRows = 192;
Block8ProductPlan block8_product_plan(unsigned n_block_rows, unsigned n_blocks, unsigned longest, unsigned n, int sm_count, const unsigned *fit);

// Gradients (k_block8_gradient): blocks of a block column that share x at most (1, 2), and CTAs that share the rows of a group (1, 2, 4, 8).
// blocks: stored ones; twos: groups of two where there are two at most.
struct Block8GradientPlan
{
    unsigned most, split;
};
constexpr unsigned kBlock8GradientRows = 64; // rows a step
Block8GradientPlan block8_gradient_plan(unsigned blocks, unsigned twos, unsigned n, int sm_count, const unsigned *fit);
} // namespace host
} // namespace asp
#endif
