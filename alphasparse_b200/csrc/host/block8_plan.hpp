// How the kernels of block-sparse 8-bit matrices are cut up: rules on sizes, without a device.
#ifndef ASP_HOST_BLOCK8_PLAN_HPP
#define ASP_HOST_BLOCK8_PLAN_HPP

namespace asp
{
namespace host
{
// Products with a few rows (k_block8_few): CTAs that share the blocks of a block row. Two CTAs fit an SM, and all run at once: with twice as many as fit
// (8192 x 8192, one row, eight CTAs a block row) a call took 17.7 us instead of 13.2.
unsigned block8_few_split(unsigned n_block_rows, unsigned longest, int sm_count);

// Products with many rows (k_block8_product): rows of X a tile (64, 128, 192), and CTAs that share the blocks of a tile (1 to 8).
struct Block8ProductPlan
{
    unsigned tile, split;
};
constexpr unsigned kBlock8ProductRows = 192;
Block8ProductPlan block8_product_plan(unsigned n_block_rows, unsigned n_blocks, unsigned longest, unsigned n, int sm_count);

// Gradients (k_block8_gradient): blocks of a block column that share x at most (1, 2), and CTAs that share the rows of a group (1, 2, 4, 8).
// blocks: stored ones; twos: groups of two where there are two at most.
struct Block8GradientPlan
{
    unsigned most, split;
};
constexpr unsigned kBlock8GradientRows = 64; // rows a step
Block8GradientPlan block8_gradient_plan(unsigned blocks, unsigned twos, unsigned n, int sm_count);
} // namespace host
} // namespace asp
#endif
