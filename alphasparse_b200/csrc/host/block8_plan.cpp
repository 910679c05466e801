#include "block8_plan.hpp"

#include <stdint.h>

#include <algorithm>

namespace asp
{
namespace host
{
namespace
{
// the largest cluster for each block row of which all run at once, on at most so many CTAs
unsigned largest(unsigned n_block_rows, unsigned longest, unsigned ctas, const unsigned *fit)
{
    for (unsigned s = std::min(8u, longest); s > 1; s--)
        if (n_block_rows <= fit[s] && n_block_rows <= ctas / s) return s;
    return 1;
}
} // namespace

// What a CTA converts and multiplies at once is not shared out: a cluster's start and sum cost more (8 rows of 12000 x 384 4.0 us instead of 5.1, 14 rows of 4096 x 256 4.0 instead of 4.8).
unsigned block8_few_split(unsigned n_block_rows, unsigned longest, unsigned per, const unsigned *fit) { return longest <= per ? 1 : largest(n_block_rows, longest, ~0u, fit); }

// One CTA an SM where its blocks are few (16 rows of 4096 x 4096: 8 blocks to each of 128 CTAs 7.5 us, 4 to each of 256 8.2), two where they are many (one row of 8192 x 8192:
// 32 to 128 11.9 us, 16 to 256 9.9).
unsigned block8_batch_split(unsigned n_block_rows, unsigned longest, int sm_count, const unsigned *fit)
{
    const unsigned one = largest(n_block_rows, longest, (unsigned)sm_count, fit);
    return (longest + one - 1) / one <= 8 ? one : largest(n_block_rows, longest, ~0u, fit);
}

// Where a CTA has many blocks tcgen05 takes them as fast as they come, while its start (tensor memory, barriers, a step's way through three kinds of
// warps) costs 0.7 us more. One row: 4096 x 4096 (4 blocks a CTA) 6.0 us by the kernel for few rows and 6.2 by that for a batch, 2048 x 8192, half of it (5), 6.0 and 5.6,
// 8192 x 8192 (16) 13.6 and 9.9. With more than 8 rows mma.sync takes longer than the blocks to come: 16 rows of 4096 x 4096 8.4 and 7.5, of 4001 x 2047 in 32 bits
// (2) 6.0 and 7.0, 32 rows of 8192 x 8192 31.2 and 17.6, of 1024 x 1024 (1) 4.4 and 5.2.
// wide: the result has 32 bits. A sum of the kernel for a batch is all of a CTA's blocks, cut off each time something is added (16 blocks: 6e-7); the other one rounds
// after each block.
bool block8_batch(unsigned n_block_rows, unsigned longest, unsigned n, bool wide, int sm_count, const unsigned *fit)
{
    const unsigned most = largest(n_block_rows, longest, ~0u, fit), split = block8_batch_split(n_block_rows, longest, sm_count, fit);
    return (longest + most - 1) / most >= (n <= 8 ? 5 : 3) && !(wide && (longest + split - 1) / split > kBlock8Sum);
}

// A step takes as long as its 16 KB of A and its rows of X take to pass shared memory twice, at 128 bytes a clock; a tile costs some 2500 clocks beside
// its steps, and as much again where sums of several CTAs are added up. Against every tile and power-of-two split on 14 shapes (40 to 8192 rows, matrices of
// 512 to 8192): within 7 % of the best; without splits 40 rows, 4096 x 4096, take 12.3 us instead of 8.6, with tiles of 192 only 700 rows, 512 x 512, 7.1 instead of 5.2.
Block8ProductPlan block8_product_plan(unsigned n_block_rows, unsigned n_blocks, unsigned longest, unsigned n, int sm_count, const unsigned *fit)
{
    Block8ProductPlan best = {kBlock8ProductRows, 1};
    double least = -1;
    for (unsigned t = kBlock8ProductRows; t >= 64; t -= 64)
        for (unsigned s = 1; s <= 8; s++)
        {
            const uint64_t tiles = (uint64_t)n_block_rows * ((n + t - 1) / t), waves = (tiles + sm_count - 1) / sm_count;
            if (s > 1 && longest < 2 * s) break;
            if (s > 1 && tiles > fit[s]) continue;
            const double steps = s > 1 ? (double)((longest + s - 1) / s) : (double)n_blocks / n_block_rows;
            const double cost = waves * ((s > 1 ? 5000.0 : 2500.0) + steps * (16384 + 128.0 * t) / 64);
            if (least < 0 || cost < least) least = cost, best = {t, s};
        }
    return best;
}

// Clocks of a step by what passes shared memory; a call takes some 10000 clocks beside the steps of its longest CTA, and 3000 more for each CTA that adds to a block
// that it shares (single blocks only: their sums stay in tensor memory).
Block8GradientPlan block8_gradient_plan(unsigned blocks, unsigned twos, unsigned n, int sm_count, const unsigned *fit)
{
    const unsigned steps = (unsigned)(((uint64_t)n + kBlock8GradientRows - 1) / kBlock8GradientRows);
    const auto clocks = [&](uint64_t groups, double step) { return (groups + sm_count - 1) / sm_count * step * steps; };
    Block8GradientPlan best = {1, 1};
    double least = clocks(blocks, 640);
    if (twos && clocks(blocks - twos, 960) < least) least = clocks(blocks - twos, 960), best.most = 2; // (with what is added up by L2)
    for (unsigned s = 2; s <= 8 && s <= steps; s *= 2)
    {
        if (blocks > fit[s]) break;
        const double time = 640.0 * ((steps + s - 1) / s) + 3000.0 * s;
        if (time < least) least = time, best = {1, s};
    }
    return best;
}
} // namespace host
} // namespace asp
