#include "block8_plan.hpp"

#include <stdint.h>

#include <algorithm>

namespace asp
{
namespace host
{
unsigned block8_few_split(unsigned n_block_rows, unsigned longest, int sm_count)
{
    return std::max(1u, std::min({8u, longest, 2u * (unsigned)sm_count / n_block_rows}));
}

// A step takes as long as its 16 KB of A and its rows of X take to pass shared memory twice, at 128 bytes a clock; a tile costs some 2500 clocks beside
// its steps, and as much again where sums of several CTAs are added up. Against every tile and power-of-two split on 14 shapes (40 to 8192 rows, matrices of
// 512 to 8192): within 7 % of the best; without splits 40 rows, 4096 x 4096, take 12.3 us instead of 8.6, with tiles of 192 only 700 rows, 512 x 512, 7.1 instead of 5.2.
Block8ProductPlan block8_product_plan(unsigned n_block_rows, unsigned n_blocks, unsigned longest, unsigned n, int sm_count)
{
    Block8ProductPlan best = {kBlock8ProductRows, 1};
    double least = -1;
    for (unsigned t = kBlock8ProductRows; t >= 64; t -= 64)
        for (unsigned s = 1; s <= 8; s++)
        {
            const uint64_t tiles = (uint64_t)n_block_rows * ((n + t - 1) / t), waves = (tiles + sm_count - 1) / sm_count;
            // (clusters find no room on the last SMs of a part of the chip)
            if (s > 1 && (tiles * s * 10 > (uint64_t)sm_count * 9 || longest < 2 * s)) break;
            const double steps = s > 1 ? (double)((longest + s - 1) / s) : (double)n_blocks / n_block_rows;
            const double cost = waves * ((s > 1 ? 5000.0 : 2500.0) + steps * (16384 + 128.0 * t) / 64);
            if (least < 0 || cost < least) least = cost, best = {t, s};
        }
    return best;
}

// Clocks of a step by what passes shared memory; a call takes some 10000 clocks beside the steps of its longest CTA, and 3000 more for each CTA that adds to a block
// that it shares (single blocks only: their sums stay in tensor memory).
Block8GradientPlan block8_gradient_plan(unsigned blocks, unsigned twos, unsigned n, int sm_count)
{
    const unsigned steps = (unsigned)(((uint64_t)n + kBlock8GradientRows - 1) / kBlock8GradientRows);
    const auto clocks = [&](uint64_t groups, double step) { return (groups + sm_count - 1) / sm_count * step * steps; };
    Block8GradientPlan best = {1, 1};
    double least = clocks(blocks, 640);
    if (twos && clocks(blocks - twos, 960) < least) least = clocks(blocks - twos, 960), best.most = 2; // (with what is added up by L2)
    // (clusters find no room on the last SMs of a part of the chip)
    for (unsigned s = 2; s <= 8 && s <= steps && (uint64_t)blocks * s * 10 <= (uint64_t)sm_count * 9; s *= 2)
    {
        const double time = 640.0 * ((steps + s - 1) / s) + 3000.0 * s;
        if (time < least) least = time, best = {1, s};
    }
    return best;
}
} // namespace host
} // namespace asp
