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

// Clocks of a step by what passes shared memory; a CTA takes some 8000 clocks beside its steps and 2000 more for each block that it stores, and each
// further CTA of a cluster another 2000 for what it adds to. With more CTAs than SMs the last ones end on average half a CTA's time after the others. Against all 12
// choices on 8 shapes (300 to 8192 rows, 16 to 2048 blocks): within 15 % of the best, where the worst choice costs 2 to 10 times as much.
Block8GradientPlan block8_gradient_plan(const unsigned sizes[4][4], unsigned n, int sm_count)
{
    static const double clocks[4] = {640, 896, 1280, 1536};
    const unsigned steps = (unsigned)(((uint64_t)n + kBlock8GradientRows - 1) / kBlock8GradientRows);
    Block8GradientPlan best = {1, 1};
    double least = -1;
    for (unsigned m = 1; m <= 4; m++)
        for (unsigned s = 1; s <= 4 && s <= steps; s *= 2)
        {
            double all = 0, longest = 0;
            uint64_t groups = 0;
            for (unsigned k = 0; k < m; k++)
            {
                if (sizes[m - 1][k] == 0) continue;
                const double one = 8000 + 2000.0 * (k + 1) * (s > 1 ? 2 : 1) + clocks[k] * ((steps + s - 1) / s);
                groups += sizes[m - 1][k];
                all += one * sizes[m - 1][k] * s;
                longest = one; // (of more blocks, longer)
            }
            const double time = groups * s <= (unsigned)sm_count ? longest : std::max(longest, all / sm_count) + longest / 2;
            if (least < 0 || time < least) least = time, best = {m, s};
        }
    return best;
}
} // namespace host
} // namespace asp
