// The pattern of a block-sparse 8-bit matrix (asp_b200_block8.h) and what its kernels are told of it.
#ifndef ASP_HOST_BLOCK8_PATTERN_HPP
#define ASP_HOST_BLOCK8_PATTERN_HPP
#include <stdint.h>

#include <string>
#include <vector>

#include "format.hpp"

namespace asp
{
namespace host
{
constexpr u64 kBlock8 = 128;

// One direction of the products: block rows with the blocks that a sum over them takes
struct Block8Side
{
    std::vector<u32> ptr;   // block rows + 1
    std::vector<u32> col;   // block column of each stored block, ascending in a row
    std::vector<u32> order; // block rows, those with most blocks first: with rows of all lengths in flight the longest do not start last
    u32 longest = 0;
    u32 rows() const { return (u32)order.size(); }
};

struct Block8Pattern
{
    u64 n_rows = 0, n_cols = 0;
    Block8Side side[2];      // of A, of A^T
    std::vector<u32> place;  // where block i of A lies among the blocks of A^T
    std::vector<u32> from;   // the other way: which block of A is block i of A^T
    // Blocks of A^T one by one, and in twos of one block column of A, those that stay alone last: where the group begins, and in bit 31 whether there are two
    std::vector<u32> groups[2];
    u32 twos = 0; // groups of two blocks among the latter
    u64 blocks() const { return side[0].col.size(); }
};

// ASP_ERR_INVALID_ARG: no matrix of this size; ASP_ERR_BOUNDS: the two arrays do not describe blocks of it
asp_status make_pattern(u64 n_rows, u64 n_cols, const int64_t *block_ptr, const u32 *block_col, Block8Pattern &out, std::string &why);
// the blocks of a matrix that have an entry
void pattern_of(const Matrix &m, std::vector<int64_t> &block_ptr, std::vector<u32> &block_col);
// values of blocks [first, end), 128 x 128 each, zero where the matrix has no entry
void block_values(const Matrix &m, const Block8Pattern &p, u64 first, u64 end, float *out);
} // namespace host
} // namespace asp
#endif
