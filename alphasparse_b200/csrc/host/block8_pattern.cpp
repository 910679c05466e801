#include "block8_pattern.hpp"

#include <string.h>

#include <algorithm>
#include <numeric>

namespace asp
{
namespace host
{
namespace
{
void finish(Block8Side &s)
{
    const u32 n = (u32)s.ptr.size() - 1;
    s.order.resize(n);
    std::iota(s.order.begin(), s.order.end(), 0u);
    const auto len = [&](u32 r) { return s.ptr[r + 1] - s.ptr[r]; };
    std::stable_sort(s.order.begin(), s.order.end(), [&](u32 a, u32 b) { return len(a) > len(b); });
    s.longest = n ? len(s.order[0]) : 0;
}
} // namespace

asp_status make_pattern(u64 n_rows, u64 n_cols, const int64_t *block_ptr, const u32 *block_col, Block8Pattern &out, std::string &why)
{
    const u64 most = (1ull << 31) - kBlock8; // rows and columns are 32-bit coordinates of the kernels' copies
    if (n_rows == 0 || n_cols == 0 || n_rows > most || n_cols > most)
    {
        why = "matrix without rows or columns, or with 2^31 - 127 or more of them";
        return ASP_ERR_INVALID_ARG;
    }
    const u64 nr = (n_rows + kBlock8 - 1) / kBlock8, nc = (n_cols + kBlock8 - 1) / kBlock8;
    why = "block_ptr does not start at 0 or decreases";
    if (block_ptr[0] != 0) return ASP_ERR_BOUNDS;
    for (u64 r = 0; r < nr; r++)
        if (block_ptr[r + 1] < block_ptr[r]) return ASP_ERR_BOUNDS;
    const u64 n = (u64)block_ptr[nr];
    if (n >= (1u << 31) / kBlock8)
    {
        why = "2^24 or more blocks";
        return ASP_ERR_UNSUPPORTED;
    }
    why = "block columns of a block row must ascend and lie inside the matrix";
    if (n > 0 && !block_col) return ASP_ERR_INVALID_ARG;
    for (u64 r = 0; r < nr; r++)
        for (int64_t j = block_ptr[r]; j < block_ptr[r + 1]; j++)
            if (block_col[j] >= nc || (j > block_ptr[r] && block_col[j] <= block_col[j - 1])) return ASP_ERR_BOUNDS;
    why.clear();
    out = Block8Pattern();
    out.n_rows = n_rows, out.n_cols = n_cols;
    Block8Side &a = out.side[0], &t = out.side[1];
    a.ptr.assign(block_ptr, block_ptr + nr + 1);
    a.col.assign(block_col, block_col + n);
    t.ptr.assign(nc + 1, 0);
    for (u64 j = 0; j < n; j++) t.ptr[block_col[j] + 1]++;
    std::partial_sum(t.ptr.begin(), t.ptr.end(), t.ptr.begin());
    t.col.resize(n);
    out.place.resize(n);
    std::vector<u32> next(t.ptr.begin(), t.ptr.end() - 1);
    for (u32 r = 0; r < nr; r++)
        for (u32 j = a.ptr[r]; j < a.ptr[r + 1]; j++)
        {
            out.place[j] = next[a.col[j]]++;
            t.col[out.place[j]] = r;
        }
    out.from.resize(n);
    for (u64 j = 0; j < n; j++) out.from[out.place[j]] = (u32)j;
    for (u32 i = 0; i < n; i++) out.groups[0].push_back(i);
    for (u64 c = 0; c < nc; c++)
        for (u32 i = t.ptr[c]; i + 1 < t.ptr[c + 1]; i += 2) out.groups[1].push_back(i | 1u << 31);
    out.twos = (u32)out.groups[1].size();
    for (u64 c = 0; c < nc; c++)
        if ((t.ptr[c + 1] - t.ptr[c]) % 2) out.groups[1].push_back(t.ptr[c + 1] - 1);
    finish(a);
    finish(t);
    return ASP_OK;
}

void pattern_of(const Matrix &m, std::vector<int64_t> &block_ptr, std::vector<u32> &block_col)
{
    const u64 nr = (m.n_rows + kBlock8 - 1) / kBlock8, nc = (m.n_cols + kBlock8 - 1) / kBlock8;
    block_ptr.assign(nr + 1, 0);
    block_col.clear();
    std::vector<u64> seen(nc, nr); // the last block row that a block column was seen in
    for (u64 r = 0; r < nr; r++)
    {
        const size_t first = block_col.size();
        const u64 lo = m.rowptr[r * kBlock8], hi = m.rowptr[std::min(m.n_rows, (r + 1) * kBlock8)];
        for (u64 k = lo; k < hi; k++)
        {
            const u32 c = m.col[k] / (u32)kBlock8;
            if (seen[c] == r) continue;
            seen[c] = r;
            block_col.push_back(c);
        }
        std::sort(block_col.begin() + first, block_col.end());
        block_ptr[r + 1] = (int64_t)block_col.size();
    }
}

void block_values(const Matrix &m, const Block8Pattern &p, u64 first, u64 end, float *out)
{
    memset(out, 0, (end - first) * kBlock8 * kBlock8 * sizeof(float));
    const Block8Side &s = p.side[0];
    std::vector<u32> at(p.side[1].rows());
    for (u64 r = 0; r < s.rows(); r++)
    {
        if (s.ptr[r + 1] <= first || s.ptr[r] >= end) continue;
        for (u32 j = s.ptr[r]; j < s.ptr[r + 1]; j++) at[s.col[j]] = j;
        for (u64 row = r * kBlock8; row < std::min(m.n_rows, (r + 1) * kBlock8); row++)
            for (u64 k = m.rowptr[row]; k < m.rowptr[row + 1]; k++)
            {
                const u64 j = at[m.col[k] / kBlock8];
                if (j < first || j >= end) continue;
                const float v = m.val.es == 4 ? reinterpret_cast<const float *>(m.val.b.data())[k] : (float)reinterpret_cast<const double *>(m.val.b.data())[k];
                out[((j - first) * kBlock8 + row % kBlock8) * kBlock8 + m.col[k] % kBlock8] += v; // (an entry given twice counts twice, as in asp_spmv)
            }
    }
}
} // namespace host
} // namespace asp
