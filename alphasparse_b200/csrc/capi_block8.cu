// C ABI of block-sparse 8-bit matrices (include/asp_b200_block8.h): handles, checks, launches.
#include <algorithm>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/asp_b200_block8.h"
#include "block8.h"
#include "ctx.h"
#include "host/block8_pattern.hpp"
#include "host/handles.hpp"

using asp::cuda_fail;
using asp::fail;

namespace
{
struct Room
{
    void *base = nullptr;
    size_t got = 0;
    int device = 0;
    ~Room() { asp::device_free(device, base, got); }
};
} // namespace

struct asp_rows8
{
    Room room;
    asp::Rows8Dev dev = {};
    uint64_t max_rows = 0;
    int from = -1; // type of what is held
};

struct asp_block8
{
    Room room;
    asp::host::Block8Pattern pattern;
    asp::Block8Dev side[2] = {};
    const unsigned *row = nullptr, *place = nullptr;
    asp::Block8Groups groups = {};
    asp::Block8Set set[2] = {};
    bool transposed = false;
    size_t bytes = 0;
};

namespace
{
using asp::host::kBlock8;

uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }
int size_of(int dtype) { return dtype == ASP_F32 ? 4 : dtype == ASP_F16 || dtype == ASP_BF16 ? 2 : 0; }

// a matrix in the caller's memory
asp_status look_at(const void *p, int dtype, uint64_t n, uint64_t width, uint64_t ld, const char *what, asp::Dense *out)
{
    const int size = size_of(dtype);
    if (size == 0) return fail(ASP_ERR_UNSUPPORTED, std::string(what) + ": f32, f16 or bf16");
    if (ld == 0) ld = width;
    if (ld < width) return fail(ASP_ERR_INVALID_ARG, std::string(what) + ": ld is less than the length of a row");
    if (ld > (1ull << 40)) return fail(ASP_ERR_INVALID_ARG, std::string(what) + ": ld is above 2^40");
    if (n > 0 && !p) return fail(ASP_ERR_INVALID_ARG, std::string(what) + " is NULL");
    if ((uintptr_t)p % size) return fail(ASP_ERR_INVALID_ARG, std::string(what) + " is not aligned to its element type");
    out->p = const_cast<void *>(p), out->dtype = dtype, out->ld = ld;
    return ASP_OK;
}

struct Piece
{
    size_t at = 0, bytes = 0;
};

template <class F> asp_status guarded(F f)
{
    try
    {
        return f();
    }
    catch (const std::bad_alloc &)
    {
        return fail(ASP_ERR_ALLOC, "host allocation failed");
    }
}

asp_status upload(asp_ctx *ctx, std::unique_ptr<asp_block8> &m)
{
    const asp::host::Block8Pattern &p = m->pattern;
    const uint64_t n = p.blocks();
    size_t at = 0;
    auto take = [&](size_t bytes) {
        Piece r;
        r.at = at, r.bytes = bytes;
        at += up(std::max<size_t>(bytes, 1), 1024);
        return r;
    };
    const int sides = m->transposed ? 2 : 1;
    Piece values[2], scales[2], scale_rows[2], col[2], rows_of[2];
    std::vector<uint4> by_length[2];
    // What is copied comes first and lies together: everything between the first array and the last is written by the copy.
    for (int s = 0; s < sides; s++)
    {
        col[s] = take(n * 4);
        for (const uint32_t r : p.side[s].order) by_length[s].push_back({r, p.side[s].ptr[r], p.side[s].ptr[r + 1] - p.side[s].ptr[r], 0});
        rows_of[s] = take(by_length[s].size() * sizeof(uint4));
    }
    const Piece row = take(n * 4), place = take(n * 4);
    std::vector<uint32_t> rows(n);
    for (uint32_t r = 0; r < p.side[0].rows(); r++) std::fill(rows.begin() + p.side[0].ptr[r], rows.begin() + p.side[0].ptr[r + 1], r);
    Piece groups[2];
    std::vector<asp::Block8Group> group[2];
    for (int g = 0; g < 2; g++)
    {
        for (const uint32_t u : p.groups[g])
        {
            asp::Block8Group of = {};
            of.n = 1 + (u >> 31);
            for (uint32_t k = 0; k < of.n; k++) of.block[k] = p.from[(u & 0x7fffffffu) + k], of.row[k] = rows[of.block[k]];
            of.col = p.side[0].col[of.block[0]];
            group[g].push_back(of);
        }
        groups[g] = take(group[g].size() * sizeof(asp::Block8Group));
    }
    for (int s = 0; s < sides; s++)
    {
        values[s] = take(n * kBlock8 * kBlock8);
        scales[s] = take(n);
        scale_rows[s] = take(n * 512);
    }
    ASP_ON_DEVICE(ctx);
    m->room.device = ctx->device;
    cudaError_t e = asp::device_alloc(ctx->device, at, &m->room.base, &m->room.got);
    if (e != cudaSuccess)
    {
        m->room.base = nullptr;
        return fail(ASP_ERR_ALLOC, std::string("device memory of the matrix: ") + cudaGetErrorString(e));
    }
    m->bytes = at;
    unsigned char *base = (unsigned char *)m->room.base;
    std::vector<asp::Stager::Segment> segments;
    auto send = [&](const Piece &to, const void *from) {
        if (to.bytes) segments.push_back({to.at, from, to.bytes});
        return reinterpret_cast<const unsigned *>(base + to.at);
    };
    for (int s = 0; s < sides; s++)
    {
        const asp::host::Block8Side &h = p.side[s];
        asp::Block8Dev &d = m->side[s];
        d.values = m->set[s].values = base + values[s].at;
        d.scales = m->set[s].scales = base + scales[s].at;
        d.scale_rows = m->set[s].scale_rows = base + scale_rows[s].at;
        d.col = send(col[s], h.col.data());
        d.rows = reinterpret_cast<const uint4 *>(send(rows_of[s], by_length[s].data()));
        d.n_block_rows = h.rows(), d.n_blocks = (unsigned)n, d.longest = h.longest;
        d.n_rows = (unsigned)(s ? p.n_cols : p.n_rows), d.n_cols = (unsigned)(s ? p.n_rows : p.n_cols);
        e = cudaMemsetAsync(base + values[s].at, 0, values[s].bytes, ctx->stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(base + scales[s].at, 127, scales[s].bytes, ctx->stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(base + scale_rows[s].at, 127, scale_rows[s].bytes, ctx->stream);
        if (e != cudaSuccess) return cuda_fail(e, "clearing the values");
    }
    m->row = send(row, rows.data());
    m->place = send(place, p.place.data());
    for (int g = 0; g < 2; g++)
    {
        m->groups.groups[g] = reinterpret_cast<const asp::Block8Group *>(send(groups[g], group[g].data()));
        m->groups.count[g] = (unsigned)p.groups[g].size();
    }
    m->groups.twos = p.twos;
    e = ctx->stager.to_device(m->room.base, segments, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) return cuda_fail(e, "upload of the pattern");
    return ASP_OK;
}

asp_status create(asp_ctx *ctx, uint64_t n_rows, uint64_t n_cols, const int64_t *block_ptr, const uint32_t *block_col, int transposed, std::unique_ptr<asp_block8> &m)
{
    m.reset(new asp_block8());
    std::string why;
    const asp_status st = asp::host::make_pattern(n_rows, n_cols, block_ptr, block_col, m->pattern, why);
    if (st != ASP_OK) return fail(st, why);
    if (!ctx) return fail(ASP_ERR_INVALID_ARG, "ctx is NULL");
    m->transposed = transposed != 0;
    return upload(ctx, m);
}

asp_status same_device(const asp_ctx *ctx, const Room &room)
{
    return ctx->device == room.device ? ASP_OK : fail(ASP_ERR_INVALID_ARG, "the context is of another device than the handle");
}

asp_status side_of(const asp_block8 *m, int transposed, const asp::Block8Dev **out)
{
    if (transposed && !m->transposed) return fail(ASP_ERR_UNSUPPORTED, "the matrix was created without its transposed blocks");
    *out = &m->side[transposed ? 1 : 0];
    return ASP_OK;
}

asp_status launched(cudaError_t e) { return e == cudaSuccess ? ASP_OK : cuda_fail(e, "kernel launch"); }
#define ASP_TRY(call)                            \
    do                                           \
    {                                            \
        const asp_status s__ = (call);           \
        if (s__ != ASP_OK) return s__;           \
    } while (0)
} // namespace

extern "C" {

asp_status asp_rows8_create(asp_ctx *ctx, uint64_t max_rows, uint64_t n_cols, asp_rows8 **out)
{
    if (!out) return fail(ASP_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (max_rows == 0 || n_cols == 0 || max_rows > (1ull << 31) - kBlock8 || n_cols > (1ull << 31) - kBlock8)
        return fail(ASP_ERR_INVALID_ARG, "no rows or columns, or 2^31 - 127 or more of them");
    if (!ctx) return fail(ASP_ERR_INVALID_ARG, "ctx is NULL");
    return guarded([&]() -> asp_status {
        std::unique_ptr<asp_rows8> r(new asp_rows8());
        r->max_rows = max_rows;
        r->dev.ld = up(n_cols, kBlock8);
        r->dev.pieces = (unsigned)(up(max_rows, kBlock8) / kBlock8);
        r->dev.n_cols = (unsigned)n_cols;
        const uint64_t values = up(max_rows * r->dev.ld, 1024);
        ASP_ON_DEVICE(ctx);
        r->room.device = ctx->device;
        const cudaError_t e = asp::device_alloc(ctx->device, values + up(r->dev.ld, 4 * kBlock8) / (4 * kBlock8) * r->dev.pieces * 512, &r->room.base, &r->room.got);
        if (e != cudaSuccess)
        {
            r->room.base = nullptr;
            return fail(ASP_ERR_ALLOC, std::string("device memory of the rows: ") + cudaGetErrorString(e));
        }
        r->dev.values = (uint8_t *)r->room.base;
        r->dev.scales = r->dev.values + values;
        *out = r.release();
        return ASP_OK;
    });
}

void asp_rows8_destroy(asp_rows8 *rows) { delete rows; }
uint64_t asp_rows8_count(const asp_rows8 *rows) { return rows ? rows->dev.n : 0; }

asp_status asp_rows8_quantize(asp_ctx *ctx, asp_rows8 *rows, const void *d_x, int dtype, uint64_t n, uint64_t ld)
{
    if (!ctx || !rows) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    if (n > rows->max_rows) return fail(ASP_ERR_INVALID_ARG, "more rows than there is room for");
    asp::Dense x;
    ASP_TRY(look_at(d_x, dtype, n, rows->dev.n_cols, ld, "x", &x));
    ASP_TRY(same_device(ctx, rows->room));
    ASP_ON_DEVICE(ctx);
    ASP_TRY(launched(asp::launch_rows8_quantize(x, (unsigned)n, rows->dev, ctx->stream)));
    rows->dev.n = (unsigned)n;
    rows->from = dtype;
    return ASP_OK;
}

asp_status asp_rows8_restore(asp_ctx *ctx, const asp_rows8 *rows, void *d_out, int dtype, uint64_t ld)
{
    if (!ctx || !rows) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    asp::Dense out;
    ASP_TRY(look_at(d_out, dtype, rows->dev.n, rows->dev.n_cols, ld, "out", &out));
    ASP_TRY(same_device(ctx, rows->room));
    ASP_ON_DEVICE(ctx);
    return launched(asp::launch_rows8_restore(rows->dev, out, ctx->stream));
}

asp_status asp_block8_create(asp_ctx *ctx, uint64_t n_rows, uint64_t n_cols, const int64_t *block_ptr, const uint32_t *block_col, int transposed, asp_block8 **out)
{
    if (!out) return fail(ASP_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!block_ptr) return fail(ASP_ERR_INVALID_ARG, "block_ptr is NULL");
    return guarded([&]() -> asp_status {
        std::unique_ptr<asp_block8> m;
        ASP_TRY(create(ctx, n_rows, n_cols, block_ptr, block_col, transposed, m));
        *out = m.release();
        return ASP_OK;
    });
}

asp_status asp_block8_from_matrix(asp_ctx *ctx, const void *matrix, int transposed, asp_block8 **out)
{
    if (!out) return fail(ASP_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!matrix) return fail(ASP_ERR_INVALID_ARG, "matrix is NULL");
    const asp::host::Matrix &h = *static_cast<const asp_matrix *>(matrix)->m;
    if (h.is_sorted || h.is_blocked || h.is_compressed) return fail(ASP_ERR_UNSUPPORTED, "the matrix has been through dense-view nodes");
    return guarded([&]() -> asp_status {
        std::vector<int64_t> ptr;
        std::vector<uint32_t> col;
        asp::host::pattern_of(h, ptr, col);
        std::unique_ptr<asp_block8> m;
        ASP_TRY(create(ctx, h.n_rows, h.n_cols, ptr.data(), col.data(), transposed, m));
        // 64 MB of values at a time
        const uint64_t n = m->pattern.blocks(), most = std::min<uint64_t>(n, 1024);
        std::vector<float> values(most * kBlock8 * kBlock8);
        ASP_ON_DEVICE(ctx);
        Room room;
        room.device = ctx->device;
        cudaError_t e = n ? asp::device_alloc(ctx->device, values.size() * 4, &room.base, &room.got) : cudaSuccess;
        if (e != cudaSuccess)
        {
            room.base = nullptr;
            return fail(ASP_ERR_ALLOC, std::string("device memory of the values: ") + cudaGetErrorString(e));
        }
        for (uint64_t b = 0; b < n && e == cudaSuccess; b += most)
        {
            const uint64_t end = std::min(n, b + most);
            asp::host::block_values(h, m->pattern, b, end, values.data());
            e = ctx->stager.to_device(room.base, values.data(), (end - b) * kBlock8 * kBlock8 * 4, ctx->stream);
            if (e == cudaSuccess)
                e = asp::launch_block8_set(m->side[0], m->row, m->place, m->set, room.base, ASP_F32, (unsigned)b, (unsigned)end, ctx->stream);
        }
        const cudaError_t done = cudaStreamSynchronize(ctx->stream);
        if (e == cudaSuccess) e = done;
        if (e != cudaSuccess) return cuda_fail(e, "upload of the values");
        *out = m.release();
        return ASP_OK;
    });
}

void asp_block8_destroy(asp_block8 *m) { delete m; }
uint64_t asp_block8_blocks(const asp_block8 *m) { return m ? m->pattern.blocks() : 0; }
uint64_t asp_block8_bytes(const asp_block8 *m) { return m ? m->bytes : 0; }

asp_status asp_block8_pattern(const asp_block8 *m, int64_t *block_ptr, uint32_t *block_col)
{
    if (!m || !block_ptr || (!block_col && m->pattern.blocks())) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    const asp::host::Block8Side &s = m->pattern.side[0];
    std::copy(s.ptr.begin(), s.ptr.end(), block_ptr);
    std::copy(s.col.begin(), s.col.end(), block_col);
    return ASP_OK;
}

asp_status asp_block8_set_values(asp_ctx *ctx, asp_block8 *m, const void *d_values, int dtype)
{
    if (!ctx || !m) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    if (size_of(dtype) == 0) return fail(ASP_ERR_UNSUPPORTED, "values: f32, f16 or bf16");
    if ((!d_values && m->pattern.blocks()) || (uintptr_t)d_values % 16) return fail(ASP_ERR_INVALID_ARG, "values are NULL or not on a 16-byte boundary");
    ASP_TRY(same_device(ctx, m->room));
    ASP_ON_DEVICE(ctx);
    return launched(asp::launch_block8_set(m->side[0], m->row, m->place, m->set, d_values, dtype, 0, (unsigned)m->pattern.blocks(), ctx->stream));
}

asp_status asp_block8_get_values(asp_ctx *ctx, const asp_block8 *m, float *d_values)
{
    if (!ctx || !m) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    if ((!d_values && m->pattern.blocks()) || (uintptr_t)d_values % 16) return fail(ASP_ERR_INVALID_ARG, "values are NULL or not on a 16-byte boundary");
    ASP_TRY(same_device(ctx, m->room));
    ASP_ON_DEVICE(ctx);
    return launched(asp::launch_block8_get(m->side[0], d_values, ctx->stream));
}

asp_status asp_block8_apply(asp_ctx *ctx, const asp_block8 *m, int transposed, const void *d_x, int x_dtype, uint64_t n, uint64_t ldx, void *d_y, int y_dtype, uint64_t ldy)
{
    if (!ctx || !m) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    if (n > ASP_BLOCK8_APPLY_ROWS) return fail(ASP_ERR_INVALID_ARG, "more than 32 rows: asp_rows8_quantize and asp_block8_product take them");
    const asp::Block8Dev *a;
    ASP_TRY(side_of(m, transposed, &a));
    asp::Dense x, y;
    ASP_TRY(look_at(d_x, x_dtype, n, a->n_cols, ldx, "x", &x));
    ASP_TRY(look_at(d_y, y_dtype, n, a->n_rows, ldy, "y", &y));
    ASP_TRY(same_device(ctx, m->room));
    ASP_ON_DEVICE(ctx);
    return launched(asp::launch_block8_few(*a, &x, nullptr, (unsigned)n, y, ctx->sm_count, ctx->fault, ctx->stream));
}

asp_status asp_block8_product(asp_ctx *ctx, const asp_block8 *m, int transposed, const asp_rows8 *x, void *d_y, int y_dtype, uint64_t ldy)
{
    if (!ctx || !m || !x) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    const asp::Block8Dev *a;
    ASP_TRY(side_of(m, transposed, &a));
    if (x->dev.n_cols != a->n_cols) return fail(ASP_ERR_INVALID_ARG, "the rows have another length than those of the matrix");
    asp::Dense y;
    ASP_TRY(look_at(d_y, y_dtype, x->dev.n, a->n_rows, ldy, "y", &y));
    ASP_TRY(same_device(ctx, m->room));
    ASP_TRY(same_device(ctx, x->room));
    ASP_ON_DEVICE(ctx);
    if (x->dev.n <= ASP_BLOCK8_APPLY_ROWS) return launched(asp::launch_block8_few(*a, nullptr, &x->dev, x->dev.n, y, ctx->sm_count, ctx->fault, ctx->stream));
    return launched(asp::launch_block8_product(*a, x->dev, y, ctx->sm_count, ctx->fault, ctx->stream));
}

asp_status asp_block8_gradient(asp_ctx *ctx, const asp_block8 *m, const asp_rows8 *x, const void *d_dy, int dtype, uint64_t ld, float *d_out, int accumulate)
{
    if (!ctx || !m || !x) return fail(ASP_ERR_INVALID_ARG, "NULL argument");
    if (x->dev.n_cols != m->side[0].n_cols) return fail(ASP_ERR_INVALID_ARG, "the rows have another length than those of the matrix");
    if (dtype != ASP_F16 && dtype != ASP_BF16) return fail(ASP_ERR_UNSUPPORTED, "dy: f16 or bf16");
    if (x->dev.n > 0 && dtype != x->from) return fail(ASP_ERR_UNSUPPORTED, "dy is of another type than what x was converted from");
    asp::Dense dy;
    ASP_TRY(look_at(d_dy, dtype, x->dev.n, m->side[0].n_rows, ld, "dy", &dy));
    if ((!d_out && m->pattern.blocks()) || (uintptr_t)d_out % 16) return fail(ASP_ERR_INVALID_ARG, "out is NULL or not on a 16-byte boundary");
    ASP_TRY(same_device(ctx, m->room));
    ASP_TRY(same_device(ctx, x->room));
    ASP_ON_DEVICE(ctx);
    return launched(asp::launch_block8_gradient(m->side[0], m->groups, x->dev, dy, d_out, accumulate != 0, ctx->sm_count, ctx->fault, ctx->stream));
}

} // extern "C"
