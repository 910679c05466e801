"""GPU: block-sparse matrices and rows in 8 bits (include/asp_b200_block8.h) against their definition in 64 bits.

Conversions are exact: every element has one right answer. Sums: the factors are exact, their products have 8 significant bits, and every
addition in 32 bits is off by at most 2^-23 of the sizes that have been added (2^-24 rounded, 2^-23 cut off, as tensor cores may), so
a sum of K products is within K * 2^-23 * sum |a| |x| of the exact one; the result is then rounded once more, by half a step of
its type.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import block8_ref as ref
from alphasparse_b200 import capi
from alphasparse_b200.block8 import Block8, Rows8

pytestmark = pytest.mark.gpu

TYPES = ref.TYPES


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(seed, n, c, dtype, pad=0, offset=0):
    """n rows of c columns, `pad` elements apart, the first one `offset` elements off a boundary. Sizes over many powers of two, some zeros."""
    g = gen(seed)
    x = torch.randn(n, c + pad, generator=g, device="cuda") * torch.exp2(torch.randint(-9, 5, (n, c + pad), generator=g, device="cuda").float())
    x[torch.rand(n, c + pad, generator=g, device="cuda") < 0.05] = 0.0
    room = torch.zeros(n * (c + pad) + offset, dtype=TYPES[dtype], device="cuda")
    room[offset:] = x.to(TYPES[dtype]).reshape(-1)
    return room[offset:].reshape(n, c + pad)[:, :c]


def pattern(seed, n_rows, n_cols, density, empty_row=None):
    rng = np.random.default_rng(seed)
    kept = rng.random((ref.blocks(n_rows), ref.blocks(n_cols))) < density
    if empty_row is not None:
        kept[empty_row] = False
    return np.concatenate([[0], np.cumsum(kept.sum(1))]).astype(np.int64), np.nonzero(kept)[1].astype(np.uint32)


def matrix(ctx, seed, n_rows, n_cols, density, transposed=True, empty_row=None):
    """(Block8, what it stands for in 64 bits)"""
    p = pattern(seed, n_rows, n_cols, density, empty_row)
    n = len(p[1])
    g = gen(seed)
    values = torch.randn(n, 128, 128, generator=g, device="cuda") * torch.exp2(torch.randint(-6, 3, (n, 1, 1), generator=g, device="cuda").float())
    values = ref.stored(p, ref.dense(p, (n_rows, n_cols), values))
    m = Block8(ctx, n_rows, n_cols, *p, transposed=transposed)
    assert m.n_blocks == n
    torch.cuda.synchronize()
    m.set_values(values.data_ptr(), "f32")
    ctx.synchronize()
    return m, ref.dense(p, (n_rows, n_cols), ref.groups_in_8_bits(values.reshape(n, -1)).reshape(n, 128, 128)) if n else torch.zeros(n_rows, n_cols, dtype=torch.float64, device="cuda")


def assert_sums(got, x, a, dtype, what):
    """got ~ x a^T"""
    want, size = x @ a.T, x.abs() @ a.T.abs()
    t = TYPES[dtype]
    room = size * (x.shape[1] * 2.0**-23) + want.abs() * (torch.finfo(t).eps / 2) + torch.finfo(t).tiny
    over = ((got.double() - want).abs() / room).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: {over} of what its roundings allow"


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


# ---- rows ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c,pad,offset", [(1, 1, 0, 0), (1, 128, 0, 0), (3, 127, 1, 0), (33, 129, 0, 1), (65, 512, 8, 0), (31, 640, 3, 1), (257, 1000, 24, 8), (100, 1801, 0, 0)])
def test_rows_to_8_bits_and_back(asp_ctx, dtype, n, c, pad, offset):
    x = rows(n + c, n, c, dtype, pad, offset)
    held = Rows8(asp_ctx, n + 2, c)
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, dtype, x.stride(0) if n > 1 else 0)
    assert len(held) == n
    want = ref.rows_in_8_bits(x)
    for out_dtype in ("f32", dtype):
        out = torch.full((n, c + 5), 7.0, dtype=TYPES[out_dtype], device="cuda")
        torch.cuda.synchronize()
        held.restore(out.data_ptr(), out_dtype, c + 5)
        asp_ctx.synchronize()
        assert torch.equal(out[:, :c].double(), want) and (out[:, c:] == 7.0).all()
    held.close()


def test_every_bf16_and_every_rounding(asp_ctx):
    """All finite bf16 numbers, a row for each exponent of its largest; all e4m3 and the points between them."""
    bits = torch.arange(0x8000, dtype=torch.int32)
    every = torch.cat([bits, bits | 0x8000]).to(torch.int16).view(torch.bfloat16)
    every = every[torch.isfinite(every)].reshape(-1, 64)
    x = torch.cat([every, every.flip(0)], 1).cuda()  # (large and small ones in a block)
    lattice = torch.arange(0, 449 * 512, dtype=torch.float32).reshape(-1, 128)[: 3584 // 2] / 512.0  # steps of 2^-9, and halves of larger steps
    lattice[:, 0] = 448.0
    for v, dtype in ((x, "bf16"), (lattice.cuda(), "f32"), (-3.0 * lattice.cuda(), "f32"), (lattice.cuda() * 2.0**-130, "f32")):
        held = Rows8(asp_ctx, v.shape[0], 128)
        out = torch.empty(v.shape, device="cuda")
        torch.cuda.synchronize()
        held.quantize(v.data_ptr(), v.shape[0], dtype)
        held.restore(out.data_ptr(), "f32")
        asp_ctx.synchronize()
        # (below 2^-126 the restored f32 is subnormal and may itself be rounded, once)
        assert torch.equal(out, ref.rows_in_8_bits(v).float())
        # What it stands for stands for itself, unless it is 2^128, which the numbers from 31/16 * 2^127 on round to (steps of 16 above 128:
        # 248 * 2^120 is a tie and goes to the even 256 * 2^120) and no 32-bit number is: restored as infinite, it is NaN the next time.
        again = torch.empty_like(out)
        held.quantize(out.data_ptr(), v.shape[0], "f32")
        held.restore(again.data_ptr(), "f32")
        asp_ctx.synchronize()
        assert torch.equal(again[out.isfinite()], out[out.isfinite()]) and again[out.isinf()].isnan().all()
        held.close()


def test_every_f16_with_neighbours_of_all_sizes(asp_ctx):
    """All 65536 of them, NaN and infinite ones included: side by side, shuffled, and each among tiny ones (whose scales fp16 itself does not have)."""
    every = torch.arange(0x10000, dtype=torch.int32).to(torch.int16).view(torch.float16)
    shuffled = every[torch.randperm(0x10000, generator=torch.Generator().manual_seed(1))]
    tiny = torch.arange(0x10000, dtype=torch.int32).remainder(16).to(torch.int16).view(torch.float16).reshape(-1, 128).repeat(8, 1)
    tiny[:, 5] = torch.arange(tiny.shape[0], dtype=torch.int32).remainder(0x400).to(torch.int16).view(torch.float16)  # every subnormal one
    for v in (every.reshape(-1, 128), shuffled.reshape(-1, 128), tiny, torch.zeros(3, 128, dtype=torch.float16)):
        v = v.contiguous().cuda()
        held, out = Rows8(asp_ctx, v.shape[0], 128), torch.empty(v.shape, device="cuda")
        torch.cuda.synchronize()
        held.quantize(v.data_ptr(), v.shape[0], "f16")
        held.restore(out.data_ptr(), "f32")
        asp_ctx.synchronize()
        assert same(out, ref.rows_in_8_bits(v))
        held.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_that_are_not_finite(asp_ctx, dtype):
    x = rows(5, 6, 300, dtype)
    x[0, 3], x[1, 200], x[2, 299], x[3, :128] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[4] = 0.0
    held = Rows8(asp_ctx, 6, 300)
    out = torch.empty(6, 300, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 6, dtype)
    held.restore(out.data_ptr(), "f32")
    asp_ctx.synchronize()
    assert same(out, ref.rows_in_8_bits(x)) and (out[4] == 0).all()


def test_fewer_rows_than_before_leave_the_others(asp_ctx):
    x, held = rows(1, 40, 256, "f32"), Rows8(asp_ctx, 40, 256)
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 40, "f32")
    other = 2.0 * x[:7].contiguous() + 1.0
    torch.cuda.synchronize()
    held.quantize(other.data_ptr(), 7, "f32")
    out = torch.full((40, 256), 7.0, device="cuda")
    torch.cuda.synchronize()
    held.restore(out.data_ptr(), "f32")
    asp_ctx.synchronize()
    assert len(held) == 7 and torch.equal(out[:7].double(), ref.rows_in_8_bits(other)) and (out[7:] == 7.0).all()
    held.quantize(0, 0, "f32")  # none
    held.restore(0, "f32")
    assert len(held) == 0


# ---- the matrix --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (300, 1000), (1000, 257)])
def test_values(asp_ctx, dtype, shape):
    p = pattern(3, *shape, 0.7)
    n = len(p[1])
    g = gen(4)
    values = (torch.randn(n, 128, 128, generator=g, device="cuda") * torch.exp2(torch.randint(-12, 9, (n, 1, 1), generator=g, device="cuda").float())).to(TYPES[dtype])
    m = Block8(asp_ctx, *shape, *p)
    out = torch.full((n, 128, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    m.get_values(out.data_ptr())
    asp_ctx.synchronize()
    assert (out == 0).all()
    m.set_values(values.data_ptr(), dtype)  # what sticks out of the matrix is not zero here, and taken as zero
    m.get_values(out.data_ptr())
    asp_ctx.synchronize()
    inside = ref.stored(p, ref.dense(p, shape, values))
    assert torch.equal(out.double(), ref.groups_in_8_bits(inside.reshape(n, -1)).reshape(out.shape))
    got = m.pattern()
    assert (got[0] == p[0]).all() and (got[1] == p[1]).all()
    m.close()


def test_values_that_are_not_finite(asp_ctx):
    values = torch.randn(2, 128, 128, generator=gen(1), device="cuda")
    values[0, 5, 6], values[1, 127, 0] = float("inf"), float("nan")
    m = Block8(asp_ctx, 128, 256, [0, 2], [0, 1], transposed=True)
    out = torch.empty_like(values)
    torch.cuda.synchronize()
    m.set_values(values.data_ptr(), "f32")
    m.get_values(out.data_ptr())
    asp_ctx.synchronize()
    assert same(out, ref.groups_in_8_bits(values.reshape(2, -1)).reshape(out.shape)) and out.isnan().sum() == 2
    # a row that meets them has a NaN, the others do not
    for transposed in (False, True):
        a = ref.dense(m.pattern(), (128, 256), out.double())
        a = a.T if transposed else a
        x, y = torch.ones(40, a.shape[1], device="cuda"), torch.empty(40, a.shape[0], device="cuda")
        held = Rows8(asp_ctx, 40, a.shape[1])
        torch.cuda.synchronize()
        held.quantize(x.data_ptr(), 40, "f32")
        m.product(held, y.data_ptr(), "f32", transposed=transposed)
        asp_ctx.synchronize()
        assert torch.equal(y.isnan(), (x.double() @ a.T).isnan())
        m.apply(x.data_ptr(), 3, "f32", y.data_ptr(), "f32", transposed=transposed)
        asp_ctx.synchronize()
        assert torch.equal(y[:3].isnan(), (x[:3].double() @ a.T).isnan())


def test_from_a_matrix_of_the_operator_graph(asp_ctx):
    from alphasparse_b200 import matrices
    from alphasparse_b200.graph import Matrix

    for dtype in (np.float32, np.float64):
        m, _ = matrices.from_row_lengths(np.random.default_rng(2).integers(0, 9, size=1000), 700, seed=2, dtype=dtype)
        hm = Matrix.from_csr(m)
        b = Block8.from_matrix(asp_ctx, hm, transposed=True)
        full = torch.zeros(1000, 700, dtype=torch.float64)
        r = np.repeat(np.arange(1000), np.diff(m.indptr))
        full[torch.from_numpy(r), torch.from_numpy(m.indices.astype(np.int64))] = torch.from_numpy(m.values.astype(np.float32)).double()
        full = full.cuda()
        p = b.pattern()
        want = ref.groups_in_8_bits(ref.stored(p, full).reshape(b.n_blocks, -1)).reshape(-1, 128, 128)
        out = torch.empty(b.n_blocks, 128, 128, device="cuda")
        torch.cuda.synchronize()
        b.get_values(out.data_ptr())
        asp_ctx.synchronize()
        assert torch.equal(out.double(), want) and ((ref.dense(p, (1000, 700), want) != 0) <= (full != 0)).all()
        x, y = rows(1, 5, 700, "f32"), torch.empty(5, 1000, device="cuda")
        torch.cuda.synchronize()
        b.apply(x.data_ptr(), 5, "f32", y.data_ptr(), "f32")
        asp_ctx.synchronize()
        assert_sums(y, ref.rows_in_8_bits(x), ref.dense(p, (1000, 700), want), "f32", "from_matrix")
        with pytest.raises(capi.AspError) as e:
            Block8.from_matrix(asp_ctx, hm.dense("dense compress"))
        assert e.value.status == 2


# ---- products --------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1.0), (128, 128, 1.0), (130, 1000, 0.5), (1000, 130, 0.5), (900, 2100, 0.3), (257, 4097, 1.0)]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n_rows,n_cols,density", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 8, 9, 17, 32])
def test_apply(asp_ctx, n, n_rows, n_cols, density, transposed):
    m, a = matrix(asp_ctx, n_rows, n_rows, n_cols, density, empty_row=2 if n_rows > 300 else None)
    a = a.T if transposed else a
    dtype = ["f32", "f16", "bf16"][(n + n_rows) % 3]
    x = rows(n, n, a.shape[1], dtype)
    for y_dtype in ("f32", dtype):
        y = torch.full((n + 1, a.shape[0]), 7.0, dtype=TYPES[y_dtype], device="cuda")
        torch.cuda.synchronize()
        m.apply(x.data_ptr(), n, dtype, y.data_ptr(), y_dtype, transposed=transposed)
        asp_ctx.synchronize()
        assert_sums(y[:n], ref.rows_in_8_bits(x), a, y_dtype, f"apply {n} {dtype} {y_dtype}")
        assert (y[n] == 7.0).all()
    m.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_rows,n_cols,density", [(1000, 130, 0.5), (900, 2100, 0.3), (4001, 600, 0.9)])
@pytest.mark.parametrize("n", [7, 16, 18, 23, 24, 25])
def test_apply_to_short_block_rows(asp_ctx, n, n_rows, n_cols, density, dtype):
    m, a = matrix(asp_ctx, n_rows + n, n_rows, n_cols, density, transposed=False, empty_row=1)
    x, held = rows(n, n, n_cols, dtype, 1), Rows8(asp_ctx, n, n_cols)
    y, other = (torch.full((n + 1, n_rows), 7.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    m.apply(x.data_ptr(), n, dtype, y.data_ptr(), "f32", n_cols + 1)
    held.quantize(x.data_ptr(), n, dtype, n_cols + 1)
    m.product(held, other.data_ptr(), "f32")
    asp_ctx.synchronize()
    assert_sums(y[:n], ref.rows_in_8_bits(x), a, "f32", f"apply {n} {dtype}")
    assert (y[n] == 7.0).all() and torch.equal(y, other)
    m.close()
    held.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_rows,n_cols,density,pad,offset", [(300, 9000, 0.9, 0, 0), (2500, 3500, 0.8, 1, 0), (5000, 2600, 1.0, 0, 3), (130, 8195, 0.6, 5, 0)])
@pytest.mark.parametrize("n", [1, 4, 8, 9, 16, 17, 20, 31, 32])
def test_apply_to_long_block_rows(asp_ctx, n, n_rows, n_cols, density, pad, offset, dtype):
    m, a = matrix(asp_ctx, n_rows + n, n_rows, n_cols, density, transposed=False, empty_row=1)
    x = rows(n, n, n_cols, dtype, pad, offset)
    ld = n_cols + pad
    got = []
    for y_dtype, y_pad in (("f32", 0), (dtype, 3), ("f32", 0)):
        y = torch.full((n + 1, n_rows + y_pad), 7.0, dtype=TYPES[y_dtype], device="cuda")
        torch.cuda.synchronize()
        m.apply(x.data_ptr(), n, dtype, y.data_ptr(), y_dtype, ld, n_rows + y_pad)
        asp_ctx.synchronize()
        assert_sums(y[:n, :n_rows], ref.rows_in_8_bits(x), a, y_dtype, f"apply {n} {dtype} {y_dtype}")
        assert (y[n] == 7.0).all() and (y[:, n_rows:] == 7.0).all()
        got.append(y)
    assert torch.equal(got[0], got[2])
    # rows that are in 8 bits already go through the same kernels
    held = Rows8(asp_ctx, n, n_cols)
    held.quantize(x.data_ptr(), n, dtype, ld)
    got[2].fill_(7.0)
    torch.cuda.synchronize()
    m.product(held, got[2].data_ptr(), "f32")
    asp_ctx.synchronize()
    assert torch.equal(got[0], got[2])
    m.close()
    held.close()


@pytest.mark.parametrize("n", [2, 12, 30])
def test_long_block_rows_and_rows_that_are_not_finite(asp_ctx, n):
    m, a = matrix(asp_ctx, 4, 260, 6000, 1.0)
    x = rows(2, n, 6000, "bf16")
    x[1, 5], x[n - 1, 5999] = float("nan"), float("inf")
    y = torch.full((n, 260), 7.0, device="cuda")
    torch.cuda.synchronize()
    m.apply(x.data_ptr(), n, "bf16", y.data_ptr(), "f32")
    asp_ctx.synchronize()
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[1] = bad[n - 1] = True
    assert torch.equal(y.isnan().all(1), bad) and torch.equal(y.isnan().any(1), bad)
    assert_sums(y[~bad], ref.rows_in_8_bits(x)[~bad], a, "f32", "the other rows")
    m.close()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n_rows,n_cols,density", SHAPES)
@pytest.mark.parametrize("n", [1, 31, 33, 100, 224, 225, 449, 1000])
def test_product(asp_ctx, n, n_rows, n_cols, density, transposed):
    m, a = matrix(asp_ctx, n_rows, n_rows, n_cols, density, empty_row=2 if n_rows > 300 else None)
    a = a.T if transposed else a
    dtype = ["f32", "f16", "bf16"][(n + n_rows) % 3]
    x, held = rows(n, n, a.shape[1], dtype), Rows8(asp_ctx, n + 7, a.shape[1])
    more = rows(n + 1, n + 7, a.shape[1], dtype)  # what lies behind the rows held must not count
    more[n:] = float("nan")
    torch.cuda.synchronize()
    held.quantize(more.data_ptr(), n + 7, dtype)
    held.quantize(x.data_ptr(), n, dtype)
    for y_dtype in ("f32", dtype):
        y = torch.full((n + 3, a.shape[0]), 7.0, dtype=TYPES[y_dtype], device="cuda")
        torch.cuda.synchronize()
        m.product(held, y.data_ptr(), y_dtype, transposed=transposed)
        asp_ctx.synchronize()
        assert_sums(y[:n], ref.rows_in_8_bits(x), a, y_dtype, f"product {n} {dtype} {y_dtype}")
        assert (y[n:] == 7.0).all()
    m.close()
    held.close()


@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("x_pad,x_off,y_pad,y_off", [(0, 0, 1, 0), (8, 0, 8, 0), (3, 1, 5, 1), (1, 0, 2, 2)])
def test_strides_and_offsets(asp_ctx, n, x_pad, x_off, y_pad, y_off):
    m, a = matrix(asp_ctx, 4, 400, 500, 0.6)
    for dtype in ("f16", "f32"):
        x = rows(7, n, 500, dtype, x_pad, x_off)
        room = torch.full((n * (400 + y_pad) + y_off,), 7.0, dtype=TYPES[dtype], device="cuda")
        y = room[y_off:].reshape(n, 400 + y_pad)
        held = Rows8(asp_ctx, n, 500)
        torch.cuda.synchronize()
        if n <= 32:
            m.apply(x.data_ptr(), n, dtype, y.data_ptr(), dtype, ldx=x.stride(0), ldy=y.stride(0))
        else:
            held.quantize(x.data_ptr(), n, dtype, x.stride(0))
            m.product(held, y.data_ptr(), dtype, y.stride(0))
        asp_ctx.synchronize()
        assert_sums(y[:, :400], ref.rows_in_8_bits(x), a, dtype, "strides")
        assert (y[:, 400:] == 7.0).all() and (room[:y_off] == 7.0).all()


@pytest.mark.parametrize("n", [3, 90])
def test_a_matrix_without_blocks_and_products_without_rows(asp_ctx, n):
    m = Block8(asp_ctx, 300, 200, [0, 0, 0, 0], [], transposed=True)
    x, y, held = rows(1, n, 200, "f32"), torch.full((n, 300), 7.0, device="cuda"), Rows8(asp_ctx, n, 200)
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, "f32")
    m.product(held, y.data_ptr(), "f32")
    asp_ctx.synchronize()
    assert (y == 0).all()
    m.set_values(0, "f32")
    m.get_values(0)
    if n <= 32:
        y.fill_(7.0)
        torch.cuda.synchronize()
        m.apply(x.data_ptr(), n, "f32", y.data_ptr(), "f32")
        asp_ctx.synchronize()
        assert (y == 0).all()
    y.fill_(7.0)
    torch.cuda.synchronize()
    held.quantize(0, 0, "f32")
    m.product(held, y.data_ptr(), "f32")
    m.apply(0, 0, "f32", 0, "f32")
    asp_ctx.synchronize()
    assert (y == 7.0).all()


@pytest.mark.parametrize("n,n_rows,n_cols", [(64, 1024, 8192), (40, 4096, 2048), (700, 512, 512), (500, 2048, 1024), (2500, 1500, 1000)])
def test_product_in_tiles_of_all_sizes(asp_ctx, n, n_rows, n_cols):
    m, a = matrix(asp_ctx, 77, n_rows, n_cols, 0.8, transposed=False, empty_row=1)
    x, held, y = rows(n, n, n_cols, "bf16"), Rows8(asp_ctx, n, n_cols), torch.empty(n, n_rows, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, "bf16")
    m.product(held, y.data_ptr(), "f32")
    asp_ctx.synchronize()
    assert_sums(y, ref.rows_in_8_bits(x), a, "f32", "tiles")
    m.close()
    held.close()


@pytest.mark.parametrize("n,n_rows", [(40, 100), (300, 2000), (20, 200), (20, 5000)])
def test_long_sums_in_32_bits_are_rounded(asp_ctx, n, n_rows):
    """128 blocks, products of one sign. A tensor core cuts off less than 2^-23 of the sum each time it adds (32 columns): over 16 blocks, 64 times, to a sum that
    grows evenly, less than 32.5 * 2^-23 in all, and eight such sums are added up with half a step each, 4 * 2^-23. (All 512 additions in one sum, of which half
    a step is cut off on average, would come to 128 * 2^-23.)"""
    m = Block8(asp_ctx, n_rows, 16384, *pattern(1, n_rows, 16384, 1.0))
    values = torch.rand(m.n_blocks, 128, 128, generator=gen(1), device="cuda") + 0.5
    x, held = torch.rand(n, 16384, generator=gen(2), device="cuda") + 0.5, Rows8(asp_ctx, n, 16384)
    y = torch.empty(n, n_rows, device="cuda")
    torch.cuda.synchronize()
    m.set_values(values.data_ptr(), "f32")
    held.quantize(x.data_ptr(), n, "f32")
    m.product(held, y.data_ptr(), "f32")
    asp_ctx.synchronize()
    a = ref.dense(m.pattern(), (n_rows, 16384), ref.groups_in_8_bits(values.reshape(m.n_blocks, -1)).reshape(-1, 128, 128))
    want = ref.rows_in_8_bits(x) @ a.T
    assert ((y.double() - want).abs() / want).max().item() < (32.5 + 4) * 2.0**-23
    m.close()
    held.close()


@pytest.mark.parametrize("n", [7, 20, 100, 400])
def test_rows_that_are_not_finite_keep_it_to_themselves(asp_ctx, n):
    m, a = matrix(asp_ctx, 78, 700, 900, 1.0)
    x = rows(2, n, 900, "f32")
    x[1, 5], x[n // 2, 899] = float("nan"), float("inf")
    held, y = Rows8(asp_ctx, n, 900), torch.empty(n, 700, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, "f32")
    for call in (lambda: m.product(held, y.data_ptr(), "f32"), lambda: m.apply(x.data_ptr(), min(n, 32), "f32", y.data_ptr(), "f32")):
        y.fill_(7.0)
        torch.cuda.synchronize()
        call()
        asp_ctx.synchronize()
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[1] = bad[n // 2] = True
        seen = n if (y[-1] != 7.0).any() else min(n, 32)
        assert torch.equal(y[:seen].isnan().all(1), bad[:seen]) and torch.equal(y[:seen].isnan().any(1), bad[:seen])
        good = ~bad[:seen]
        assert_sums(y[:seen][good], ref.rows_in_8_bits(x)[:seen][good], a, "f32", "the other rows")


@pytest.mark.parametrize("n", [4, 200])
def test_scales_far_apart(asp_ctx, n):
    """Exponents whose sum no 32-bit number has, though the sums of products are ordinary; and rows of the largest numbers."""
    m = Block8(asp_ctx, 128, 256, [0, 2], [0, 1])
    values = torch.randn(2, 128, 128, generator=gen(2), device="cuda")
    values[0] *= 2.0**-100
    values[1] *= 2.0**90
    x = torch.randn(n, 256, generator=gen(3), device="cuda")
    x[:, :128] *= 2.0**100
    x[:, 128:] *= 2.0**-95
    x[1] = 0.0
    y, held = torch.empty(n, 128, device="cuda"), Rows8(asp_ctx, n, 256)
    torch.cuda.synchronize()
    m.set_values(values.data_ptr(), "f32")
    if n <= 32:
        m.apply(x.data_ptr(), n, "f32", y.data_ptr(), "f32")
    else:
        held.quantize(x.data_ptr(), n, "f32")
        m.product(held, y.data_ptr(), "f32")
    asp_ctx.synchronize()
    a = ref.dense(m.pattern(), (128, 256), ref.groups_in_8_bits(values.reshape(2, -1)).reshape(2, 128, 128))
    assert_sums(y, ref.rows_in_8_bits(x), a, "f32", "far apart")


@pytest.mark.parametrize("n,n_cols", [(4, 256), (4, 6016), (20, 6016), (200, 256)])
@pytest.mark.parametrize("k", [70, -70])
def test_scales_whose_product_no_32_bit_number_is(asp_ctx, n, n_cols, k):
    """Two exponents that add up to 140 or -140, and products that 32 bits have: of elements far below (above) the largest of their blocks."""
    blocks = n_cols // 128
    m = Block8(asp_ctx, 128, n_cols, [0, blocks], list(range(blocks)))
    values, x = torch.zeros(blocks, 128, 128, device="cuda"), torch.zeros(n, n_cols, device="cuda")
    values[0, 0, 0] = x[:, 0] = 2.0 ** (k + 8)  # what makes the scale 2^k; their product, 2^(2 k + 16), is row 0
    values[0, 1:, 1] = x[:, 1] = 2.0 ** (k - 6)
    y, held = torch.empty(n, 128, device="cuda"), Rows8(asp_ctx, n, n_cols)
    torch.cuda.synchronize()
    m.set_values(values.data_ptr(), "f32")
    if n <= 32:
        m.apply(x.data_ptr(), n, "f32", y.data_ptr(), "f32")
    else:
        held.quantize(x.data_ptr(), n, "f32")
        m.product(held, y.data_ptr(), "f32")
    asp_ctx.synchronize()
    want = torch.full((n, 128), 4.0 ** (k - 6), dtype=torch.float64, device="cuda")
    want[:, 0] = 4.0 ** (k + 8)
    assert torch.equal(y, want.float())
    m.close()
    held.close()


# ---- gradients -------------------------------------------------------------------------------------------------------
def assert_gradient(got, dy, x, p, before=0.0):
    want, size = ref.stored(p, dy.double().T @ x), ref.stored(p, dy.double().abs().T @ x.abs())
    room = size * ((dy.shape[0] + 1) * 2.0**-23) + (want + before).abs() * 2.0**-24 + 2.0**-126
    over = ((got.double() - before - want).abs() / room).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"gradient: {over} of what its roundings allow"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_rows,n_cols,density", [(1, 1, 1.0), (128, 128, 1.0), (130, 1000, 0.5), (900, 2100, 0.3), (1000, 384, 0.8)])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 200, 1000])
def test_gradient(asp_ctx, n, n_rows, n_cols, density, dtype):
    p = pattern(n_rows, n_rows, n_cols, density)
    m = Block8(asp_ctx, n_rows, n_cols, *p)
    x, dy = rows(n, n, n_cols, dtype), rows(n + 1, n, n_rows, dtype)
    held = Rows8(asp_ctx, n + 5, n_cols)
    more = torch.full((n + 5, n_cols), float("nan"), dtype=TYPES[dtype], device="cuda")
    out = torch.full((m.n_blocks, 128, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    held.quantize(more.data_ptr(), n + 5, dtype)
    held.quantize(x.data_ptr(), n, dtype)
    m.gradient(held, dy.data_ptr(), dtype, out.data_ptr())
    asp_ctx.synchronize()
    want = ref.rows_in_8_bits(x)
    assert_gradient(out, dy, want, p)
    assert torch.equal(out, ref.stored(p, ref.dense(p, (n_rows, n_cols), out)))  # zero outside the matrix
    # added to what is there
    m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), accumulate=True)
    asp_ctx.synchronize()
    once = ref.stored(p, dy.double().T @ want)
    size = ref.stored(p, dy.double().abs().T @ want.abs())
    assert ((out.double() - 2 * once).abs() <= size * (2 * (n + 1) * 2.0**-23) + once.abs() * 2.0**-22 + 2.0**-126).all()
    m.close()
    held.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n", [(1, 3, 1000), (1, 60, 400), (2, 100, 150), (3, 100, 70), (4, 100, 150), (5, 100, 130), (7, 40, 300), (2, 80, 5000), (1, 150, 4500), (2, 2, 9000)])
def test_gradient_of_columns_of_blocks(asp_ctx, blocks, columns, n, dtype):
    """Columns of 1 to 7 blocks, which are taken one by one or in twos, by one CTA or a cluster that shares the rows, in sums of 2048 rows."""
    n_rows, n_cols = 128 * blocks - 3, 128 * columns - 5
    p = pattern(1, n_rows, n_cols, 1.0)
    m, held = Block8(asp_ctx, n_rows, n_cols, *p), Rows8(asp_ctx, n, n_cols)
    g = gen(n)
    x, dy = torch.randn(n, n_cols, generator=g, device="cuda").to(TYPES[dtype]), torch.randn(n, (n_rows + 7) // 8 * 8, generator=g, device="cuda").to(TYPES[dtype])
    out = torch.full((m.n_blocks, 128, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, dtype)
    m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), dy.stride(0))
    asp_ctx.synchronize()
    assert_gradient(out, dy[:, :n_rows], ref.rows_in_8_bits(x), p)
    m.close()
    held.close()


def test_many_gradients_and_products_one_after_the_other(asp_ctx):
    """Copies that overtake one another, warps ahead of others: 300 calls on a busy chip give the bits of the first."""
    n = 4096
    m, _ = matrix(asp_ctx, 6, 2048, 2048, 0.4)
    x, dy = rows(1, n, 2048, "bf16"), rows(2, n, 2048, "bf16")
    held, grads = Rows8(asp_ctx, n, 2048), Rows8(asp_ctx, n, 2048)
    first = None
    for k in range(6):
        out = [torch.full((m.n_blocks, 128, 128), 7.0, device="cuda"), torch.full((n, 2048), 7.0, device="cuda"), torch.full((n, 2048), 7.0, device="cuda")]
        torch.cuda.synchronize()
        for _ in range(50):
            held.quantize(x.data_ptr(), n, "bf16")
            m.gradient(held, dy.data_ptr(), "bf16", out[0].data_ptr())
            m.product(held, out[1].data_ptr(), "f32")
            grads.quantize(dy.data_ptr(), n, "bf16")
            m.product(grads, out[2].data_ptr(), "f32", transposed=True)
        asp_ctx.synchronize()
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 0), (0, 1), (7, 8)])
def test_gradient_of_strided_rows(asp_ctx, pad, offset):
    p = pattern(9, 300, 500, 0.7)
    m, held = Block8(asp_ctx, 300, 500, *p), Rows8(asp_ctx, 150, 500)
    x, dy = rows(1, 150, 500, "bf16"), rows(2, 150, 300, "bf16", pad, offset)
    out = torch.empty(m.n_blocks, 128, 128, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 150, "bf16")
    m.gradient(held, dy.data_ptr(), "bf16", out.data_ptr(), dy.stride(0))
    asp_ctx.synchronize()
    assert_gradient(out, dy, ref.rows_in_8_bits(x), p)


def test_gradient_of_no_rows(asp_ctx):
    m, held = Block8(asp_ctx, 200, 200, [0, 1, 2], [0, 1]), Rows8(asp_ctx, 4, 200)
    out = torch.full((2, 128, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    held.quantize(0, 0, "bf16")
    m.gradient(held, 0, "bf16", out.data_ptr(), accumulate=True)
    asp_ctx.synchronize()
    assert (out == 7.0).all()
    m.gradient(held, 0, "bf16", out.data_ptr())
    asp_ctx.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_gradient_where_x_is_not_finite(asp_ctx, dtype):
    """An element that is not finite reaches its own column of the blocks, and no other."""
    p = (np.array([0, 2]), np.array([0, 1], dtype=np.uint32))
    m, held = Block8(asp_ctx, 128, 256, *p), Rows8(asp_ctx, 70, 256)
    x, dy = rows(1, 70, 256, dtype), rows(2, 70, 128, dtype)
    x[69, 200] = float("inf")
    out = torch.empty(2, 128, 128, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 70, dtype)
    m.gradient(held, dy.data_ptr(), dtype, out.data_ptr())
    asp_ctx.synchronize()
    bad = out.isnan()
    assert bad[1, :, 72].all() and bad.sum() == 128


def test_gradients_are_those_of_the_formula_and_of_differences(asp_ctx):
    """L = sum of w * (A x), linear in A and in x: differences of L over whole steps are its gradients, up to the roundings of L's own sums."""
    p = (np.array([0, 1, 2]), np.array([1, 0], dtype=np.uint32))
    g = gen(8)
    values = torch.randint(-8, 9, (2, 128, 128), generator=g, device="cuda").float()  # (whole numbers to 8: exact in 8 bits, and so are sums)
    x = torch.randint(-4, 5, (40, 256), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randint(-2, 3, (40, 256), generator=g, device="cuda").to(torch.bfloat16)
    m, held, grads = Block8(asp_ctx, 256, 256, *p, transposed=True), Rows8(asp_ctx, 40, 256), Rows8(asp_ctx, 40, 256)

    def loss(values, x):
        y = torch.empty(40, 256, device="cuda")
        torch.cuda.synchronize()
        m.set_values(values.data_ptr(), "f32")
        held.quantize(x.data_ptr(), 40, "bf16")
        m.product(held, y.data_ptr(), "f32")
        asp_ctx.synchronize()
        return (w.double() * y.double()).sum().item()

    at = loss(values, x)
    da, dx = torch.empty(2, 128, 128, device="cuda"), torch.empty(40, 256, device="cuda")
    m.gradient(held, w.data_ptr(), "bf16", da.data_ptr())
    grads.quantize(w.data_ptr(), 40, "bf16")
    m.product(grads, dx.data_ptr(), "f32", transposed=True)
    asp_ctx.synchronize()
    for b, r, c in ((0, 0, 0), (0, 127, 5), (1, 64, 127), (1, 3, 3)):
        step = values.clone()
        step[b, r, c] += 1.0 if step[b, r, c] < 8 else -1.0
        d = (step - values)[b, r, c].item()
        assert loss(step, x) - at == d * da[b, r, c].item()
    for t, c in ((0, 0), (39, 255), (17, 130)):
        step = x.clone()
        step[t, c] += 1.0
        assert loss(values, step) - at == dx[t, c].item()


# ---- together ----------------------------------------------------------------------------------------------------------
def test_steps_of_training_and_serving(asp_ctx):
    """Forward and backward passes of two layers, new values, another step, then one row at a time: as a program would use it."""
    shapes = [(500, 300), (200, 500)]
    layers = [matrix(asp_ctx, 20 + i, *s, 0.6) for i, s in enumerate(shapes)]
    n = 77
    for step in range(2):
        x = rows(step, n, 300, "bf16")
        kept, act = [], x
        for m, a in layers:
            held = Rows8(asp_ctx, n, a.shape[1])
            y = torch.empty(n, a.shape[0], dtype=torch.bfloat16, device="cuda")
            torch.cuda.synchronize()
            held.quantize(act.data_ptr(), n, "bf16")
            m.product(held, y.data_ptr(), "bf16")
            asp_ctx.synchronize()
            assert_sums(y, ref.rows_in_8_bits(act), a, "bf16", "forward")
            kept.append((held, act))
            act = y
        d = rows(50 + step, n, 200, "bf16")
        for i in (1, 0):
            (m, a), (held, act) = layers[i], kept[i]
            p = m.pattern()
            da = torch.empty(m.n_blocks, 128, 128, device="cuda")
            dx = torch.empty(n, a.shape[1], dtype=torch.bfloat16, device="cuda")
            grads = Rows8(asp_ctx, n, a.shape[0])
            torch.cuda.synchronize()
            m.gradient(held, d.data_ptr(), "bf16", da.data_ptr())
            grads.quantize(d.data_ptr(), n, "bf16")
            m.product(grads, dx.data_ptr(), "bf16", transposed=True)
            asp_ctx.synchronize()
            assert_gradient(da, d, ref.rows_in_8_bits(act), p)
            assert_sums(dx, ref.rows_in_8_bits(d), a.T, "bf16", "dx")
            values = torch.empty_like(da)
            torch.cuda.synchronize()
            m.get_values(values.data_ptr())
            asp_ctx.synchronize()
            values -= 0.01 * da / da.abs().max()
            torch.cuda.synchronize()
            m.set_values(values.data_ptr(), "f32")
            asp_ctx.synchronize()
            layers[i] = (m, ref.dense(p, a.shape, ref.groups_in_8_bits(values.reshape(len(values), -1)).reshape(values.shape)))
            d = dx
    x = rows(9, 1, 300, "bf16")
    for m, a in layers:
        y = torch.empty(1, a.shape[0], dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        m.apply(x.data_ptr(), 1, "bf16", y.data_ptr(), "bf16")
        asp_ctx.synchronize()
        assert_sums(y, ref.rows_in_8_bits(x), a, "bf16", "serving")
        x = y


def test_captured_and_replayed(asp_ctx):
    m, a = matrix(asp_ctx, 31, 500, 700, 0.5)
    n = 150
    x, dy = rows(1, n, 700, "bf16"), rows(2, n, 500, "bf16")
    y, da = torch.empty(n, 500, device="cuda"), torch.empty(m.n_blocks, 128, 128, device="cuda")
    y1 = torch.empty(3, 500, device="cuda")
    held = Rows8(asp_ctx, n, 700)

    def step():
        held.quantize(x.data_ptr(), n, "bf16")
        m.product(held, y.data_ptr(), "f32")
        m.gradient(held, dy.data_ptr(), "bf16", da.data_ptr())
        m.apply(x.data_ptr(), 3, "bf16", y1.data_ptr(), "f32")

    step()
    asp_ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(asp_ctx.stream)):
        step()
    for k in range(3):
        x.copy_(rows(10 + k, n, 700, "bf16"))
        dy.copy_(rows(20 + k, n, 500, "bf16"))
        y.fill_(7.0), da.fill_(7.0), y1.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.rows_in_8_bits(x)
        assert_sums(y, want, a, "f32", "replayed product")
        assert_sums(y1, want[:3], a, "f32", "replayed apply")
        assert_gradient(da, dy, want, m.pattern())


def test_same_bits_every_time_and_on_two_streams_at_once(asp_ctx):
    m, a = matrix(asp_ctx, 32, 1500, 1100, 0.4)
    other = capi.Context(0)
    n = 260
    x, dy = rows(1, n, 1100, "f16"), rows(2, n, 1500, "f16")
    got = []
    for _ in range(3):
        sets = []
        for ctx in (asp_ctx, other):
            held = Rows8(ctx, n, 1100)
            y, y1, da = torch.empty(n, 1500, device="cuda"), torch.empty(9, 1500, device="cuda"), torch.empty(m.n_blocks, 128, 128, device="cuda")
            sets.append((ctx, held, y, y1, da))
        torch.cuda.synchronize()
        for ctx, held, y, y1, da in sets:
            with_ctx = ctx.handle
            from alphasparse_b200.block8 import _lib

            held.quantize(x.data_ptr(), n, "f16")
            capi.check(_lib().asp_block8_product(with_ctx, m._h, 0, held._h, y.data_ptr(), capi.F32, 0))
            capi.check(_lib().asp_block8_gradient(with_ctx, m._h, held._h, dy.data_ptr(), 6, 0, da.data_ptr(), 0))
            capi.check(_lib().asp_block8_apply(with_ctx, m._h, 0, x.data_ptr(), 6, 9, 0, y1.data_ptr(), capi.F32, 0))
        asp_ctx.synchronize()
        other.synchronize()
        got += [s[2:] for s in sets]
    for g in got[1:]:
        assert all(torch.equal(u, v) for u, v in zip(g, got[0]))
    assert_sums(got[0][0], ref.rows_in_8_bits(x), a, "f32", "two streams")
    other.close()


def test_calls_of_all_kinds_in_any_order_on_two_streams(asp_ctx):
    """Kernels that share SMs, shared memory and tensor memory with others: the same bits as when each runs alone."""
    other, calls, kept = capi.Context(0), [], []
    for ctx in (asp_ctx, other):
        for n_rows, n_cols, density in ((260, 6000, 0.9), (4096, 2048, 1.0), (1000, 1000, 0.5)):
            m = Block8(ctx, n_rows, n_cols, *pattern(n_rows, n_rows, n_cols, density))
            values = torch.randn(m.n_blocks, 128, 128, generator=gen(n_rows), device="cuda")
            torch.cuda.synchronize()
            m.set_values(values.data_ptr(), "f32")
            ctx.synchronize()
            for n, dtype in ((1, "bf16"), (7, "f16"), (13, "bf16"), (20, "f32"), (32, "f16"), (300, "f32"), (500, "bf16")):
                x, y, held = rows(n, n, n_cols, dtype), torch.empty(n, n_rows, device="cuda"), Rows8(ctx, n, n_cols)
                torch.cuda.synchronize()
                held.quantize(x.data_ptr(), n, dtype)
                ctx.synchronize()
                kept.append((m, x, held))
                if n <= 32:
                    calls.append((lambda m=m, x=x, n=n, dtype=dtype, y=y: m.apply(x.data_ptr(), n, dtype, y.data_ptr(), "f32"), y))
                else:
                    calls.append((lambda m=m, held=held, y=y: m.product(held, y.data_ptr(), "f32"), y))
                if dtype == "bf16":
                    dy, da = rows(n + 1, n, n_rows, dtype), torch.empty(m.n_blocks, 128, 128, device="cuda")
                    kept.append(dy)
                    calls.append((lambda m=m, held=held, dy=dy, da=da: m.gradient(held, dy.data_ptr(), "bf16", da.data_ptr()), da))
    torch.cuda.synchronize()
    alone = []
    for call, out in calls:
        call()
        asp_ctx.synchronize()
        other.synchronize()
        alone.append(out.clone())
    rng = np.random.default_rng(1)
    for _ in range(5):
        for _, out in calls:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for i in np.concatenate([rng.permutation(len(calls)) for _ in range(3)]):
            calls[i][0]()
        asp_ctx.synchronize()
        other.synchronize()
        assert all(torch.equal(out, want) for (_, out), want in zip(calls, alone))
    other.close()


def test_more_than_2_to_the_31_bytes_of_rows(asp_ctx):
    """Rows behind byte 2^32 of X and of Y; values behind byte 2^32 of A would need 2^18 blocks and are held to 64-bit products in the code."""
    n, c = 600_000, 8192
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    held = Rows8(asp_ctx, n, c)
    x = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    tail = rows(3, 300, c, "bf16")
    x[-300:] = tail
    m, a = matrix(asp_ctx, 5, 256, c, 0.1, transposed=False)
    y = torch.full((n, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, "bf16")
    m.product(held, y.data_ptr(), "bf16")
    asp_ctx.synchronize()
    assert_sums(y[-300:], ref.rows_in_8_bits(tail), a, "bf16", "far rows") 
    assert (y[:-300] == 0).all()
    held.restore(x.data_ptr(), "bf16")
    asp_ctx.synchronize()
    assert torch.equal(x[-300:].double(), ref.rows_in_8_bits(tail))
    held.close()


def test_refusals(asp_ctx):
    """Wrong calls are errors of the call: nothing is launched, the context goes on."""
    m, _ = matrix(asp_ctx, 1, 300, 200, 1.0, transposed=False)
    held = Rows8(asp_ctx, 40, 200)
    x, y = rows(1, 40, 200, "bf16"), torch.full((40, 300), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 40, "bf16")
    asp_ctx.synchronize()

    def refused(status, call, *args, **kw):
        with pytest.raises(capi.AspError) as e:
            call(*args, **kw)
        assert e.value.status == status, e.value

    refused(1, held.quantize, x.data_ptr(), 41, "bf16")
    refused(1, held.quantize, x.data_ptr(), 40, "bf16", 199)
    refused(1, held.quantize, x.data_ptr() + 1, 3, "bf16")
    refused(1, held.quantize, 0, 3, "bf16")
    refused(1, held.restore, 0, "f32")
    refused(2, m.product, held, y.data_ptr(), "bf16", transposed=True)
    refused(1, m.product, Rows8(asp_ctx, 4, 201), y.data_ptr(), "bf16")
    refused(1, m.product, held, y.data_ptr(), "bf16", 299)
    refused(1, m.apply, x.data_ptr(), 33, "bf16", y.data_ptr(), "bf16")
    refused(2, m.apply, x.data_ptr(), 3, "bf16", y.data_ptr(), "bf16", transposed=True)
    refused(1, m.set_values, y.data_ptr() + 4, "f32")
    refused(1, m.get_values, 0)
    out = torch.empty(m.n_blocks, 128, 128, device="cuda")
    refused(2, m.gradient, held, y.data_ptr(), "f32", out.data_ptr())
    refused(2, m.gradient, held, y.data_ptr(), "f16", out.data_ptr())  # x was bf16
    refused(1, m.gradient, held, y.data_ptr(), "bf16", out.data_ptr() + 4)
    refused(1, m.gradient, held, 0, "bf16", out.data_ptr())
    L = capi.lib()
    assert L.asp_block8_product(asp_ctx.handle, m._h, 0, held._h, C.c_void_p(y.data_ptr()), capi.F64, C.c_uint64(0)) == 2
    asp_ctx.synchronize()
    assert (y == 7.0).all()
