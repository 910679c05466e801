"""GPU: block-sparse matrices in 8 bits (include/asp_b200_block8.h) at the ends of their types, and right after they are made. Tolerances as in test_gpu_block8.py."""
import numpy as np
import pytest
import torch

import block8_ref as ref
from alphasparse_b200 import capi
from alphasparse_b200.block8 import Block8, Rows8
from test_gpu_block8 import TYPES, assert_gradient, gen, pattern, rows

pytestmark = pytest.mark.gpu

# blocks of a block column, block columns, rows, elements between the rows of dy, by what takes them: a cluster that shares the rows, single blocks, twos, twos in
# several sums, single blocks in several sums, rows of dy that begin anywhere
WAYS = [(1, 3, 1000, 0), (1, 150, 200, 0), (2, 100, 150, 0), (2, 100, 2000, 0), (1, 150, 1500, 0), (2, 5, 300, 1), (3, 70, 150, 1), (3, 50, 70, 0)]


def gradient(ctx, blocks, columns, x, dy, dtype, before=None):
    """(the gradient by all blocks of a matrix of blocks x columns of them, added to `before` where it is given; the pattern)"""
    n, n_rows, n_cols = x.shape[0], dy.shape[1], x.shape[1]
    assert ref.blocks(n_rows) == blocks and ref.blocks(n_cols) == columns
    p = pattern(1, n_rows, n_cols, 1.0)
    m, held = Block8(ctx, n_rows, n_cols, *p), Rows8(ctx, n, n_cols)
    out = torch.full((m.n_blocks, 128, 128), 7.0, device="cuda") if before is None else before.clone()
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), n, dtype)
    m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), dy.stride(0) if n > 1 else 0, accumulate=before is not None)
    ctx.synchronize()
    m.close()
    held.close()
    return out, p


def factors(blocks, columns, n, pad, dtype):
    """x and dy of whole numbers of steps and not, dy with rows of zeros."""
    x, dy = rows(n, n, 128 * columns - 5, dtype), rows(n + 1, n, (128 * blocks - 8), dtype, 8 if pad == 0 else pad)
    dy[torch.rand(n, generator=gen(3), device="cuda") < 0.2] = 0.0
    return x, dy


def with_largest(x, dtype, share, seed=4):
    """x, where `share` of the rows' blocks have some of the largest numbers of the type, which 8 bits round up to what the type does not have"""
    g, (n, c) = gen(seed), x.shape
    large = torch.tensor([63424.0, 63488.0, 65504.0] if dtype == "f16" else [247.0 * 2.0**120, 248.0 * 2.0**120, 255.0 * 2.0**120], device="cuda")
    which = (torch.rand(n, ref.blocks(c), generator=g, device="cuda") < share).repeat_interleave(128, 1)[:, :c]
    some = which & (torch.rand(n, c, generator=g, device="cuda") < 0.1)
    v = large[torch.randint(0, 3, (n, c), generator=g, device="cuda")] * (torch.randint(0, 2, (n, c), generator=g, device="cuda") * 2 - 1)
    return torch.where(some, v.to(TYPES[dtype]), x)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
@pytest.mark.parametrize("share", [0.02, 1.0])
def test_gradient_of_the_largest_numbers(asp_ctx, blocks, columns, n, pad, share, dtype):
    """What 8 bits make of them, 2^16 and 2^128, is no number of the type. It still counts as what it is, and nothing where dy is zero."""
    x, dy = factors(blocks, columns, n, pad, dtype)
    x = with_largest(x, dtype, share)
    if dtype == "bf16":
        dy *= 2.0**-30  # (in place: its rows stay where they are)
    want = ref.rows_in_8_bits(x)
    assert (want.abs() > torch.finfo(TYPES[dtype]).max).any() and want.isfinite().all()
    out, p = gradient(asp_ctx, blocks, columns, x, dy, dtype)
    assert_gradient(out, dy, want, p)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
def test_gradient_where_dy_is_not_finite(asp_ctx, blocks, columns, n, pad, dtype):
    """Beside rows of the largest numbers and others: infinite and NaN as the formula has them, element by element."""
    x, dy = factors(blocks, columns, n, pad, dtype)
    x = torch.where(x == 0, torch.ones_like(x), with_largest(x, dtype, 0.02))
    x[min(n - 1, 65), 7] = 0.0
    dy *= 2.0**-30 if dtype == "bf16" else 1.0
    dy[0, 5], dy[n // 2, 9], dy[min(n - 1, 65), 11], dy[n - 1, 1] = float("inf"), -float("inf"), float("inf"), float("nan")
    out, p = gradient(asp_ctx, blocks, columns, x, dy, dtype)
    xq, dyd = ref.rows_in_8_bits(x), dy.double()
    want = ref.stored(p, dyd.T @ xq)
    assert want.isnan().any() and want.isinf().any()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf()) and torch.equal(out[want.isinf()].double(), want[want.isinf()])
    clean = torch.where(dyd.isfinite().all(0), dyd, 0.0)  # (columns of dy without any: rows of the blocks)
    finite = ref.stored(p, (dyd.isfinite().all(0).double()[:, None] * torch.ones(1, x.shape[1], dtype=torch.float64, device="cuda")))
    assert_gradient(torch.where(finite > 0, out, 0.0), clean, xq, p)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
def test_gradient_of_scales_of_all_sizes(asp_ctx, blocks, columns, n, pad, dtype):
    """Blocks of subnormal numbers, and of numbers far above what 8 bits hold without a scale.

    What is cut off goes by the exponents of the factors as they are stored, and a subnormal number has that of the smallest normal one, N: where x is j 2^-24 in fp16,
    dy x counts as one of size 2^-14 |dy|. (-16.1875 * 2^-24 in fp16, 2^-20 in size, has the exponent 4 - 14 = -10 and made a sum be 2^-34.8 off, a step of 2^-24 below
    that exponent; 71 rows of 2^-23 of its own size were 2^-36.) So a sum is within (n + 1) * 2^-23 * sum max(|dy|, N) max(|x|, N), factors of zero left out."""
    x, dy = factors(blocks, columns, n, pad, dtype)
    low, high = (-24, 15) if dtype == "f16" else (-133, 100)
    size = torch.exp2(torch.randint(low, high + 1, (n, columns), generator=gen(8), device="cuda").double()).repeat_interleave(128, 1)[:, : x.shape[1]]
    x = (torch.randint(-15, 16, x.shape, generator=gen(9), device="cuda").double() / 8 * size).to(TYPES[dtype])
    least = torch.finfo(TYPES[dtype]).tiny
    for part, factor in ((x, 2.0**-20), (torch.where(size <= 2.0 ** (low + 12), x, torch.zeros_like(x)), 2.0**80)):
        dy *= factor if dtype == "bf16" else 1.0
        out, p = gradient(asp_ctx, blocks, columns, part, dy, dtype)
        xq, dyd = ref.rows_in_8_bits(part), dy.double()
        assert torch.equal(xq.to(TYPES[dtype]).double(), xq) and (xq != 0).any()
        want = ref.stored(p, dyd.T @ xq)
        sizes = ref.stored(p, torch.where(dyd != 0, dyd.abs().clamp(min=least), 0.0).T @ torch.where(xq != 0, xq.abs().clamp(min=least), 0.0))
        room = sizes * ((n + 1) * 2.0**-23) + want.abs() * 2.0**-24 + 2.0**-126
        assert ((out.double() - want).abs() <= room).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
def test_gradient_added_to_what_is_there(asp_ctx, blocks, columns, n, pad, dtype):
    x, dy = factors(blocks, columns, n, pad, dtype)
    before = torch.randn(blocks * columns, 128, 128, generator=gen(5), device="cuda") * 100.0
    once, p = gradient(asp_ctx, blocks, columns, x, dy, dtype)
    out, _ = gradient(asp_ctx, blocks, columns, x, dy, dtype, before)
    want = ref.rows_in_8_bits(x)
    gradient_of = ref.stored(p, dy.double().T @ want)
    size = ref.stored(p, dy.double().abs().T @ want.abs())
    inside = ref.stored(p, torch.ones(dy.shape[1], x.shape[1], dtype=torch.float64, device="cuda")) > 0
    # the sum's own roundings, and one for each of its parts that is added to what is there (parts of at least 768 rows, and 8 at most that share them)
    parts = n // 768 + 9
    room = size * ((n + 1) * 2.0**-23) + parts * (before.double().abs() + size) * 2.0**-24
    assert ((out.double() - before.double() - gradient_of).abs() <= room)[inside].all()
    assert torch.equal(out[~inside], before[~inside]) and (once[~inside] == 0).all()


@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
def test_gradient_added_to_the_smallest_numbers(asp_ctx, blocks, columns, n, pad):
    """Numbers below 2^-126 may count as zero where something is added to them or they are added (each time by less than 2^-126), and nothing more is lost."""
    x, dy = factors(blocks, columns, n, pad, "bf16")
    n_rows = dy.shape[1]
    before = torch.randint(-40, 41, (blocks * columns, 128, 128), generator=gen(5), device="cuda").float() * 2.0**-130
    dy *= 0.0
    dy[0, : n_rows // 2] = 2.0**-40  # (the other rows of the blocks: nothing is added)
    x[0] = 2.0**-80
    out, p = gradient(asp_ctx, blocks, columns, x, dy, "bf16", before)
    added = ref.stored(p, dy.double().T @ ref.rows_in_8_bits(x))
    want = before.double() + added
    assert ((out.double() - want).abs() < 2.0**-126).all()
    kept = (before.abs() >= 2.0**-126) | (before == 0)
    assert torch.equal(out[kept].double(), want[kept].float().double()) and kept.any() and not kept.all()


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_zeros_keep_their_sign_whatever_is_beside_them(asp_ctx, dtype):
    x = torch.zeros(20, 512, dtype=TYPES[dtype], device="cuda")
    x[:, ::3] = -0.0
    x[5:, 7], x[10:, 200] = float("inf"), 3.0
    held, out = Rows8(asp_ctx, 20, 512), torch.empty(20, 512, device="cuda")
    m, blocks = Block8(asp_ctx, 128, 640, [0, 5], range(5)), torch.empty(5, 128, 128, device="cuda")
    values = x.flatten().repeat(8)[: 5 * 128 * 128].contiguous()
    torch.cuda.synchronize()
    held.quantize(x.data_ptr(), 20, dtype)
    held.restore(out.data_ptr(), "f32")
    m.set_values(values.data_ptr(), dtype)
    m.get_values(blocks.data_ptr())
    asp_ctx.synchronize()
    zero = x == 0
    assert same_bits(out[zero], x.float()[zero])
    assert same_bits(blocks.flatten()[values == 0], values.float()[values == 0])
    held.close()
    m.close()


@pytest.mark.parametrize("rows_of_blocks,columns", [(3, 5), (40, 50)])
def test_transposed_blocks_are_zero_until_they_have_values(asp_ctx, rows_of_blocks, columns):
    """Whatever the context has copied to the device before: here a matrix without a zero among its values."""
    from alphasparse_b200 import matrices
    from alphasparse_b200.graph import Matrix

    full, _ = matrices.from_row_lengths(np.full(2048, 2048), 2048, seed=2)
    Block8.from_matrix(asp_ctx, Matrix.from_csr(full), transposed=True).close()
    n_rows, n_cols = 128 * rows_of_blocks, 128 * columns
    m = Block8(asp_ctx, n_rows, n_cols, *pattern(1, n_rows, n_cols, 1.0), transposed=True)
    for transposed in (False, True):
        c, r = (n_rows, n_cols) if transposed else (n_cols, n_rows)
        for n in (1, 20, 100):
            x, held = torch.ones(n, c, device="cuda"), Rows8(asp_ctx, n, c)
            y, y1 = torch.full((n, r), 7.0, device="cuda"), torch.full((min(n, 32), r), 7.0, device="cuda")
            torch.cuda.synchronize()
            held.quantize(x.data_ptr(), n, "f32")
            m.product(held, y.data_ptr(), "f32", transposed=transposed)
            m.apply(x.data_ptr(), min(n, 32), "f32", y1.data_ptr(), "f32", transposed=transposed)
            asp_ctx.synchronize()
            assert (y == 0).all() and (y1 == 0).all(), (transposed, n)
            held.close()
    m.close()


@pytest.mark.parametrize("dtype,rows_a_sum", [("bf16", 1280), ("f16", 768)])
@pytest.mark.parametrize("blocks,columns,n,pad", [(1, 150, 9000, 0), (2, 100, 9000, 0), (1, 2, 9000, 0), (2, 3, 9000, 1), (3, 70, 9000, 1)])
def test_long_sums_of_gradients_are_rounded(asp_ctx, blocks, columns, n, pad, dtype, rows_a_sum):
    """Products of one sign. A tensor core cuts off less than 2^-23 of the sum each time it adds (16 rows): to a sum that grows evenly, over 1280 (768) rows, less than
    (80 + 1) / 2 (24.5) times 2^-23; the sums are added up with half a step each. Sums that are shared by up to 8 CTAs are shorter, and as many more are added.
    (All 9000 rows in one sum came to 55 and 201 times 2^-23.)"""
    g = gen(n)
    n_rows, n_cols = 128 * blocks - 8, 128 * columns - 5
    x = (torch.rand(n, n_cols, generator=g, device="cuda") + 0.5).to(TYPES[dtype])
    dy = (torch.rand(n, n_rows + (8 if pad == 0 else pad), generator=g, device="cuda") + 0.5).to(TYPES[dtype])[:, :n_rows]
    out, p = gradient(asp_ctx, blocks, columns, x, dy, dtype)
    want = ref.stored(p, dy.double().T @ ref.rows_in_8_bits(x))
    inside = want > 0
    sums = -(-n // rows_a_sum) + 8
    off = ((out.double() - want).abs() / want)[inside].max().item()
    assert off < ((rows_a_sum / 16 + 1) / 2 + sums / 2) * 2.0**-23, off * 2.0**23


def test_contexts_are_made_while_another_stream_is_captured():
    x, made = torch.zeros(8, device="cuda"), []
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        x.add_(1.0)
        made.append(capi.Context(0))
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1.0).all()
    ctx = made[0]
    m, y = Block8(ctx, 128, 128, [0, 1], [0]), torch.full((1, 128), 7.0, device="cuda")
    rows_of_ones = torch.ones(1, 128, device="cuda")
    torch.cuda.synchronize()
    m.apply(rows_of_ones.data_ptr(), 1, "f32", y.data_ptr(), "f32")
    ctx.synchronize()
    assert (y == 0.0).all()
    m.close()
    ctx.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("blocks,columns,n,pad", WAYS)
def test_gradient_of_the_largest_numbers_added_replayed_and_beside_another(asp_ctx, blocks, columns, n, pad, dtype):
    x, dy = factors(blocks, columns, n, pad, dtype)
    x = with_largest(x, dtype, 0.1)
    if dtype == "bf16":
        dy *= 2.0**-30
    want = ref.rows_in_8_bits(x)
    once, p = gradient(asp_ctx, blocks, columns, x, dy, dtype)
    other = capi.Context(0)
    sets = []
    for ctx in (asp_ctx, other):
        m, held = Block8(ctx, dy.shape[1], x.shape[1], *p), Rows8(ctx, n, x.shape[1])
        sets.append((ctx, m, held, torch.full_like(once, 7.0)))
    torch.cuda.synchronize()
    for k in range(3):  # both at once
        for ctx, m, held, out in sets:
            held.quantize(x.data_ptr(), n, dtype)
            m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), dy.stride(0))
    for ctx, m, held, out in sets:
        ctx.synchronize()
        assert torch.equal(out, once)
    # captured: set, then added to twice
    ctx, m, held, out = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream)):
        held.quantize(x.data_ptr(), n, dtype)
        m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), dy.stride(0))
        m.gradient(held, dy.data_ptr(), dtype, out.data_ptr(), dy.stride(0), accumulate=True)
    for _ in range(2):
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        sizes = ref.stored(p, dy.double().abs().T @ want.abs())
        parts = n // 768 + 10  # that are added to what is there, half a step each
        assert ((out.double() - 2 * once.double()).abs() <= sizes * (2 * (n + 1) + parts) * 2.0**-23 + 2.0**-126).all()
    del graph
    for ctx, m, held, out in sets:
        m.close()
        held.close()
    other.close()
