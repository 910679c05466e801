"""CPU suite: patterns of block-sparse 8-bit matrices and the refusals of their entry points, which come before any device is touched; the
64-bit definition that the GPU tests compare with, against torch's own e4m3."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import block8_ref as ref
from alphasparse_b200 import block8, capi
from test_capi_load import declared_functions


def test_every_declared_function_is_exported_and_bound():
    L = block8._lib()
    names = declared_functions("asp_b200_block8.h")
    assert set(block8.EXPORTS) == set(names)
    for n in names:
        assert getattr(L, n).argtypes is not None


def status(n_rows, n_cols, ptr, col):
    """asp_block8_create without a context: 1 with "ctx is NULL" where the pattern is a good one."""
    L = block8._lib()
    ptr, col = np.asarray(ptr, dtype=np.int64), np.asarray(col, dtype=np.uint32)
    out = C.c_void_p(1)
    st = L.asp_block8_create(None, n_rows, n_cols, ptr.ctypes.data, col.ctypes.data if col.size else None, 1, C.byref(out))
    assert not out.value
    return st, L.asp_last_error()


@pytest.mark.parametrize("n_rows,n_cols,ptr,col", [
    (1, 1, [0, 1], [0]), (128, 128, [0, 0], []), (129, 300, [0, 3, 3], [0, 1, 2]), (300, 129, [0, 0, 2, 3], [0, 1, 1]),
])
def test_good_patterns(n_rows, n_cols, ptr, col):
    assert status(n_rows, n_cols, ptr, col) == (1, b"ctx is NULL")


@pytest.mark.parametrize("n_rows,n_cols,ptr,col,want", [
    (0, 1, [0], [], 1), (1, 0, [0, 0], [], 1), (2**31 - 1, 1, [0, 0], [], 1), (1, 2**40, [0, 0], [], 1),
    (129, 300, [1, 3, 3], [0, 1, 2], 5),   # does not start at 0
    (129, 300, [0, 3, 2], [0, 1, 2], 5),   # decreases
    (129, 300, [0, 2, 3], [0, 3, 0], 5),   # behind the last block column
    (129, 300, [0, 2, 3], [1, 0, 0], 5),   # descends
    (129, 300, [0, 2, 3], [1, 1, 0], 5),   # twice
    (129, 300, [0, 2, 3], [], 1),          # no columns
    (129, 300, [0, 0, 2**24], [], 2),
])
def test_bad_patterns(n_rows, n_cols, ptr, col, want):
    st, why = status(n_rows, n_cols, ptr, col)
    assert st == want and why and why != b"ctx is NULL"


def test_null_arguments():
    L = block8._lib()
    out = C.c_void_p(1)
    assert L.asp_block8_create(None, 1, 1, None, None, 0, C.byref(out)) == 1 and not out.value
    assert L.asp_block8_create(None, 1, 1, None, None, 0, None) == 1
    assert L.asp_block8_from_matrix(None, None, 0, C.byref(out)) == 1
    assert L.asp_rows8_create(None, 0, 5, C.byref(out)) == 1 and L.asp_rows8_create(None, 5, 2**31, C.byref(out)) == 1
    assert L.asp_rows8_create(None, 5, 5, C.byref(out)) == 1 and L.asp_last_error() == b"ctx is NULL"
    assert L.asp_rows8_quantize(None, None, None, 4, 0, 0) == 1
    assert L.asp_rows8_restore(None, None, None, 4, 0) == 1
    assert L.asp_block8_set_values(None, None, None, 4) == 1 and L.asp_block8_get_values(None, None, None) == 1
    assert L.asp_block8_apply(None, None, 0, None, 4, 0, 0, None, 4, 0) == 1
    assert L.asp_block8_product(None, None, 0, None, None, 4, 0) == 1
    assert L.asp_block8_gradient(None, None, None, None, 7, 0, None, 0) == 1
    assert L.asp_block8_pattern(None, None, None) == 1
    assert L.asp_rows8_count(None) == 0 and L.asp_block8_blocks(None) == 0 and L.asp_block8_bytes(None) == 0
    L.asp_rows8_destroy(None)
    L.asp_block8_destroy(None)


def test_python_refuses_arrays_that_do_not_fit():
    for ptr, col in (([0, 1], [0]), ([0, 1, 1], []), ([0, 1, 1], [0, 0]), ([[0, 1, 1]], [0])):
        with pytest.raises(ValueError):
            block8.Block8(None, 200, 200, ptr, col)


def test_definition_against_torch():
    """torch rounds to e4m3 the same way; the scale is the smallest power of two that keeps the block's largest within 448."""
    g = torch.Generator()
    g.manual_seed(1)
    x = torch.randn(300, 128, generator=g) * torch.exp2(torch.randint(-40, 40, (300, 1), generator=g).float())
    x[7] = 0.0
    x[8, 0], x[8, 1:] = 448.0, 1.0
    x[9, 0], x[9, 1:] = 448.00003, 1.0
    got = ref.rows_in_8_bits(x)
    most = x.abs().amax(1, keepdim=True).double()
    k = torch.where(most > 0, torch.ceil(torch.log2(most / 448.0)), -126.0)
    assert k[8] == 0 and k[9] == 1
    want = (x.double() * torch.exp2(-k)).float().to(torch.float8_e4m3fn).double() * torch.exp2(k)
    assert torch.equal(got, want) and torch.equal(ref.rows_in_8_bits(got), got)
    assert ((got - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0**-4, torch.exp2(k - 10))).all()


def test_definition_where_numbers_are_not_finite():
    x = torch.ones(2, 200)
    x[0, 3], x[0, 4], x[1, 130] = float("inf"), float("nan"), -float("inf")
    got = ref.rows_in_8_bits(x)
    assert got.isnan().sum() == 3 and got[0, 3].isnan() and got[0, 4].isnan() and got[1, 130].isnan()
    assert (got[~got.isnan()] == 1.0).all()


def test_blocks_of_a_dense_matrix():
    full = torch.arange(300 * 200, dtype=torch.float64).reshape(300, 200)
    p = (np.array([0, 2, 2, 3]), np.array([0, 1, 1]))
    s = ref.stored(p, full)
    assert s.shape == (3, 128, 128) and (s[1, :, 72:] == 0).all() and (s[2, 44:] == 0).all()
    back = ref.dense(p, (300, 200), s)
    assert torch.equal(back[:128], full[:128]) and (back[128:256] == 0).all() and (back[256:, :128] == 0).all() and torch.equal(back[256:, 128:], full[256:, 128:])


def test_rules_on_sizes(tmp_path):
    exe = str(tmp_path / "block8_plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", os.path.join(os.path.dirname(os.path.abspath(__file__)), "block8_plan.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("args", [(0, None, 4, 0, 0, 0, 4, 0), (0, 0, 4, 0.0, 0, 0, 4, 0), (0, 0, 4, 0, 0, 0, 4), (0, 0, "f32", 0, 0, 0, 4, 0)])
def test_apply_without_ctypes_takes_ints_only(args):
    handle, matrix = C.c_void_p(), C.c_void_p()
    call = capi._native().Apply(C.cast(block8._lib().asp_block8_apply, C.c_void_p).value, C.addressof(handle), C.addressof(matrix))
    with pytest.raises(TypeError):
        call(*args)
    # handles are read at the call: a closed context or matrix is NULL to the library
    assert call(0, 16, 4, 1, 0, 16, 4, 0) == 1 and capi.lib().asp_last_error() == b"NULL argument"


def test_apply_with_and_without_the_binding(monkeypatch):
    def matrix():
        m = object.__new__(block8.Block8)
        m.ctx = object.__new__(capi.Context)
        m.ctx._h, m._h = C.c_void_p(), C.c_void_p()
        m._apply = block8._bind_apply(m.ctx._h, m._h)
        return m

    def none():
        raise ImportError

    for _ in range(2):
        m = matrix()
        for x in (16, None, C.c_void_p(16)):
            with pytest.raises(capi.AspError) as e:
                m.apply(x, 1, "f32", 16, "f32")
            assert e.value.status == 1
        with pytest.raises(C.ArgumentError):
            m.apply(1.5, 1, "f32", 16, "f32")
        monkeypatch.setattr(capi, "_native", none)


CALLS = {
    "asp_rows8_quantize": (C.c_void_p, C.c_int, C.c_uint64, C.c_uint64),
    "asp_rows8_restore": (C.c_void_p, C.c_int, C.c_uint64),
    "asp_block8_set_values": (C.c_void_p, C.c_int),
    "asp_block8_get_values": (C.c_void_p,),
    "asp_block8_product": (C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_uint64),
    "asp_block8_gradient": (C.c_void_p, C.c_void_p, C.c_int, C.c_uint64, C.c_void_p, C.c_int),
}


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_ctypes_hand_on_what_they_are_given(name):
    seen = []
    fn = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p, *CALLS[name])(lambda *args: seen.append(args) or 3)
    ctx, handle = C.c_void_p(0x1230), C.c_void_p(0x4560)
    call = capi._native().Bound(name, C.cast(fn, C.c_void_p).value, C.addressof(ctx), C.addressof(handle))
    args = [2**63 + 16 * i if t in (C.c_void_p, C.c_uint64) else i + 1 for i, t in enumerate(CALLS[name])]
    assert call(*args) == 3 and list(seen[-1]) == [0x1230, 0x4560] + args
    handle.value = ctx.value = None  # both are read at the call
    assert call(*args) == 3 and list(seen[-1]) == [None, None] + args
    for bad in ([None] + args[1:], args[1:], args + [0], args[:-1] + [1.5]):
        with pytest.raises(TypeError):
            call(*bad)
    with pytest.raises(ValueError):
        capi._native().Bound("asp_" + name, 0, 0, 0)


def test_closed_handles_and_other_pointers(monkeypatch):
    def none():
        raise ImportError

    for _ in range(2):
        h, ctx = C.c_void_p(), C.c_void_p()
        quantize, product = block8._bind("asp_rows8_quantize", ctx, h), block8._bind("asp_block8_product", ctx, h)
        for x in (16, None, C.c_void_p(16)):
            for call, args in ((quantize, (x, 4, 1, 0)), (product, (False, 0, x, 4, 0))):
                with pytest.raises(capi.AspError) as e:
                    block8._run(call, *args)
                assert e.value.status == 1
        with pytest.raises(C.ArgumentError):
            block8._run(quantize, 1.5, 4, 1, 0)
        monkeypatch.setattr(capi, "_native", none)
