"""Block-sparse matrices in 8 bits, rows in 8 bits, their products and gradients (include/asp_b200_block8.h).

Everything takes device pointers (ints) and runs on the stream of its Context, like PlanGroup.spmv; types are "f32", "f16" and
"bf16". `ld` is the distance of two rows in elements, 0 for rows that lie side by side.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from . import capi, graph

BLOCK = 128
APPLY_ROWS = 32  # most rows of Block8.apply
TYPES = {"f32": capi.F32, "f16": 6, "bf16": 7}

EXPORTS = [
    "asp_rows8_create", "asp_rows8_destroy", "asp_rows8_quantize", "asp_rows8_restore", "asp_rows8_count", "asp_block8_create", "asp_block8_from_matrix",
    "asp_block8_destroy", "asp_block8_blocks", "asp_block8_pattern", "asp_block8_bytes", "asp_block8_set_values", "asp_block8_get_values", "asp_block8_apply",
    "asp_block8_product", "asp_block8_gradient",
]

_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = capi.lib()
        p, u64, i32, out = C.c_void_p, C.c_uint64, C.c_int, C.POINTER(C.c_void_p)
        for name, args, result in (
            ("asp_rows8_create", [p, u64, u64, out], i32), ("asp_rows8_destroy", [p], None), ("asp_rows8_quantize", [p, p, p, i32, u64, u64], i32),
            ("asp_rows8_restore", [p, p, p, i32, u64], i32), ("asp_rows8_count", [p], u64), ("asp_block8_create", [p, u64, u64, p, p, i32, out], i32),
            ("asp_block8_from_matrix", [p, p, i32, out], i32), ("asp_block8_destroy", [p], None), ("asp_block8_blocks", [p], u64),
            ("asp_block8_pattern", [p, p, p], i32), ("asp_block8_bytes", [p], u64), ("asp_block8_set_values", [p, p, p, i32], i32),
            ("asp_block8_get_values", [p, p, p], i32), ("asp_block8_apply", [p, p, i32, p, i32, u64, u64, p, i32, u64], i32),
            ("asp_block8_product", [p, p, i32, p, p, i32, u64], i32), ("asp_block8_gradient", [p, p, p, p, i32, u64, p, i32], i32),
        ):
            fn = getattr(L, name)
            fn.argtypes, fn.restype = args, result
        _bound = L
    return _bound


def _bind_apply(ctx_handle, handle):
    """asp_block8_apply(ctx, matrix, ...) with the first two given, without ctypes where that binding has been built. Both handles are read at every
    call; the caller keeps them alive."""
    try:
        native = capi._native().Apply
    except (ImportError, AttributeError):
        fn = _lib().asp_block8_apply
        return lambda *args: fn(ctx_handle, handle, *args)
    return native(C.cast(_lib().asp_block8_apply, C.c_void_p).value, C.addressof(ctx_handle), C.addressof(handle))


def _bind(name, ctx_handle, handle):
    """Another call of (context, handle, ...) with the two given: without ctypes where that binding has been built, and through it. Both handles are read at
    every call; the caller keeps them alive."""
    fn = getattr(_lib(), name)
    plain = functools.partial(fn, ctx_handle, handle)
    try:
        native = capi._native().Bound
    except (ImportError, AttributeError):
        return plain, plain
    return native(name, C.cast(fn, C.c_void_p).value, C.addressof(ctx_handle), C.addressof(handle)), plain


def _run(call, *args) -> None:
    try:
        status = call[0](*args)
    except TypeError:  # whatever else ctypes takes for a pointer
        status = call[1](*args)
    if status:
        capi.check(status)


class Rows8:
    """asp_rows8: up to max_rows rows of n_cols columns in 8 bits, a scale for each row and 128 columns."""

    def __init__(self, ctx: capi.Context, max_rows: int, n_cols: int):
        self._h = C.c_void_p()
        self.ctx, self.max_rows, self.n_cols = ctx, max_rows, n_cols
        capi.check(_lib().asp_rows8_create(ctx.handle, max_rows, n_cols, C.byref(self._h)))
        self._ctx_handle = ctx.handle  # kept alive: calls may have no more than its address and that of our own
        self._quantize, self._restore = (_bind(name, self._ctx_handle, self._h) for name in ("asp_rows8_quantize", "asp_rows8_restore"))

    def __len__(self) -> int:
        """Rows held."""
        return int(_lib().asp_rows8_count(self._h))

    def quantize(self, x: int, n: int, dtype: str, ld: int = 0) -> None:
        """n rows at x to 8 bits."""
        _run(self._quantize, x, TYPES[dtype], n, ld)

    def restore(self, out: int, dtype: str, ld: int = 0) -> None:
        """What the rows held stand for."""
        _run(self._restore, out, TYPES[dtype], ld)

    def close(self):
        if self._h:
            _lib().asp_rows8_destroy(self._h)
            self._h.value = None  # (in place: its address is held)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Block8:
    """asp_block8: an n_rows x n_cols matrix of which 128 x 128 blocks are stored, in 8 bits with a scale each. block_ptr, block_col:
    the blocks by block row, as in CSR. transposed: products with the transposed matrix are wanted, too."""

    def __init__(self, ctx: capi.Context, n_rows: int, n_cols: int, block_ptr, block_col, transposed: bool = False):
        ptr, col = np.asarray(block_ptr), np.asarray(block_col)
        for a in (ptr, col):
            if a.dtype.kind not in "iu" and a.size and not (a.dtype.kind in "bf" and np.isfinite(a).all() and (a == np.trunc(a)).all()):
                raise ValueError("block_ptr, block_col: whole numbers")
        ptr = np.ascontiguousarray(ptr, dtype=np.int64)
        if col.size and (col.min() < 0 or col.max() >= 2**32):
            raise ValueError("block_col: block columns")
        col = np.ascontiguousarray(col, dtype=np.uint32)
        if ptr.ndim != 1 or ptr.shape[0] != -(-n_rows // BLOCK) + 1 or col.ndim != 1 or (ptr[-1] != col.shape[0]):
            raise ValueError("block_ptr has an entry for each block row and one more, the last of them the number of blocks")
        h = C.c_void_p()
        capi.check(_lib().asp_block8_create(ctx.handle, n_rows, n_cols, ptr.ctypes.data, col.ctypes.data, int(transposed), C.byref(h)))
        self._take(ctx, h, n_rows, n_cols)

    @classmethod
    def from_matrix(cls, ctx: capi.Context, matrix: graph.Matrix, transposed: bool = False) -> "Block8":
        """The blocks of `matrix` that have an entry, with its values."""
        self = cls.__new__(cls)
        h = C.c_void_p()
        capi.check(_lib().asp_block8_from_matrix(ctx.handle, matrix._h, int(transposed), C.byref(h)))
        self._take(ctx, h, *matrix.shape)
        return self

    def _take(self, ctx, h, n_rows, n_cols):
        self._h, self.ctx, self.n_rows, self.n_cols = h, ctx, n_rows, n_cols
        self._ctx_handle = ctx.handle  # kept alive: calls may have no more than its address and that of our own
        self._apply = _bind_apply(self._ctx_handle, h)
        self._set, self._get, self._product, self._gradient = (
            _bind(f"asp_block8_{name}", self._ctx_handle, h) for name in ("set_values", "get_values", "product", "gradient"))
        self.n_blocks = int(_lib().asp_block8_blocks(h))

    def pattern(self):
        """(block_ptr, block_col)"""
        ptr, col = np.zeros(-(-self.n_rows // BLOCK) + 1, dtype=np.int64), np.zeros(self.n_blocks, dtype=np.uint32)
        capi.check(_lib().asp_block8_pattern(self._h, ptr.ctypes.data, col.ctypes.data))
        return ptr, col

    def bytes(self) -> int:
        return int(_lib().asp_block8_bytes(self._h))

    def set_values(self, values: int, dtype: str) -> None:
        """New values of all stored blocks, [n_blocks, 128, 128]."""
        _run(self._set, values, TYPES[dtype])

    def get_values(self, values: int) -> None:
        """What the stored blocks stand for, [n_blocks, 128, 128] in 32 bits."""
        _run(self._get, values)

    def apply(self, x: int, n: int, x_dtype: str, y: int, y_dtype: str, ldx: int = 0, ldy: int = 0, transposed: bool = False) -> None:
        """y = A x (transposed: A^T x) for n <= 32 rows x in 16 or 32 bits, converted to 8 bits on the way."""
        args = (transposed, x, TYPES[x_dtype], n, ldx, y, TYPES[y_dtype], ldy)
        try:
            status = self._apply(*args)
        except TypeError:  # whatever else ctypes takes for a pointer
            status = _lib().asp_block8_apply(self.ctx.handle, self._h, *args)
        if status:
            capi.check(status)

    def product(self, x: Rows8, y: int, dtype: str, ld: int = 0, transposed: bool = False) -> None:
        """y = A x (transposed: A^T x) for the rows that x holds."""
        _run(self._product, transposed, x._h.value or 0, y, TYPES[dtype], ld)

    def gradient(self, x: Rows8, dy: int, dtype: str, out: int, ld: int = 0, accumulate: bool = False) -> None:
        """The gradient by the stored blocks, [n_blocks, 128, 128] in 32 bits, from dy and the rows x kept in 8 bits."""
        _run(self._gradient, x._h.value or 0, dy, TYPES[dtype], ld, out, int(accumulate))

    def close(self):
        if self._h:
            _lib().asp_block8_destroy(self._h)
            self._h.value = None  # (in place: its address is held)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
