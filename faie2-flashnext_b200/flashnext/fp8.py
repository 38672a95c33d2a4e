"""8-bit rows, weights and their product over torch tensors (include/faie2fn.h, fn_fp8_*): e4m3 codes with a scale for each 128
columns of a row, or each 128 x 128 block of a weight. The reference's GEMVs take fp32 rows (engine/faie2fn.cu:690-1042).

    fn = FN()
    w = Fp8Weight.quantise(fn, weight)                 # [n][k] fp32 or bf16, once; or Fp8Weight(fn, codes, scales)
    x = quantise_rows(fn, h, add=y, total=h, weight=norm, eps=1e-6)    # h += y; rows = 8-bit RMSNorm(h) * norm
    out = w.product(x, dtype=torch.bfloat16)           # [rows][n]; add=: added in
    add_norm(fn, h, y, norm, 1e-6, h, n)               # the residual's addition and the norm alone: h += y, n = RMSNorm(h) * norm

Everything runs on the current stream and returns at once.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from fn import FnFp8
from kv4 import _TYPE, Fixed, _stream

GROUP = 128  # columns (and weight rows) that share a scale
CODES = torch.float8_e4m3fn


class Fp8Rows(NamedTuple):
    """q: e4m3 codes [rows][cols]; scale: fp32 [rows][ceil(cols / 128)]; a code stands for code * scale."""
    q: torch.Tensor
    scale: torch.Tensor

    def values(self) -> torch.Tensor:
        """What the codes stand for, fp32."""
        return self.q.float() * self.scale.repeat_interleave(GROUP, 1)[:, :self.q.shape[1]]


def _wants(name, x, shape, dtype, index):
    """The error for a matrix that is not fp32 or bf16 (or of the given type) [rows][cols] (or of the given shape) with adjacent columns
    on CUDA device `index` (< 0: any)."""
    raise ValueError(f"{name}: {'fp32 or bf16' if dtype is None else dtype} {'[rows][cols]' if shape is None else tuple(shape)} on "
                     f"{'a CUDA device' if index < 0 else f'cuda:{index}'} with adjacent columns is wanted, got {x.dtype} {tuple(x.shape)} with "
                     f"strides {x.stride()} on {x.device}")


def _like(name, x, shape, dtype, index):
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index or (x.stride(1) != 1 and shape[1] > 1):
        _wants(name, x, shape, dtype, index)


def _codes(name, q, scale, down, index):
    """Contiguous codes [rows][cols] and their scales; down: rows that share one."""
    if q.dtype is not CODES or q.dim() != 2 or not q.is_contiguous() or q.get_device() != index or index < 0 or q.shape[1] % 16 or q.shape[1] < 16:
        raise ValueError(f"{name}: contiguous {CODES} [rows][cols], cols a multiple of 16, on {'a CUDA device' if index < 0 else f'cuda:{index}'} "
                         f"is wanted, got {q.dtype} {tuple(q.shape)} on {q.device}")
    rows, cols = q.shape
    if scale.shape != (-(-rows // down), -(-cols // GROUP)) or scale.dtype is not torch.float32 or not scale.is_contiguous() or \
            scale.get_device() != index:
        raise ValueError(f"{name}: contiguous fp32 scales {(-(-rows // down), -(-cols // GROUP))} on cuda:{index} are wanted, got {scale.dtype} "
                         f"{tuple(scale.shape)} on {scale.device}")


def empty_rows(rows: int, cols: int, device="cuda") -> Fp8Rows:
    return Fp8Rows(torch.empty(rows, cols, dtype=CODES, device=device), torch.empty(rows, -(-cols // GROUP), dtype=torch.float32, device=device))


def quantise_rows(fn, x, add=None, total=None, weight=None, eps: float = 1e-6, normed=None, out: Fp8Rows | None = None) -> Fp8Rows:
    """x [rows][cols] fp32 or bf16 (any row stride) as 8-bit rows. add: rows added first (the sum is rounded to x's type); total: gets
    the sum (may be x or add); weight: fp32 [cols] of an RMSNorm of the sum, else none is taken; normed: gets the normed rows in x's
    type (may be x or add, not total). out: buffers of those sizes, apart from the others, written again."""
    shape, dtype, index = x.shape, x.dtype, x.get_device()
    if len(shape) != 2 or dtype not in _TYPE or index < 0 or x.stride(1) != 1:
        _wants("x", x, None, None, -1)
    rows, cols = shape
    if cols % 16 or cols < 16:
        raise ValueError("x: columns in multiples of 16 are wanted")
    a = t = n = w = None
    at = tt = nt = 0
    if add is not None:
        _like("add", add, shape, dtype, index)
        a, at = add.data_ptr(), add.stride(0)
    if total is not None:
        _like("total", total, shape, dtype, index)
        t, tt = total.data_ptr(), total.stride(0)
    if normed is not None:
        _like("normed", normed, shape, dtype, index)
        n, nt = normed.data_ptr(), normed.stride(0)
    if weight is not None:
        if weight.shape != (cols,) or weight.dtype is not torch.float32 or not weight.is_contiguous() or weight.get_device() != index:
            raise ValueError(f"weight: contiguous fp32 [{cols}] on cuda:{index} is wanted")
        w = weight.data_ptr()
    if out is None:
        out = empty_rows(rows, cols, x.device)
    else:
        _codes("out", out.q, out.scale, 1, index)
        if out.q.shape != shape:
            raise ValueError("out: x's shape is wanted")
    fn.fp8_rows(_TYPE[dtype], x.data_ptr(), x.stride(0), a, at, w, eps, rows, cols, t, tt, n, nt, out.q.data_ptr(), out.scale.data_ptr(),
                _stream(x.device))
    return out


def add_norm(fn, x, add, weight, eps: float, total, normed) -> None:
    """total = x + add (rounded to x's type; total may be x or add), normed = RMSNorm(total) * weight, without 8-bit rows. All fp32 or bf16
    [rows][cols] of one type, any row stride; weight fp32 [cols]."""
    shape, dtype, index = x.shape, x.dtype, x.get_device()
    if len(shape) != 2 or dtype not in _TYPE or index < 0 or x.stride(1) != 1 or shape[1] % 16 or shape[1] < 16:
        _wants("x (columns in multiples of 16)", x, None, None, -1)
    for name, t in (("add", add), ("total", total), ("normed", normed)):
        _like(name, t, shape, dtype, index)
    if weight.shape != (shape[1],) or weight.dtype is not torch.float32 or not weight.is_contiguous() or weight.get_device() != index:
        raise ValueError(f"weight: contiguous fp32 [{shape[1]}] on cuda:{index} is wanted")
    fn.fp8_rows(_TYPE[dtype], x.data_ptr(), x.stride(0), add.data_ptr(), add.stride(0), weight.data_ptr(), eps, shape[0], shape[1], total.data_ptr(),
                total.stride(0), normed.data_ptr(), normed.stride(0), None, None, _stream(x.device))


class Fp8Weight(Fixed):
    """A weight [n][k]: codes q (float8_e4m3fn) and scales of 128 x 128 blocks, fp32 [ceil(n / 128)][ceil(k / 128)]. Their values may be
    written anew (by q.copy_, say), the tensors stay these."""
    FIXED = frozenset(("q", "scale", "rows", "cols"))

    def __init__(self, fn, q, scale):
        _codes("weight", q, scale, GROUP, q.get_device())
        if q.shape[0] < 1 or q.data_ptr() % 16:
            raise ValueError("weight: rows are wanted, codes aligned to 16 bytes")
        self._keep(fn, q, scale)

    def _keep(self, fn, q, scale):
        rows, cols = q.shape  # (a dictionary's update: attributes one by one cost a weight's quantising 1.6 us)
        self.__dict__.update(fn=fn, q=q, scale=scale, dev=q.device, index=q.get_device(), c=None, rows=rows, cols=cols)

    @classmethod
    def quantise(cls, fn, w):
        """From w [n][k] fp32 or bf16 (any row stride)."""
        if w.dim() != 2 or w.dtype not in _TYPE or w.get_device() < 0 or w.stride(1) != 1:
            _wants("w", w, None, None, -1)
        rows, cols = w.shape
        if rows < 1 or cols % 16 or cols < 16:
            raise ValueError("w: rows, and columns in multiples of 16, are wanted")
        q = torch.empty(rows, cols, dtype=CODES, device=w.device)
        scale = torch.empty(-(-rows // GROUP), -(-cols // GROUP), dtype=torch.float32, device=w.device)
        fn.fp8_blocks(_TYPE[w.dtype], w.data_ptr(), w.stride(0), rows, cols, q.data_ptr(), scale.data_ptr(), _stream(w.device))
        self = cls.__new__(cls)
        self._keep(fn, q, scale)
        return self

    def values(self) -> torch.Tensor:
        """What the codes stand for, fp32."""
        s = self.scale.repeat_interleave(GROUP, 0)[:self.rows].repeat_interleave(GROUP, 1)[:, :self.cols]
        return self.q.float() * s

    def product(self, x: Fp8Rows, dtype=torch.float32, add=None, out=None):
        """x weight^T [rows][n], in out's type if it is given, else in dtype (fp32 or bf16); add: added before the one rounding, of
        the result's type (may be out). out: apart from the rows' and the weight's codes and scales."""
        q, scale = x
        _codes("x", q, scale, 1, self.index)
        rows, cols = q.shape
        if self.c is None:
            self.c = C.byref(FnFp8(self.q.data_ptr(), self.scale.data_ptr(), self.rows, self.cols))
        if cols != self.cols:
            raise ValueError(f"x: rows of {self.cols} columns are wanted")
        shape = (rows, self.rows)
        if out is None:
            if dtype not in _TYPE:
                raise ValueError("dtype: fp32 or bf16 is wanted")
            out = torch.empty(shape, dtype=dtype, device=self.dev)
        else:
            dtype = out.dtype
            if dtype not in _TYPE:
                _wants("out", out, shape, None, self.index)
            _like("out", out, shape, dtype, self.index)
        a, at = None, 0
        if add is not None:
            _like("add", add, shape, dtype, self.index)
            a, at = add.data_ptr(), add.stride(0)
        self.fn.fp8_product(self.c, q.data_ptr(), scale.data_ptr(), rows, _TYPE[dtype], a, at, out.data_ptr(), out.stride(0), _stream(self.dev))
        return out
