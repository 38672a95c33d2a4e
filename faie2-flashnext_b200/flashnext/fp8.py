"""8-bit rows, weights and their product over torch tensors (include/faie2fn.h, fn_fp8_*): e4m3 codes with a scale for each 128
columns of a row, or each 128 x 128 block of a weight. The reference's GEMVs take fp32 rows (engine/faie2fn.cu:690-1042).

    fn = FN()
    w = Fp8Weight.quantise(fn, weight)                 # [n][k] fp32 or bf16, once; or Fp8Weight(fn, codes, scales)
    x = quantise_rows(fn, h, add=y, total=h, weight=norm, eps=1e-6)    # h += y; rows = 8-bit RMSNorm(h) * norm
    out = w.product(x, dtype=torch.bfloat16)           # [rows][n]; add=: added in

Everything runs on the current stream and returns at once.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from fn import FnFp8
from kv4 import _TYPE, _stream

GROUP = 128  # columns (and weight rows) that share a scale
CODES = torch.float8_e4m3fn


class Fp8Rows(NamedTuple):
    """q: e4m3 codes [rows][cols]; scale: fp32 [rows][ceil(cols / 128)]; a code stands for code * scale."""
    q: torch.Tensor
    scale: torch.Tensor

    def values(self) -> torch.Tensor:
        """What the codes stand for, fp32."""
        return self.q.float() * self.scale.repeat_interleave(GROUP, 1)[:, :self.q.shape[1]]


def _matrix(name, x, shape=None, dtype=None, dev=None):
    """An fp32 or bf16 matrix on the GPU with adjacent columns, of the given shape, type and device."""
    if x.dim() != 2 or x.dtype not in _TYPE or (x.stride(1) != 1 and x.shape[1] > 1) or not x.is_cuda or \
            (shape is not None and x.shape != shape) or (dtype is not None and x.dtype != dtype) or (dev is not None and x.device != dev):
        raise ValueError(f"{name}: {'fp32 or bf16' if dtype is None else dtype} {'[rows][cols]' if shape is None else tuple(shape)} on "
                         f"{'a CUDA device' if dev is None else dev} with adjacent columns is wanted, got {x.dtype} {tuple(x.shape)} on {x.device}")


def _codes(name, q, scale, down, dev=None):
    """Contiguous codes [rows][cols] and their scales; down: rows that share one."""
    if q.dim() != 2 or q.dtype != CODES or not q.is_contiguous() or not q.is_cuda or q.shape[1] % 16 or q.shape[1] < 16 or \
            (dev is not None and q.device != dev):
        raise ValueError(f"{name}: contiguous {CODES} [rows][cols], cols a multiple of 16, on {'a CUDA device' if dev is None else dev} is "
                         f"wanted, got {q.dtype} {tuple(q.shape)} on {q.device}")
    want = (-(-q.shape[0] // down), -(-q.shape[1] // GROUP))
    if scale.shape != want or scale.dtype != torch.float32 or not scale.is_contiguous() or scale.device != q.device:
        raise ValueError(f"{name}: contiguous fp32 scales {want} on {q.device} are wanted, got {scale.dtype} {tuple(scale.shape)} on "
                         f"{scale.device}")


def empty_rows(rows: int, cols: int, device="cuda") -> Fp8Rows:
    return Fp8Rows(torch.empty(rows, cols, dtype=CODES, device=device), torch.empty(rows, -(-cols // GROUP), device=device))


def quantise_rows(fn, x, add=None, total=None, weight=None, eps: float = 1e-6, normed=None, out: Fp8Rows | None = None) -> Fp8Rows:
    """x [rows][cols] fp32 or bf16 (any row stride) as 8-bit rows. add: rows added first (the sum is rounded to x's type); total: gets
    the sum (may be x or add); weight: fp32 [cols] of an RMSNorm of the sum, else none is taken; normed: gets the normed rows in x's
    type. out: buffers of those sizes, written again."""
    _matrix("x", x)
    rows, cols = x.shape
    if cols % 16 or cols < 16:
        raise ValueError("x: columns in multiples of 16 are wanted")
    for name, t in (("add", add), ("total", total), ("normed", normed)):
        if t is not None:
            _matrix(name, t, x.shape, x.dtype, x.device)
    if weight is not None and (weight.shape != (cols,) or weight.dtype != torch.float32 or not weight.is_contiguous() or weight.device != x.device):
        raise ValueError(f"weight: contiguous fp32 [{cols}] on {x.device} is wanted")
    if out is None:
        out = empty_rows(rows, cols, x.device)
    else:
        _codes("out", out.q, out.scale, 1, x.device)
        if out.q.shape != x.shape:
            raise ValueError("out: x's shape is wanted")
    p = lambda t: (None, 0) if t is None else (t.data_ptr(), t.stride(0))  # noqa: E731
    fn.fp8_rows(_TYPE[x.dtype], *p(x), *p(add), p(weight)[0], eps, rows, cols, *p(total), *p(normed), out.q.data_ptr(),
                out.scale.data_ptr(), _stream(x.device))
    return out


class Fp8Weight:
    """A weight [n][k]: codes q (float8_e4m3fn) and scales of 128 x 128 blocks, fp32 [ceil(n / 128)][ceil(k / 128)]."""

    def __init__(self, fn, q, scale):
        _codes("weight", q, scale, GROUP)
        if q.shape[0] < 1 or q.data_ptr() % 16:
            raise ValueError("weight: rows are wanted, codes aligned to 16 bytes")
        self.fn, self.q, self.scale, self.dev = fn, q, scale, q.device
        self.rows, self.cols = q.shape
        self.c = C.byref(FnFp8(q.data_ptr(), scale.data_ptr(), self.rows, self.cols))

    @classmethod
    def quantise(cls, fn, w):
        """From w [n][k] fp32 or bf16 (any row stride)."""
        _matrix("w", w)
        rows, cols = w.shape
        if rows < 1 or cols % 16 or cols < 16:
            raise ValueError("w: rows, and columns in multiples of 16, are wanted")
        q = torch.empty(rows, cols, dtype=CODES, device=w.device)
        scale = torch.empty(-(-rows // GROUP), -(-cols // GROUP), device=w.device)
        fn.fp8_blocks(_TYPE[w.dtype], w.data_ptr(), w.stride(0), rows, cols, q.data_ptr(), scale.data_ptr(), _stream(w.device))
        return cls(fn, q, scale)

    def values(self) -> torch.Tensor:
        """What the codes stand for, fp32."""
        s = self.scale.repeat_interleave(GROUP, 0)[:self.rows].repeat_interleave(GROUP, 1)[:, :self.cols]
        return self.q.float() * s

    def product(self, x: Fp8Rows, dtype=torch.float32, add=None, out=None):
        """x weight^T [rows][n], in out's type if it is given, else in dtype (fp32 or bf16); add: added before the one rounding, of
        the result's type (may be out)."""
        _codes("x", x.q, x.scale, 1, self.dev)
        if x.q.shape[1] != self.cols:
            raise ValueError(f"x: rows of {self.cols} columns are wanted")
        shape = (x.q.shape[0], self.rows)
        if out is None:
            if dtype not in _TYPE:
                raise ValueError("dtype: fp32 or bf16 is wanted")
            out = torch.empty(shape, dtype=dtype, device=self.dev)
        else:
            _matrix("out", out, shape, None, self.dev)
        if add is not None:
            _matrix("add", add, shape, out.dtype, self.dev)
        self.fn.fp8_product(self.c, x.q.data_ptr(), x.scale.data_ptr(), shape[0], _TYPE[out.dtype], None if add is None else add.data_ptr(),
                            0 if add is None else add.stride(0), out.data_ptr(), out.stride(0), _stream(self.dev))
        return out
