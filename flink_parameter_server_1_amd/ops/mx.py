"""Microscaled tables: rows in 4 or 8 bits per value, written by index, read back and scored.

A row is cut into blocks of 32 consecutive values; a block is 32 elements and one shared
power of two (an E8M0 byte ``s``, value ``2^(s - 127)``, 255 = NaN):

* ``fp4``: E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives): 4.25 bits a value,
  7.5x smaller than the fp32 table it is written from;
* ``fp8``: E4M3 elements (up to 448): 8.25 bits a value.

The shared exponent is the largest magnitude's less the element format's largest
(``floor(log2 max|x|) - 2`` or ``- 8``), elements are rounded to nearest even and saturated.
A block that holds an infinity or a NaN reads back as NaN.  Every read of an element is
exact in fp32 (and in bf16 down to its smallest normal number), so the only rounding is the
write's: half an element step, ``eps / 2`` of the element type relative to a value that does
not saturate.

Dispatch is by the table's device as for every op: the gfx950 kernels on a GPU, the plain
PyTorch twin (``ops.reference``) on the CPU.  Nothing here is differentiated: tables are
written from rows that the update kernels already produced.
"""
from __future__ import annotations

import sys
from typing import Optional

import torch

from . import _native as N
from . import reference as R

MX_BLOCK = 32
#: bits per element of a table format
MX_FORMATS = {"fp4": 4, "fp8": 8}
_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT_MAX = 2**31 - 1  # (of the kernels' 32-bit sizes)


_pkg = sys.modules[__package__]  # (for the debug switch; an import inside the calls costs a microsecond)


def _launch(what: str, device: int, *args) -> None:
    """``fps_<what>(*args, stream)`` on the current stream of GPU ``device``, made current for the launch."""
    fn = getattr(N.require(), "fps_" + what)
    if device == torch.cuda.current_device():
        rc = fn(*args, N.stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, N.stream_ptr())
    N.check(rc, what)


def _same_device(what: str, a: torch.Tensor, *ts) -> None:
    d = a.get_device()  # -1: the CPU
    for t in ts:
        if t is not None and t.get_device() != d:
            raise ValueError(f"{what}: operands on {a.device} and {t.device}")


class MXTable:
    """``rows x dim`` values in a microscaled format.

    ``data`` uint8 ``[rows, dim_padded * bits / 8]`` (two fp4 elements per byte, the even
    one in the low nibble), ``scale`` uint8 ``[rows, dim_padded / 32]``; ``dim_padded`` is
    ``dim`` rounded up to 32, the elements behind ``dim`` are zero.
    """

    def __init__(self, rows: int, dim: int, fmt: str = "fp4", device="cpu"):
        """A table of zero rows."""
        bits, nblk = self._layout(rows, dim, fmt)
        self._set(torch.zeros((rows, nblk * MX_BLOCK * bits // 8), dtype=torch.uint8, device=device),
                  torch.zeros((rows, nblk), dtype=torch.uint8, device=device), dim, fmt)

    @staticmethod
    def _layout(rows: int, dim: int, fmt: str):
        if fmt not in MX_FORMATS:
            raise ValueError(f"MXTable: format must be one of {tuple(MX_FORMATS)}, not {fmt!r}")
        if dim < 1 or rows < 0 or dim > _INT_MAX - MX_BLOCK:
            raise ValueError(f"MXTable: {rows} rows of {dim} values")
        return MX_FORMATS[fmt], (dim + MX_BLOCK - 1) // MX_BLOCK

    def _set(self, data, scale, dim, fmt):
        self.data, self.scale, self.dim, self.fmt = data, scale, int(dim), fmt
        self.bits = MX_FORMATS[fmt]
        self.rows = data.shape[0]

    @classmethod
    def wrap(cls, data: torch.Tensor, scale: torch.Tensor, dim: int, fmt: str = "fp4") -> "MXTable":
        """A table over existing (contiguous) buffers, not copied.  The elements behind
        ``dim`` must be zero codes."""
        rows = data.shape[0] if data.dim() == 2 else -1
        bits, nblk = cls._layout(max(rows, 0), dim, fmt)
        if data.dtype != torch.uint8 or scale.dtype != torch.uint8:
            raise ValueError("MXTable.wrap: data and scale are uint8")
        if rows < 0 or tuple(data.shape) != (rows, nblk * MX_BLOCK * bits // 8) or tuple(scale.shape) != (rows, nblk):
            raise ValueError(f"MXTable.wrap: data {tuple(data.shape)}, scale {tuple(scale.shape)} do not hold {fmt} rows "
                             f"of {dim} values")
        if not (data.is_contiguous() and scale.is_contiguous()):
            raise ValueError("MXTable.wrap: data and scale must be contiguous")
        if data.data_ptr() % 16:
            raise ValueError("MXTable.wrap: data must start on 16 bytes")
        _same_device("MXTable.wrap", data, scale)
        t = cls.__new__(cls)
        t._set(data, scale, dim, fmt)
        return t

    @classmethod
    def from_rows(cls, rows: torch.Tensor, fmt: str = "fp4") -> "MXTable":
        """The table of the float rows ``rows [n, dim]`` (one launch on the GPU)."""
        if rows.dim() != 2:
            raise ValueError(f"MXTable.from_rows: expected [n, dim] rows, got {tuple(rows.shape)}")
        n, dim = rows.shape
        bits, nblk = cls._layout(n, dim, fmt)
        t = cls.__new__(cls)
        t._set(torch.empty((n, nblk * MX_BLOCK * bits // 8), dtype=torch.uint8, device=rows.device),
               torch.empty((n, nblk), dtype=torch.uint8, device=rows.device), dim, fmt)
        return mx_set_rows(t, None, rows)

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel() + self.scale.numel()

    def values(self, dtype=torch.float32) -> torch.Tensor:
        """All rows as floats."""
        return mx_gather_rows(self, None, out_dtype=dtype)


def _index(what: str, table: MXTable, idx: torch.Tensor) -> torch.Tensor:
    if idx.dtype not in (torch.int32, torch.int64) or idx.dim() != 1 or not idx.is_contiguous():
        raise ValueError(f"{what}: idx must be a contiguous 1-d int32 or int64 tensor")
    _same_device(what, table.data, idx)
    if _pkg.DEBUG:
        _pkg.check_index(idx, table.rows, what, allow_negative=True)
    return idx


def mx_set_rows(table: MXTable, idx: Optional[torch.Tensor], rows: torch.Tensor) -> MXTable:
    """Write ``table[idx[r]] = quantised(rows[r])`` in place; ``idx=None``: row ``r`` to slot ``r``.

    ``rows [n, dim]`` fp32 / bf16 / fp16, contiguous.  An index outside ``[0, table.rows)`` is a
    padding slot and skipped (as ``idx < 0`` of ``apply_rows``; ``FPS_DEBUG=1`` raises for one past
    the table); where an index repeats, the last of its rows is stored whole.  Slots that no row
    names stay as they were.  Calls on one table from several streams must not name the same slot.
    An indexed write of more than one row takes a workspace of 4 bytes per slot."""
    if rows.dim() != 2 or rows.shape[1] != table.dim or rows.dtype not in _TYPE:
        raise ValueError(f"mx_set_rows: rows must be fp32 / bf16 / fp16 [n, {table.dim}], got {rows.dtype} "
                         f"{tuple(rows.shape)}")
    if not rows.is_contiguous():
        raise ValueError("mx_set_rows: rows must be contiguous")
    _same_device("mx_set_rows", table.data, rows)
    n = rows.shape[0]
    if idx is None:
        if n > table.rows:
            raise ValueError(f"mx_set_rows: {n} rows into a table of {table.rows}")
    else:
        idx = _index("mx_set_rows", table, idx)
        if idx.numel() != n:
            raise ValueError(f"mx_set_rows: {idx.numel()} indices for {n} rows")
        if n > _INT_MAX:
            raise ValueError(f"mx_set_rows: {n} indexed rows in one write, at most 2^31 - 1")
    if not rows.is_cuda:
        R.mx_set_rows(table.data, table.scale, table.bits, idx, rows)
        return table
    owner = None
    if idx is not None and n > 1:  # which of a repeated index's rows its slot gets
        owner = torch.empty(table.rows, dtype=torch.int32, device=table.device)
    _launch("mx_set_rows", rows.get_device(), rows.data_ptr(), _TYPE[rows.dtype], N.ptr(idx),
            int(idx is not None and idx.dtype == torch.int64), n, table.dim, table.rows, table.data.data_ptr(),
            table.scale.data_ptr(), table.bits, N.ptr(owner))
    return table


def mx_gather_rows(table: MXTable, idx: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   out_dtype=torch.float32) -> torch.Tensor:
    """Read rows back: ``out[r] = values of table[idx[r]]`` (``idx=None``: all rows), fp32 /
    bf16 / fp16.  An index outside ``[0, table.rows)`` gives a zero row (as ``gather_rows``'
    padding slots)."""
    if idx is not None:
        idx = _index("mx_gather_rows", table, idx)
    n = table.rows if idx is None else idx.numel()
    if out is None:
        if out_dtype not in _TYPE:
            raise ValueError(f"mx_gather_rows: out_dtype must be fp32, bf16 or fp16, not {out_dtype}")
        out = torch.empty((n, table.dim), dtype=out_dtype, device=table.device)
    else:
        if tuple(out.shape) != (n, table.dim) or out.dtype not in _TYPE or not out.is_contiguous():
            raise ValueError(f"mx_gather_rows: out must be contiguous fp32 / bf16 / fp16 [{n}, {table.dim}], got "
                             f"{out.dtype} {tuple(out.shape)}")
        _same_device("mx_gather_rows", table.data, out)
    if not out.is_cuda:
        out.copy_(R.mx_gather_rows(table.data, table.scale, table.bits, table.dim, idx))
        return out
    _launch("mx_gather_rows", out.get_device(), table.data.data_ptr(), table.scale.data_ptr(), table.rows, table.dim,
            table.bits, N.ptr(idx), int(idx is not None and idx.dtype == torch.int64), n, out.data_ptr(), _TYPE[out.dtype])
    return out


def mx_score(Q, X: MXTable, out: Optional[torch.Tensor] = None, out_dtype=torch.float32) -> torch.Tensor:
    """Scores ``out[b, i] = <Q[b], X[i]>`` of every query with every row of a microscaled table
    (K8's product, ``score_gemm``, against 4 or 8 bits).

    ``Q``: bf16 queries ``[B, dim]`` (contiguous), or an fp4 ``MXTable`` against an fp4 ``X`` (both
    sides in 4 bits).  ``out``: fp32 / bf16 / fp16 ``[B, rows]``, its rows may be strided (a column
    slice of a wider score matrix).  Sums are held in fp32 and rounded once.  Against bf16 queries a
    table's values take part as bf16: exact, but for elements of fp8 blocks whose largest value is below
    2^-116, which are rounded to whole multiples of 2^-133.  A NaN in a query row or a NaN block in a
    table row makes its scores NaN."""
    mx = isinstance(Q, MXTable)
    if not isinstance(X, MXTable):
        raise ValueError("mx_score: X must be an MXTable")
    if mx:
        if Q.fmt != "fp4" or X.fmt != "fp4":
            raise ValueError(f"mx_score: {Q.fmt} queries against an {X.fmt} table: microscaled queries are fp4 against "
                             "fp4 (pass bf16 queries otherwise)")
        B, dim = Q.rows, Q.dim
    else:
        if Q.dim() != 2 or Q.dtype != torch.bfloat16 or not Q.is_contiguous():
            raise ValueError(f"mx_score: queries must be contiguous bf16 [B, dim] or an fp4 MXTable, got {Q.dtype} "
                             f"{tuple(Q.shape)}")
        B, dim = Q.shape
    if dim != X.dim:
        raise ValueError(f"mx_score: queries of {dim} values, table rows of {X.dim}")
    if B > _INT_MAX:
        raise ValueError(f"mx_score: {B} queries in one call, at most 2^31 - 1")
    if out is None:
        if out_dtype not in _TYPE:
            raise ValueError(f"mx_score: out_dtype must be fp32, bf16 or fp16, not {out_dtype}")
        out = torch.empty((B, X.rows), dtype=out_dtype, device=X.device)
    elif tuple(out.shape) != (B, X.rows) or out.dtype not in _TYPE:
        raise ValueError(f"mx_score: out must be fp32 / bf16 / fp16 [{B}, {X.rows}], got {out.dtype} {tuple(out.shape)}")
    elif out.numel() and (out.stride(1) != 1 and X.rows > 1 or B > 1 and out.stride(0) < X.rows):
        raise ValueError(f"mx_score: out's rows must be contiguous and apart, got strides {out.stride()}")
    _same_device("mx_score", X.data, Q.data if mx else Q, out)
    if out.numel() == 0:
        return out
    if not out.is_cuda:
        q = R.mx_decode(Q.data, Q.scale, Q.bits, dim) if mx else Q.float()
        out.copy_(q.detach() @ R.mx_decode(X.data, X.scale, X.bits, dim).t())
        return out
    ld = out.stride(0) if B > 1 else X.rows
    _launch("mx_score", out.get_device(), Q.data.data_ptr() if mx else Q.data_ptr(), Q.scale.data_ptr() if mx else None,
            X.data.data_ptr(), X.scale.data_ptr(), X.bits, B, X.rows, dim, out.data_ptr(), _TYPE[out.dtype], ld)
    return out
