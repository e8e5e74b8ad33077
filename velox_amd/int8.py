"""Products of 8-bit integers on torch tensors: weights with a scale for each output channel, activations with one for each
token.

Thin calls of the C ABI (include/velox_hip.h, "8-bit integer products"), in the manner of velox_amd.paged: a call checks
types, shapes and devices (ValueError), launches on the current stream of the matrix's device and returns without waiting;
a status other than 0 raises. No backward pass: with gradients enabled, tensors that require one are refused. Calls can be
captured into a graph once `out` and `workspace` are given. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .paged import _DTYPES, _call, _gpu, _need, _no_gradient, _numbers, _space


_ROWS = 1 << 23  # of many more rows, those of a call (the C ABI takes fewer than 2^24)


def _plain(t: torch.Tensor, device: torch.device, what: str, width: int = 0, rows: int = -1) -> tuple[L.Rows, int]:
    """[row][element] as VeloxHipRows, and its rows; the elements of a row are next to each other."""
    code = _DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if code is None or t.device != device or t.dim() != 2:
        raise ValueError(f"{what}: a float32, float16 or bfloat16 tensor [row][element] on {device} is wanted")
    if t.requires_grad:
        _no_gradient(t, what)
    n, d = t.shape
    if (n | d) >> 32:
        _numbers(what, n, d)
    if (width and d != width) or (rows >= 0 and n != rows):
        raise ValueError(f"{what}: {rows if rows >= 0 else n} rows of {width or d} elements are wanted, got {n} of {d}")
    rs, es = t.stride()
    if es != 1 and d > 1:
        raise ValueError(f"{what}: a row's elements have to be next to each other")
    return L.Rows(t.data_ptr(), code, 1, rs, 0), n


def _result(t: torch.Tensor, device: torch.device, width: int, rows: int) -> L.Rows:
    """The given output: as _plain, its rows apart from each other."""
    o, n = _plain(t, device, "out", width, rows)
    if n > 1 and o.row_stride < width:
        raise ValueError(f"out: rows that do not overlap are wanted, got {width} elements every {o.row_stride}")
    return o


def _floats(t: torch.Tensor, shape: tuple, device: torch.device, what: str) -> int:
    """The address of a contiguous float32 tensor of a shape."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous float32 tensor of shape {shape} on {device} is wanted")
    if t.requires_grad:
        _no_gradient(t, what)
    return t.data_ptr()


def _memory(n: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


class Int8Rows:
    """Activation rows in 8 bits: codes int8 [row][k filled up to a multiple of 128], scales float32 [row]; a value is
    code * scale."""

    def __init__(self, rows: int, k: int, device="cuda"):
        _need(rows >= 0 and k > 0, "rows >= 0 and k > 0 are wanted")
        self.k = k
        self.codes = torch.empty(rows, -(-k // 128) * 128, dtype=torch.int8, device=device)
        self.scales = torch.empty(rows, dtype=torch.float32, device=device)
        self.desc = L.Int8RowsDesc(self.codes.data_ptr(), self.scales.data_ptr(), self.codes.shape[1])

    def _part(self, first: int, last: int) -> "Int8Rows":
        """Rows first .. last - 1, in their place."""
        p = Int8Rows.__new__(Int8Rows)
        p.k, p.codes, p.scales = self.k, self.codes[first:last], self.scales[first:last]
        p.desc = L.Int8RowsDesc(p.codes.data_ptr(), p.scales.data_ptr(), self.codes.shape[1])
        return p

    def __len__(self) -> int:
        return self.codes.shape[0]


class Int8Matrix:
    """Laid-out weights: codes int8 [n][k] with scales float32 [n], or `count` matrices [count][n][k] with [count][n] (the
    experts of experts.ffn). paired: the first n / 2 rows are gate rows, the others their up rows (SwiGLU products).
    Lays them out once; the tensors given are not kept."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, *, paired: bool = False):
        device = _gpu(codes, "codes")
        _need(codes.dtype == torch.int8 and codes.dim() in (2, 3) and codes.stride(-1) == 1 and min(codes.shape) > 0,
              "codes: int8 [n][k] or [matrix][n][k], the elements of a row next to each other")
        if codes.dim() == 2:
            codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
        self.count, self.n, self.k = codes.shape
        self.paired, self.device = bool(paired), device
        self.outputs = self.n // 2 if self.paired else self.n  # values of a product's row
        at = _floats(scales, (self.count, self.n), device, "scales")
        _numbers("codes", self.count, self.n, self.k)
        self.lib = L.load()
        d = L.Int8MatrixDesc(None, None, self.n, self.k, self.count, int(self.paired))
        sizes = C.c_uint64(), C.c_uint64()
        rc = self.lib.velox_hip_int8_layout(C.byref(d), *map(C.byref, sizes))
        _need(rc == 0, "codes: n up to 2^20 (even if paired), k up to 2^17 and up to 1024 matrices are wanted")
        self._codes, self._scales = (torch.empty(s.value, dtype=torch.uint8, device=device) for s in sizes)
        d.codes, d.scales = self._codes.data_ptr(), self._scales.data_ptr()
        self.desc, self._ref, self._index = d, C.byref(d), device.index
        _call(self.lib.velox_hip_int8_pack, device.index, self._ref, 0, self.count, codes.data_ptr(), codes.stride(0), codes.stride(1),
              at, self.n)

    @classmethod
    def quantized(cls, w: torch.Tensor, *, paired: bool = False) -> "Int8Matrix":
        """Of weights [n][k] or [matrix][n][k] of float32, float16 or bfloat16: each row by its largest value (quantize)."""
        _need(isinstance(w, torch.Tensor) and w.dim() in (2, 3) and min(w.shape) > 0, "w: [n][k] or [matrix][n][k] is wanted")
        x = w.reshape(-1, w.shape[-1])
        rows = Int8Rows(*x.shape, _gpu(x, "w"))
        for r in range(0, len(rows), _ROWS):
            quantize(x[r:r + _ROWS], rows._part(r, r + _ROWS))
        return cls(rows.codes.view(*w.shape[:-1], -1)[..., :w.shape[-1]], rows.scales.view(w.shape[:-1]), paired=paired)


def quantize(x: torch.Tensor, out: Int8Rows | None = None) -> Int8Rows:
    """Rows of x [row][k] in 8 bits, each by its largest value."""
    device = _gpu(x, "x")
    xr, n = _plain(x, device, "x")
    k = x.shape[1]
    if out is None:
        out = Int8Rows(n, k, device)
    else:
        _need(out.k == k and len(out) == n and out.codes.device == device, f"out: {n} rows of {k} values on {device} are wanted")
    if n:
        _call(L.load().velox_hip_int8_quantize, device.index, xr, n, k, out.desc)
    return out


def product_workspace(w: Int8Matrix, rows: int) -> torch.Tensor | None:
    """What product() needs for up to `rows` rows that come in another type than 8 bits (None: nothing)."""
    n = C.c_uint64()
    _numbers("rows", rows)
    L.check(w.lib.velox_hip_int8_product_bytes(w._ref, rows, C.byref(n)), "int8_product_bytes")
    return _memory(n.value, w.device)


def product(x: torch.Tensor | Int8Rows, w: Int8Matrix, *, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
            dtype: torch.dtype | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """x w^T (+ bias float32 [n]) (+ residual, which may be out), or silu(gate) * up of a paired w. x: rows [row][k], put
    into 8 bits on the way (workspace: product_workspace, None: made here), or Int8Rows. out: a new tensor of `dtype`
    (default: x's type, float32 for Int8Rows), or the one given."""
    device = w.device
    if w.count != 1:
        raise ValueError("w: one matrix is wanted (experts.ffn takes several)")
    if isinstance(x, Int8Rows):
        _need(x.k == w.k and x.codes.device == device, "x: rows of the matrix's k values on its device are wanted")
        n, xr, xq, space, size, kind = len(x), None, x.desc, None, 0, torch.float32
    else:
        xr, n = _plain(x, device, "x", w.k)
        xq, kind = None, x.dtype
        if workspace is None and n:
            workspace = product_workspace(w, n)
        space, size = _space(workspace, device)
    if out is None:
        kind = dtype or kind
        if kind not in _DTYPES:
            raise ValueError("dtype: float32, float16 or bfloat16 is wanted")
        cols = w.outputs
        out = torch.empty((n, cols), dtype=kind, device=device)
        o = L.Rows(out.data_ptr(), _DTYPES[kind], 1, cols, 0)
    else:
        _need(dtype is None or out.dtype == dtype, "out: another type than dtype")
        o = _result(out, device, w.outputs, n)
    if w.paired and (bias is not None or residual is not None):
        raise ValueError("a paired product takes no bias and no residual")
    at = _floats(bias, (w.n,), device, "bias") if bias is not None else None
    res, mode = None, L.GEMV_SWIGLU if w.paired else L.GEMV_STORE
    if residual is not None:
        res, _ = _plain(residual, device, "residual", w.n, n)
        mode = L.GEMV_RESIDUAL
    if n:
        _call(w.lib.velox_hip_int8_product, w._index, w._ref, xr, xq, n, at, res, o, mode, space, size)
    return out
