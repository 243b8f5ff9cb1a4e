"""Microscaled 4-bit rows (MXFP4) over the C ABI: quantise, dequantise, products and sparse convolutions.

A row of channels is held in blocks of 32: one power of two per block and 32 four-bit values (see "microscaled 4-bit
rows" in scn_c_api.h for the format).  PyTorch only owns memory and streams; there is no CPU path.

  quantize_rows     fp16 / fp32 / int8 rows -> MxRows
  dequantize_rows   MxRows -> fp16 / fp32 rows
  product           rows x weight rows^T, with bias, ReLU and residual
  Conv, Rulebook    sparse convolution on MxRows (scn_conv_* with SCN_PRECISION_MXFP4)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch

from . import capi
from .scn import _stream_ptr

_DTYPE = {torch.float16: capi.DTYPE_FP16, torch.float32: capi.DTYPE_FP32, torch.int8: capi.DTYPE_INT8}


def row_bytes(channels: int) -> int:
    """Bytes of a row in the one-buffer form: 16 per block of 32 channels, then the scales, in whole 16-byte chunks."""
    blocks = (channels + 31) // 32
    return (16 * blocks + (blocks + 3) // 4 * 4 + 15) // 16 * 16


class MxRows:
    """codes [n, >= 16 * blocks] and scales [n, >= round_up(blocks, 4)] (uint8, unit stride inside a row) of n rows."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, channels: int):
        for t, need in ((codes, 16 * ((channels + 31) // 32)), (scales, ((channels + 31) // 32 + 3) // 4 * 4)):
            if t.dtype != torch.uint8 or t.dim() != 2 or not t.is_cuda:
                raise ValueError("codes and scales must be 2-D uint8 device tensors")
            if t.shape[1] < need or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError(f"rows of {channels} channels need {need} contiguous bytes")
        if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise ValueError("codes and scales must have the same rows on the same device")
        self.codes, self.scales, self.channels = codes, scales, int(channels)

    @property
    def num_rows(self) -> int:
        return int(self.codes.shape[0])

    @property
    def device(self):
        return self.codes.device

    @classmethod
    def empty(cls, n: int, channels: int, device="cuda") -> "MxRows":
        """Uninitialised rows in the one-buffer form."""
        if channels < 1 or n < 0:
            raise ValueError("rows need at least one channel")
        blocks = (channels + 31) // 32
        buf = torch.empty((n, row_bytes(channels)), dtype=torch.uint8, device=device)
        return cls(buf[:, :16 * blocks], buf[:, 16 * blocks:16 * blocks + (blocks + 3) // 4 * 4], channels)


def _check_rows(x: torch.Tensor, dtypes, what: str) -> None:
    if not isinstance(x, torch.Tensor) or x.dtype not in dtypes or x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{what} must be a 2-D device tensor of {' or '.join(str(d) for d in dtypes)}")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError(f"{what} must have unit stride inside a row")
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        raise ValueError(f"{what} must not have overlapping rows")


def _ld(x: torch.Tensor) -> int:
    return int(x.stride(0)) if x.shape[0] > 1 else max(int(x.stride(0)), int(x.shape[1]))


def _count_ptr(num: Optional[torch.Tensor], device) -> Optional[int]:
    if num is None:
        return None
    if num.dtype not in (torch.int32, torch.uint32) or num.numel() != 1 or num.device != device:
        raise ValueError("num must be one int32 / uint32 on the rows' device")
    return num.data_ptr()


def _same_device(device, *others) -> None:
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")


def quantize_rows(x: torch.Tensor, relu: bool = False, dynamic_range: float = 0.0, num: Optional[torch.Tensor] = None,
                  out: Optional[MxRows] = None, stream=None) -> MxRows:
    """x: fp16, fp32 or int8 (value = q * dynamic_range / 127) rows [n, c]; num: device-side row count (rows beyond it are
    left as they were)."""
    _check_rows(x, (torch.float16, torch.float32, torch.int8), "x")
    n, c = x.shape
    if out is None:
        out = MxRows.empty(n, c, x.device)
    elif out.num_rows < n or out.channels != c:
        raise ValueError("out does not fit x")
    _same_device(x.device, out)
    with torch.cuda.device(x.device):
        capi.check(capi.lib().scn_mx_quantize_rows(
            x.data_ptr(), _DTYPE[x.dtype], c, _ld(x), float(dynamic_range), int(bool(relu)), out.codes.data_ptr(), _ld(out.codes),
            out.scales.data_ptr(), _ld(out.scales), n, _count_ptr(num, x.device), _stream_ptr(stream)))
    return out


def dequantize_rows(rows: MxRows, dtype: torch.dtype = torch.float16, num: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    n, c = rows.num_rows, rows.channels
    if out is None:
        out = torch.empty((n, c), dtype=dtype, device=rows.device)
    _check_rows(out, (torch.float16, torch.float32), "out")
    if out.shape[0] < n or out.shape[1] != c:
        raise ValueError("out does not fit the rows")
    _same_device(rows.device, out)
    with torch.cuda.device(rows.device):
        capi.check(capi.lib().scn_mx_dequantize_rows(
            rows.codes.data_ptr(), _ld(rows.codes), rows.scales.data_ptr(), _ld(rows.scales), c, out.data_ptr(),
            _DTYPE[out.dtype], _ld(out), n, _count_ptr(num, rows.device), _stream_ptr(stream)))
    return out


def product(a, b: MxRows, bias: Optional[torch.Tensor] = None, relu: bool = False, residual: Optional[torch.Tensor] = None,
            relu_after_add: bool = False, out_dtype: torch.dtype = torch.float16, num: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """relu2(relu(a b^T + bias) + residual): a is MxRows, or fp16 / fp32 rows that are quantised on the way; b the rows of a
    weight matrix.  workspace: uint8 scratch for the quantised rows (a new one is allocated when it is needed and not
    given); calls that may overlap need one each."""
    L = capi.lib()
    io = capi.MxProductIO()
    if isinstance(a, MxRows):
        m, k = a.num_rows, a.channels
        io.a_dev, io.a_dtype, io.a_ld = a.codes.data_ptr(), capi.DTYPE_MXFP4, _ld(a.codes)
        io.a_scales_dev, io.a_scales_ld = a.scales.data_ptr(), _ld(a.scales)
    else:
        _check_rows(a, (torch.float16, torch.float32), "a")
        m, k = a.shape
        io.a_dev, io.a_dtype, io.a_ld = a.data_ptr(), _DTYPE[a.dtype], _ld(a)
    n = b.num_rows
    if b.channels != k:
        raise ValueError(f"rows of {k} channels times weights of {b.channels}")
    device = b.device
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=device)
    _check_rows(out, (torch.float16, torch.float32), "out")
    if out.shape[0] < m or out.shape[1] != n:
        raise ValueError("out does not fit the product")
    if bias is not None and (bias.dtype not in (torch.float16, torch.float32) or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be {n} contiguous fp16 or fp32 values")
    if residual is not None:
        _check_rows(residual, (torch.float16, torch.float32), "residual")
        if residual.shape[0] < m or residual.shape[1] != n:
            raise ValueError("residual does not fit the product")
    _same_device(device, a, out, bias, residual, workspace)
    with torch.cuda.device(device):
        if not isinstance(a, MxRows):
            need = int(L.scn_mx_product_workspace(m, k))
            if need and workspace is None:
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
            if workspace is not None:
                io.workspace_dev, io.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        io.b_codes_dev, io.b_codes_ld = b.codes.data_ptr(), _ld(b.codes)
        io.b_scales_dev, io.b_scales_ld = b.scales.data_ptr(), _ld(b.scales)
        io.m, io.n, io.k = m, n, k
        io.m_dev = _count_ptr(num, device)
        if bias is not None:
            io.bias_dev, io.bias_dtype = bias.data_ptr(), _DTYPE[bias.dtype]
        io.relu, io.relu_after_add = int(bool(relu)), int(bool(relu_after_add))
        if residual is not None:
            io.res_dev, io.res_dtype, io.res_ld = residual.data_ptr(), _DTYPE[residual.dtype], _ld(residual)
        io.out_dev, io.out_dtype, io.out_ld = out.data_ptr(), _DTYPE[out.dtype], _ld(out)
        capi.check(L.scn_mx_product(C.byref(io), _stream_ptr(stream)))
    return out


class Rulebook:
    """scn_rulebook: the neighbour table of a convolution (built once per set of coordinates, shared by its layers)."""

    def __init__(self, max_in: int, max_out: int, kernel_volume: int):
        self._h = capi.lib().scn_rulebook_create(max_in, max_out, kernel_volume)
        if not self._h:
            raise RuntimeError("rulebook creation failed: " + capi.lib().scn_last_error().decode())
        self._keep = None
        self.max_in, self.max_out = int(max_in), int(max_out)
        self.rows_in = self.rows_out = None   # bounds of the last build: rows the convolution may read / write

    def _check(self, indices: torch.Tensor):
        if indices.dtype != torch.int32 or indices.dim() != 2 or indices.shape[1] != 4 or not indices.is_contiguous() or not indices.is_cuda:
            raise ValueError("indices must be a contiguous int32 device tensor [n, 4]")

    def build_subm(self, indices: torch.Tensor, grid: Sequence[int], kernel_size, dilation=(1, 1, 1), num=None, stream=None):
        self._check(indices)
        self._keep = (indices, num)
        capi.check(capi.lib().scn_rulebook_build_subm(
            self._h, indices.data_ptr(), int(indices.shape[0]), _count_ptr(num, indices.device), capi.i3(*grid),
            capi.i3(*kernel_size), capi.i3(*dilation), _stream_ptr(stream)))
        self.rows_in = self.rows_out = min(int(indices.shape[0]), self.max_in)

    def build_sparse(self, indices: torch.Tensor, grid: Sequence[int], kernel_size, stride, padding, dilation=(1, 1, 1),
                     num=None, stream=None):
        self._check(indices)
        self._keep = (indices, num)
        capi.check(capi.lib().scn_rulebook_build_sparse(
            self._h, indices.data_ptr(), int(indices.shape[0]), _count_ptr(num, indices.device), capi.i3(*grid),
            capi.i3(*kernel_size), capi.i3(*stride), capi.i3(*padding), capi.i3(*dilation), _stream_ptr(stream)))
        self.rows_in, self.rows_out = min(int(indices.shape[0]), self.max_in), self.max_out

    def close(self):
        if getattr(self, "_h", None):
            capi.lib().scn_rulebook_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()


class Conv:
    """A sparse convolution on microscaled rows: weight fp16 [Cout, K0, K1, K2, Cin], bias fp16 [Cout] or None (host
    arrays); both are laid out once."""

    def __init__(self, weight: np.ndarray, bias: Optional[np.ndarray] = None):
        w = np.ascontiguousarray(weight, np.float16)
        if w.ndim != 5:
            raise ValueError("weight must be [Cout, K0, K1, K2, Cin]")
        b = None if bias is None else np.ascontiguousarray(bias, np.float16)
        if b is not None and b.shape != (w.shape[0],):
            raise ValueError(f"bias must be {w.shape[0]} values")
        self._h = capi.lib().scn_conv_create(w.ctypes.data_as(C.c_void_p), capi.i5(*w.shape), None,
                                             None if b is None else b.ctypes.data_as(C.c_void_p), capi.PRECISION_MXFP4)
        if not self._h:
            raise RuntimeError("convolution creation failed: " + capi.lib().scn_last_error().decode())
        self.cout, self.cin = int(w.shape[0]), int(w.shape[4])

    def forward(self, x: MxRows, rulebook: Rulebook, max_rows: int, relu: bool = False, residual: Optional[torch.Tensor] = None,
                relu_after_add: bool = False, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """x: MxRows in the one-buffer form (what quantize_rows makes).  Returns fp16 [max_rows, Cout]; rows beyond the
        rulebook's count are left as they were.  residual: fp16 [max_rows, >= Cout rounded up to 16]."""
        blocks = (self.cin + 31) // 32
        if rulebook.rows_in is None:
            raise ValueError("the rulebook has not been built")
        if x.num_rows < rulebook.rows_in or max_rows < rulebook.rows_out:
            raise ValueError(f"the rulebook covers {rulebook.rows_in} input rows and up to {rulebook.rows_out} output rows")
        if x.channels != self.cin:
            raise ValueError(f"input rows have {x.channels} channels, the weight expects {self.cin}")
        if _ld(x.codes) != _ld(x.scales) or x.scales.data_ptr() != x.codes.data_ptr() + 16 * blocks:
            raise ValueError("the convolution reads rows in the one-buffer form (codes, then scales)")
        wide = (self.cout + 15) // 16 * 16
        if out is None:
            out = torch.empty((max_rows, wide), dtype=torch.float16, device=x.device)
        _check_rows(out, (torch.float16,), "out")
        if out.shape[0] < max_rows or out.shape[1] < wide:
            raise ValueError(f"out must hold {max_rows} rows of {wide} channels")
        _same_device(x.device, out, residual)
        io = capi.ConvIO()
        io.x_dev, io.x_ld = x.codes.data_ptr(), _ld(x.codes)
        io.relu, io.out_dtype, io.out_dev, io.out_ld = int(bool(relu)), capi.DTYPE_FP16, out.data_ptr(), _ld(out)
        if residual is not None:
            _check_rows(residual, (torch.float16,), "residual")
            if residual.shape[0] < max_rows or residual.shape[1] < wide:
                raise ValueError(f"residual must hold {max_rows} rows of {wide} channels")
            io.res_dev, io.res_dtype, io.res_ld, io.mid_dtype = residual.data_ptr(), capi.DTYPE_FP16, _ld(residual), capi.DTYPE_FP16
            io.relu_after_add = int(bool(relu_after_add))
        with torch.cuda.device(x.device):
            capi.check(capi.lib().scn_conv_forward(self._h, rulebook._h, C.byref(io), _stream_ptr(stream)))
        return out[:max_rows, :self.cout]

    def close(self):
        if getattr(self, "_h", None):
            capi.lib().scn_conv_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()
