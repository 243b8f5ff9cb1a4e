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
import struct
from typing import Optional, Sequence

import numpy as np
import torch

from . import capi
from .scn import _stream_ptr

_DTYPE = {torch.float16: capi.DTYPE_FP16, torch.float32: capi.DTYPE_FP32, torch.int8: capi.DTYPE_INT8}
_FLOATS = (torch.float16, torch.float32)
_ROWS = (torch.float16, torch.float32, torch.int8)
_COUNT = 1 << 32        # rows and strides are 32-bit numbers in the C ABI
_L = None


def _lib():
    global _L
    if _L is None:
        _L = capi.lib()
    return _L


# (a call here takes a few microseconds: a device context is entered only where needed, and the cheaper of equal calls is taken)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_devices = {}


def _device(index: int) -> torch.device:
    device = _devices.get(index)
    if device is None:
        device = _devices[index] = torch.device("cuda", index)
    return device


def _new(n: int, c: int, dtype: torch.dtype, index: int) -> torch.Tensor:
    return torch.empty_strided((n, c), (c, 1), dtype=dtype, device=_device(index))      # (0.5 us less than torch.empty)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # (a tenth of the time of building a Stream object)


def _stream(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _using(stream, index: int):
    """A context in which `stream` (a torch stream or a hipStream_t) is the current one: what a call allocates then belongs
    to the stream that its kernels run on."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=index) if int(stream) else torch.cuda.default_stream(index)
    elif stream.device_index != index:
        raise ValueError(f"a stream of cuda:{stream.device_index} for rows on cuda:{index}")
    return torch.cuda.stream(stream)


def row_bytes(channels: int) -> int:
    """Bytes of a row in the one-buffer form: 16 per block of 32 channels, then the scales, in whole 16-byte chunks."""
    blocks = (channels + 31) // 32
    return (16 * blocks + (blocks + 3) // 4 * 4 + 15) // 16 * 16


class MxRows:
    """codes [n, >= 16 * blocks] and scales [n, >= round_up(blocks, 4)] (uint8, unit stride inside a row) of n rows."""

    __slots__ = ("_codes", "_scales", "_buffer", "channels", "num_rows", "index", "codes_ptr", "codes_ld", "scales_ptr", "scales_ld")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, channels: int):
        if not 1 <= channels <= 1 << 30:
            raise ValueError("rows need 1 to 2^30 channels")
        blocks = (channels + 31) // 32
        for t, need in ((codes, 16 * blocks), (scales, (blocks + 3) // 4 * 4)):
            if t.dtype != torch.uint8 or t.dim() != 2 or not t.is_cuda:
                raise ValueError("codes and scales must be 2-D uint8 device tensors")
            if t.shape[1] < need or t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < need):
                raise ValueError(f"rows of {channels} channels need {need} contiguous bytes of their own")
        if codes.shape[0] >= _COUNT or max(_ld(codes), _ld(scales)) >= _COUNT:
            raise ValueError("rows must be fewer than 2^32, less than 2^32 bytes apart")
        if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise ValueError("codes and scales must have the same rows on the same device")
        self._codes, self._scales, self._buffer = codes, scales, None
        self.channels, self.num_rows, self.index = int(channels), int(codes.shape[0]), codes.get_device()
        self.codes_ptr, self.codes_ld = codes.data_ptr(), _ld(codes)
        self.scales_ptr, self.scales_ld = scales.data_ptr(), _ld(scales)

    @classmethod
    def empty(cls, n: int, channels: int, device="cuda") -> "MxRows":
        """Uninitialised rows in the one-buffer form."""
        if not 1 <= channels <= 1 << 30 or not 0 <= n < _COUNT:
            raise ValueError("rows need 1 to 2^30 channels, and are fewer than 2^32")
        self = cls.__new__(cls)
        blocks = (channels + 31) // 32
        size = (16 * blocks + (blocks + 3) // 4 * 4 + 15) // 16 * 16      # row_bytes(channels)
        buf = torch.empty(n * size, dtype=torch.uint8, device=device)     # (flat: made in two thirds of the time)
        self._codes = self._scales = None
        self._buffer, self.channels, self.num_rows, self.index = buf, channels, n, buf.get_device()
        if self.index < 0:
            raise ValueError(f"rows live on a GPU, not on {buf.device}")
        self.codes_ptr = ptr = buf.data_ptr()
        self.scales_ptr = ptr + 16 * blocks
        self.codes_ld = self.scales_ld = size
        return self

    def _columns(self, first: int, last: int) -> torch.Tensor:
        return self._buffer.view(self.num_rows, self.codes_ld)[:, first:last]

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._columns(0, 16 * ((self.channels + 31) // 32))
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            blocks = (self.channels + 31) // 32
            self._scales = self._columns(16 * blocks, 16 * blocks + (blocks + 3) // 4 * 4)
        return self._scales

    @property
    def device(self) -> torch.device:
        return _device(self.index)


def _check_rows(x: torch.Tensor, dtypes, what: str) -> int:
    """Refuses what is not rows of a device tensor; returns the row stride in elements."""
    if not isinstance(x, torch.Tensor) or x.dtype not in dtypes or x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{what} must be a 2-D device tensor of {' or '.join(str(d) for d in dtypes)}")
    n, c = x.shape
    ld, step = x.stride()
    if c > 1 and step != 1:
        raise ValueError(f"{what} must have unit stride inside a row")
    if n > 1 and ld < c:
        raise ValueError(f"{what} must not have overlapping rows")
    if n <= 1:
        ld = max(ld, c)
    if n >= _COUNT or ld >= _COUNT:
        raise ValueError(f"{what} must have fewer than 2^32 rows, less than 2^32 elements apart")
    return ld


def _ld(x: torch.Tensor) -> int:
    return int(x.stride(0)) if x.shape[0] > 1 else max(int(x.stride(0)), int(x.shape[1]))


def _count_ptr(num: Optional[torch.Tensor], index: int) -> Optional[int]:
    if num is None:
        return None
    if num.dtype not in (torch.int32, torch.uint32) or num.numel() != 1 or not num.is_cuda or num.get_device() != index:
        raise ValueError("num must be one int32 / uint32 on the rows' device")
    return num.data_ptr()


def _same_device(index: int, *others) -> None:
    for t in others:
        if t is not None and (t.index if isinstance(t, MxRows) else t.get_device()) != index:
            raise ValueError(f"tensors on different devices (rows on cuda:{index})")


def _overlap(a, b) -> bool:
    """Whether two runs of rows (address, rows, bytes of a row, stride in bytes) share a byte; rows of one stride may lie side
    by side.  (The C library checks its row operators like this; of a convolution it knows only bounds of the row counts.)"""
    (pa, na, wa, la), (pb, nb, wb, lb) = a, b
    if pa + (na - 1) * la + wa <= pb or pb + (nb - 1) * lb + wb <= pa or not (na and nb):
        return False
    if na > 1 and nb > 1 and la != lb or na == nb == 1:
        return True
    ld = la if na > 1 else lb
    d = (pb - pa) % ld
    return d < wa or d + wb > ld


def quantize_rows(x: torch.Tensor, relu: bool = False, dynamic_range: float = 0.0, num: Optional[torch.Tensor] = None,
                  out: Optional[MxRows] = None, stream=None) -> MxRows:
    """x: fp16, fp32 or int8 (value = q * dynamic_range / 127) rows [n, c]; num: device-side row count (rows beyond it are
    left as they were)."""
    ld = _check_rows(x, _ROWS, "x")
    n, c = x.shape
    index = x.get_device()
    if stream is not None:
        with _using(stream, index):
            return quantize_rows(x, relu, dynamic_range, num, out)
    if index != _current_device():
        with torch.cuda.device(index):
            return quantize_rows(x, relu, dynamic_range, num, out)
    if out is None:
        out = MxRows.empty(n, c, x.device)
    elif out.num_rows < n or out.channels != c or out.index != index:
        raise ValueError("out does not fit x")
    rc = _lib().scn_mx_quantize_rows(x.data_ptr(), _DTYPE[x.dtype], c, ld, dynamic_range, relu, out.codes_ptr, out.codes_ld,
                                     out.scales_ptr, out.scales_ld, n, None if num is None else _count_ptr(num, index),
                                     _stream(index))
    if rc:
        capi.check(rc)
    return out


def dequantize_rows(rows: MxRows, dtype: torch.dtype = torch.float16, num: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    n, c, index = rows.num_rows, rows.channels, rows.index
    if stream is not None:
        with _using(stream, index):
            return dequantize_rows(rows, dtype, num, out)
    if index != _current_device():
        with torch.cuda.device(index):
            return dequantize_rows(rows, dtype, num, out)
    if out is None:
        if dtype not in _FLOATS:
            raise ValueError("dtype must be float16 or float32")
        out, ld = _new(n, c, dtype, index), c
    else:
        ld = _check_rows(out, _FLOATS, "out")
        if out.shape[0] < n or out.shape[1] != c:
            raise ValueError("out does not fit the rows")
        _same_device(index, out)
    rc = _lib().scn_mx_dequantize_rows(rows.codes_ptr, rows.codes_ld, rows.scales_ptr, rows.scales_ld, c, out.data_ptr(),
                                       _DTYPE[out.dtype], ld, n, None if num is None else _count_ptr(num, index),
                                       _stream(index))
    if rc:
        capi.check(rc)
    return out


# scn_mx_product_io as native bytes (same layout as capi.MxProductIO, filled in one go)
_PRODUCT_IO = struct.Struct("PiIPIPIPIIIIPPiiPiIiPiIPN")
assert _PRODUCT_IO.size == C.sizeof(capi.MxProductIO)


def product(a, b: MxRows, bias: Optional[torch.Tensor] = None, relu: bool = False, residual: Optional[torch.Tensor] = None,
            relu_after_add: bool = False, out_dtype: torch.dtype = torch.float16, num: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """relu2(relu(a b^T + bias) + residual): a is MxRows, or fp16 / fp32 rows that are quantised on the way; b the rows of a
    weight matrix.  A NaN stays one through both ReLUs (quantize_rows and the convolutions make it 0).  workspace: uint8 scratch for the quantised rows (a new one is allocated when it is needed and not
    given); calls that may overlap need one each."""
    L = _lib()
    n, index = b.num_rows, b.index
    if stream is not None:
        with _using(stream, index):
            return product(a, b, bias, relu, residual, relu_after_add, out_dtype, num, out, workspace)
    if index != _current_device():
        with torch.cuda.device(index):
            return product(a, b, bias, relu, residual, relu_after_add, out_dtype, num, out, workspace)
    ws_ptr = ws_bytes = 0
    if isinstance(a, MxRows):
        m, k, a_index = a.num_rows, a.channels, a.index
        a_ptr, a_dtype, a_ld, as_ptr, as_ld = a.codes_ptr, capi.DTYPE_MXFP4, a.codes_ld, a.scales_ptr, a.scales_ld
    else:
        a_ld = _check_rows(a, _FLOATS, "a")
        (m, k), a_index = a.shape, a.get_device()
        a_ptr, a_dtype, as_ptr, as_ld = a.data_ptr(), _DTYPE[a.dtype], 0, 0
        if workspace is None:
            ws_bytes = L.scn_mx_product_workspace(m, n, k)
            if ws_bytes:
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=_device(index))
        if workspace is not None:
            if not workspace.is_contiguous():
                raise ValueError("workspace must be contiguous")
            _same_device(index, workspace)
            ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if a_index != index:
        raise ValueError(f"rows on cuda:{a_index}, weights on cuda:{index}")
    if b.channels != k:
        raise ValueError(f"rows of {k} channels times weights of {b.channels}")
    if out is None:
        if out_dtype not in _FLOATS:
            raise ValueError("out_dtype must be float16 or float32")
        out, out_ld = _new(m, n, out_dtype, index), n
    else:
        out_ld = _check_rows(out, _FLOATS, "out")
        if out.shape[0] < m or out.shape[1] != n:
            raise ValueError("out does not fit the product")
        _same_device(index, out)
    bias_ptr = bias_dtype = res_ptr = res_dtype = res_ld = 0
    if bias is not None:
        if bias.dtype not in _FLOATS or bias.shape != (n,) or not bias.is_contiguous():
            raise ValueError(f"bias must be {n} contiguous fp16 or fp32 values")
        _same_device(index, bias)
        bias_ptr, bias_dtype = bias.data_ptr(), _DTYPE[bias.dtype]
    if residual is not None:
        res_ld = _check_rows(residual, _FLOATS, "residual")
        if residual.shape[0] < m or residual.shape[1] != n:
            raise ValueError("residual does not fit the product")
        _same_device(index, residual)
        res_ptr, res_dtype = residual.data_ptr(), _DTYPE[residual.dtype]
    rc = L.scn_mx_product(_PRODUCT_IO.pack(a_ptr, a_dtype, a_ld, as_ptr, as_ld, b.codes_ptr, b.codes_ld, b.scales_ptr, b.scales_ld,
                                           m, n, k, 0 if num is None else _count_ptr(num, index), bias_ptr, bias_dtype, bool(relu), res_ptr,
                                           res_dtype, res_ld, bool(relu_after_add), out.data_ptr(), _DTYPE[out.dtype], out_ld,
                                           ws_ptr, ws_bytes), _stream(index))
    if rc:
        capi.check(rc)
    return out


class Rulebook:
    """scn_rulebook: the neighbour table of a convolution (built once per set of coordinates, shared by its layers).  It
    lives on the device that is current when it is made."""

    def __init__(self, max_in: int, max_out: int, kernel_volume: int):
        self._h = capi.lib().scn_rulebook_create(max_in, max_out, kernel_volume)
        if not self._h:
            raise RuntimeError("rulebook creation failed: " + capi.lib().scn_last_error().decode())
        self._keep = None
        self.index = torch.cuda.current_device()
        self.max_in, self.max_out = int(max_in), int(max_out)
        self.rows_in = self.rows_out = None   # bounds of the last build: rows the convolution may read / write

    def _check(self, indices: torch.Tensor, stream):
        there = getattr(stream, "device_index", self.index)
        if there != self.index:
            raise ValueError(f"a stream of cuda:{there} for a rulebook on cuda:{self.index}")
        if indices.dtype != torch.int32 or indices.dim() != 2 or indices.shape[1] != 4 or not indices.is_contiguous() or not indices.is_cuda:
            raise ValueError("indices must be a contiguous int32 device tensor [n, 4]")
        if not indices.get_device() == self.index == _current_device():
            raise ValueError(f"the rulebook lives on cuda:{self.index}: indices and the current device must be that one")

    def build_subm(self, indices: torch.Tensor, grid: Sequence[int], kernel_size, dilation=(1, 1, 1), num=None, stream=None):
        self._check(indices, stream)
        self.rows_in = self.rows_out = None     # (a build that fails leaves no table that may be read)
        self._keep = (indices, num)
        capi.check(capi.lib().scn_rulebook_build_subm(
            self._h, indices.data_ptr(), int(indices.shape[0]), _count_ptr(num, indices.get_device()), capi.i3(*grid),
            capi.i3(*kernel_size), capi.i3(*dilation), _stream_ptr(stream)))
        self.rows_in = self.rows_out = min(int(indices.shape[0]), self.max_in)

    def build_sparse(self, indices: torch.Tensor, grid: Sequence[int], kernel_size, stride, padding, dilation=(1, 1, 1),
                     num=None, stream=None):
        self._check(indices, stream)
        self.rows_in = self.rows_out = None     # (a build that fails leaves no table that may be read)
        self._keep = (indices, num)
        capi.check(capi.lib().scn_rulebook_build_sparse(
            self._h, indices.data_ptr(), int(indices.shape[0]), _count_ptr(num, indices.get_device()), capi.i3(*grid),
            capi.i3(*kernel_size), capi.i3(*stride), capi.i3(*padding), capi.i3(*dilation), _stream_ptr(stream)))
        self.rows_in, self.rows_out = min(int(indices.shape[0]), self.max_in), self.max_out

    def close(self):
        if getattr(self, "_h", None):
            capi.lib().scn_rulebook_destroy(self._h)
            self._h = None

    def __del__(self):
        if capi is not None:      # (None while the interpreter ends)
            self.close()


class Conv:
    """A sparse convolution on microscaled rows: weight fp16 [Cout, K0, K1, K2, Cin], bias fp16 [Cout] or None (host
    arrays); both are laid out once, on the device that is current then."""

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
        self.cout, self.cin, self.index = int(w.shape[0]), int(w.shape[4]), torch.cuda.current_device()

    def forward(self, x: MxRows, rulebook: Rulebook, max_rows: int, relu: bool = False, residual: Optional[torch.Tensor] = None,
                relu_after_add: bool = False, out=None, stream=None):
        """x: MxRows in the one-buffer form (what quantize_rows makes).  Returns fp16 [max_rows, Cout]; rows beyond the
        rulebook's count are left as they were.  residual: fp16 [max_rows, >= Cout rounded up to 16].  out: fp16 rows of at
        least Cout rounded up to 16 channels, or MxRows in the one-buffer form, which get the rows that quantize_rows would
        make of the fp16 result (layers of at most 128 input channels)."""
        blocks = (self.cin + 31) // 32
        if rulebook.rows_in is None:
            raise ValueError("the rulebook has not been built")
        if x.num_rows < rulebook.rows_in or max_rows < rulebook.rows_out:
            raise ValueError(f"the rulebook covers {rulebook.rows_in} input rows and up to {rulebook.rows_out} output rows")
        if not x.index == rulebook.index == self.index:
            raise ValueError(f"rows on cuda:{x.index}, rulebook on cuda:{rulebook.index}, weights on cuda:{self.index}")
        if x.channels != self.cin:
            raise ValueError(f"input rows have {x.channels} channels, the weight expects {self.cin}")
        to_mx = isinstance(out, MxRows)
        for r, b in ((x, blocks),) + (((out, (self.cout + 31) // 32),) if to_mx else ()):
            if r.codes_ld != r.scales_ld or r.scales_ptr != r.codes_ptr + 16 * b:
                raise ValueError("the convolution reads and writes rows in the one-buffer form (codes, then scales)")
        wide = (self.cout + 15) // 16 * 16
        if stream is not None:
            with _using(stream, x.index):
                return self.forward(x, rulebook, max_rows, relu, residual, relu_after_add, out)
        if x.index != _current_device():
            with torch.cuda.device(x.index):
                return self.forward(x, rulebook, max_rows, relu, residual, relu_after_add, out)
        if out is None:
            out, out_ld = _new(max_rows, wide, torch.float16, x.index), wide
        elif to_mx:
            out_ld = out.codes_ld
            if out.num_rows < max_rows or out.channels != self.cout or out.index != x.index:
                raise ValueError(f"out must hold {max_rows} rows of {self.cout} channels on cuda:{x.index}")
        else:
            out_ld = _check_rows(out, (torch.float16,), "out")
            if out.shape[0] < max_rows or out.shape[1] < wide:
                raise ValueError(f"out must hold {max_rows} rows of {wide} channels")
            _same_device(x.index, out)
        n_out = rulebook.rows_out
        rows_out = (out.codes_ptr, n_out, row_bytes(self.cout), out_ld) if to_mx else (out.data_ptr(), n_out, 2 * wide, 2 * out_ld)
        if _overlap((x.codes_ptr, rulebook.rows_in, row_bytes(self.cin), x.codes_ld), rows_out):
            raise RuntimeError("out must not overlap the input rows")
        io = capi.ConvIO()
        io.x_dev, io.x_ld = x.codes_ptr, x.codes_ld
        io.relu, io.out_ld = int(bool(relu)), out_ld
        io.out_dtype, io.out_dev = (capi.DTYPE_MXFP4, out.codes_ptr) if to_mx else (capi.DTYPE_FP16, out.data_ptr())
        if residual is not None:
            io.res_ld = _check_rows(residual, (torch.float16,), "residual")
            if residual.shape[0] < max_rows or residual.shape[1] < wide:
                raise ValueError(f"residual must hold {max_rows} rows of {wide} channels")
            _same_device(x.index, residual)
            res = (residual.data_ptr(), n_out, 2 * wide, 2 * io.res_ld)
            if _overlap(rows_out, res) and (to_mx or res[0] != rows_out[0] or n_out > 1 and res[3] != rows_out[3]):
                raise RuntimeError("out must be the residual, of the same stride, or not overlap it")
            io.res_dev, io.res_dtype, io.mid_dtype = residual.data_ptr(), capi.DTYPE_FP16, capi.DTYPE_FP16
            io.relu_after_add = int(bool(relu_after_add))
        capi.check(_lib().scn_conv_forward(self._h, rulebook._h, C.byref(io), _stream(x.index)))
        if to_mx or out.shape == (max_rows, self.cout):
            return out
        return out[:max_rows, :self.cout]

    def close(self):
        if getattr(self, "_h", None):
            capi.lib().scn_conv_destroy(self._h)
            self._h = None

    def __del__(self):
        if capi is not None:      # (None while the interpreter ends)
            self.close()
