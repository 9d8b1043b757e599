"""8-bit integer dense operators: codes in -127 .. 127, one f32 scale per row (token, or output channel).

  quantize     activations or weights (f32, bf16, f16) -> Int8Tensor
  from_codes   stored codes and scales -> Int8Tensor
  linear       x W^T on the tensor cores' 8-bit integer rate, x quantised on the way or already

What does not bear 4 bits (``deepseeker.mx4``) is served in 8.  Serving only:
the results have no derivatives, and an input that asks for one (a gradient, or
a forward-mode tangent) is refused.
"""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from ._dev import has_tangent, on_device, raw_stream, rows_of, stream_handle

_DTYPES = {torch.float32: _abi.DS_F32, torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}
_MOST = 1 << 17   # values of a row: below, so that sums of products stay inside 32 bits


def _up(n: int, a: int) -> int:
    return (n + a - 1) // a * a


def _workspace_bytes(rows: int, cols: int) -> int:
    """Codes and scales of a quantised matrix, each on 256 bytes."""
    return _up(rows * _up(cols, 16), 256) + _up(4 * rows, 256)


def _x_bytes(rows: int, cols: int) -> int:
    """Workspace for x given as values: a single row the product quantises itself."""
    return _workspace_bytes(rows, cols) if rows > 1 else 0


class Int8Tensor:
    """A quantised matrix: ``codes`` i8 and ``scales`` f32 of its rows (value =
    code * scale; scale NaN for a row that held a NaN or an infinity); ``shape``:
    the shape it stands for, leading dimensions included."""

    __slots__ = ("rows", "cols", "pitch", "shape", "device", "_hold", "_pc", "_ps", "_codes", "_scales", "_c")

    def __init__(self, rows, shape, pitch, device, hold, codes, scales, views=(None, None)):
        """``hold``: what owns the memory at the addresses ``codes`` and ``scales``."""
        self.rows, self.cols, self.pitch, self.shape, self.device = rows, shape[-1], pitch, shape, device
        self._hold, self._pc, self._ps = hold, codes, scales
        self._codes, self._scales = views
        self._c = None

    @property
    def codes(self) -> torch.Tensor:
        """i8, of ``shape``; its rows lie ``pitch`` bytes apart."""
        if self._codes is None:
            at = (self._pc - self._ps) // 4
            rows = self._hold[at:].view(torch.int8).view(self.rows, self.pitch)[:, :self.cols]
            self._codes = rows.unflatten(0, self.shape[:-1]) if len(self.shape) > 1 else rows[0]
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        """f32, of ``shape`` without the last dimension."""
        if self._scales is None:
            scales = self._hold[:self.rows]
            self._scales = scales if len(self.shape) == 2 else scales.view(self.shape[:-1])
        return self._scales

    def _ref(self):
        if self._c is None:
            self._c = _abi.DsInt8(self._pc, self._ps, self.rows, self.cols, self.pitch)
        return ctypes.byref(self._c)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """code * scale as f32, or rounded from there to bf16 or f16."""
        if dtype not in _DTYPES:
            raise ValueError("dtype must be f32, bf16 or f16")
        dev = self.device
        out = torch.empty(self.shape, dtype=dtype, device=dev)
        with on_device(dev):
            _abi.check(_abi.lib().ds_int8_dequantize(self._pc, self.pitch, self._ps, self.rows, self.cols,
                                                     out.data_ptr(), _DTYPES[dtype], raw_stream(dev)),
                       "ds_int8_dequantize")
        return out


def _check_x(x) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a f32, bf16 or f16 CUDA tensor (or an Int8Tensor where one is taken)")
    if x.dim() < 1 or not 1 <= x.shape[-1] < _MOST:
        raise ValueError("x must be [..., cols] with cols in [1, 2^17)")
    _check_no_derivative(x, "x")


def _check_no_derivative(t, name) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"8-bit operators have no backward pass: detach {name} or use torch.no_grad()")
    if has_tangent(t):
        raise ValueError(f"8-bit operators have no forward-mode derivatives: {name} is a dual tensor")


def _matrix(x):
    """x [..., cols] as rows, and their distance in elements."""
    return rows_of(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))


def quantize(x: torch.Tensor) -> Int8Tensor:
    """x [..., cols] -> Int8Tensor.  A row's scale is its largest magnitude times
    1 / 127 (in f32), a code the whole number nearest to the exact quotient of
    value and scale, ties to the even one.  A NaN or an infinity makes its whole row NaN.

    The product is the rule, not the quotient maximum / 127: they differ by a unit
    of the last place in about one row of twenty, and half of the maximum can then get
    another code.  What is quantised elsewhere and has to meet these codes takes the
    product; ``from_codes`` serves codes and scales of either rule as they are."""
    _check_x(x)
    rows, ld = _matrix(x)
    n, cols = rows.shape
    dev, pitch = x.device, _up(cols, 16)
    at = _up(4 * n, 256)
    buf = torch.empty((at + n * pitch) // 4, dtype=torch.float32, device=dev)   # scales, codes
    p = buf.data_ptr()
    with on_device(dev):
        _abi.check(_abi.lib().ds_int8_quantize(rows.data_ptr(), _DTYPES[x.dtype], n, cols, ld, p + at, pitch, p,
                                               raw_stream(dev)), "ds_int8_quantize")
    return Int8Tensor(n, x.shape, pitch, dev, buf, p + at, p)


def from_codes(codes: torch.Tensor, scales: torch.Tensor) -> Int8Tensor:
    """Int8Tensor over stored codes i8 [rows, cols] and scales f32 [rows]: used
    in place where contiguous in rows that are a multiple of 16 bytes apart, on
    16 bytes; copied otherwise.  -128 is a code like any other here."""
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or codes.dtype != torch.int8 or codes.dim() != 2:
        raise ValueError("codes must be a 2-D i8 CUDA tensor")
    rows, cols = codes.shape
    if rows < 1 or not 1 <= cols < _MOST:
        raise ValueError("codes must be [rows, cols] with rows >= 1 and cols in [1, 2^17)")
    if (not isinstance(scales, torch.Tensor) or scales.get_device() != codes.get_device()
            or scales.dtype != torch.float32 or scales.shape != (rows,)):
        raise ValueError("scales must be a f32 tensor [rows] on the codes' device")
    _check_no_derivative(scales, "scales")
    scales, pitch = scales.contiguous(), codes.stride(0)
    if (cols > 1 and codes.stride(1) != 1) or codes.data_ptr() % 16 or pitch % 16 or pitch < cols:
        pitch = _up(cols, 16)
        held = torch.empty((rows, pitch), dtype=torch.int8, device=codes.device)[:, :cols]
        codes = held.copy_(codes)
    return Int8Tensor(rows, torch.Size((rows, cols)), pitch, codes.device, (codes, scales), codes.data_ptr(),
                      scales.data_ptr(), (codes, scales))


def linear(x, w: Int8Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] (a tensor, quantised on the way, or an Int8Tensor) times W^T,
    W [N, K] -> [..., N] in out_dtype (default: x's type; bf16 for an
    Int8Tensor).  The sums of products of codes are exact; their conversion to
    f32, both scales and the final rounding are one rounding each."""
    if not isinstance(w, Int8Tensor) or len(w.shape) != 2:
        raise ValueError("w must be a 2-D Int8Tensor")
    if w.device != getattr(x, "device", None):
        raise ValueError("w must be on x's device")
    dev, ws, n = w.device, None, 0
    if isinstance(x, Int8Tensor):
        px, ps, dt, rows, ld, kind = x._pc, x._ps, _abi.DS_I8, x.rows, x.pitch, torch.bfloat16
    else:
        _check_x(x)
        m, ld = _matrix(x)
        px, ps, dt, rows, kind = m.data_ptr(), None, _DTYPES[x.dtype], m.shape[0], x.dtype
    if x.shape[-1] != w.cols:
        raise ValueError(f"x must be [..., {w.cols}]")
    if out_dtype is None:
        out_dtype = kind
    if out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be f32, bf16 or f16")
    if ps is None:
        n = _x_bytes(rows, w.cols)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    out = torch.empty((*x.shape[:-1], w.rows), dtype=out_dtype, device=dev)
    if not w.rows:
        return out
    with on_device(dev):
        _abi.check(_abi.lib().ds_int8_linear(px, ps, dt, rows, ld, w._ref(), out.data_ptr(), _DTYPES[out_dtype],
                                             None if ws is None else ws.data_ptr(), n, raw_stream(dev)),
                   "ds_int8_linear")
    return out


def status(device: torch.device | None = None) -> int:
    """Error bits of this module's calls on `device` since the last query (2: a
    bounded device wait gave up; outputs are then undefined).  Waits for the stream."""
    err = torch.zeros(1, dtype=torch.int32)
    with torch.cuda.device(device):
        _abi.check(_abi.lib().ds_int8_status(err.data_ptr(), stream_handle(device)), "ds_int8_status")
        torch.cuda.current_stream(device).synchronize()
    return int(err[0])
