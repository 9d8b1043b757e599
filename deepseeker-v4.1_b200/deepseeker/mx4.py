"""Microscaled 4-bit dense operators: e2m1 codes, one ue8m0 scale per 32 values of a row.

  quantize     activations (f32, bf16, f16) -> MX4Tensor
  from_packed  stored codes and scales (the FP4 bank layout, one expert's matrix) -> MX4Tensor
  linear       x W^T on the tensor cores' 4-bit rate, x quantised on the way or already
  gated_ffn    the gated block (deepseeker.gated) over quantised weights

Serving only: the results have no derivatives, and an input that asks for one
(a gradient, or a forward-mode tangent) is refused.
"""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from ._dev import LEAST_LIMIT, has_tangent, new_like, on_device, raw_stream, rows_of, stream_handle

BLOCK = 32
_DTYPES = {torch.float32: _abi.DS_F32, torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}


def _blocks(cols: int) -> int:
    return (cols + BLOCK - 1) // BLOCK


def _atoms_bytes(rows: int, cols: int) -> int:
    return (rows + 127) // 128 * ((cols + 127) // 128) * 512


def _workspace_bytes(rows: int, cols: int) -> int:
    """Codes and atoms of a quantised matrix, each on 256 bytes."""
    return (rows * _blocks(cols) * 16 + 255) // 256 * 256 + (_atoms_bytes(rows, cols) + 255) // 256 * 256


def _x_bytes(rows: int, cols: int) -> int:
    """Workspace for x given as values: up to 16 rows the product quantises itself."""
    return _workspace_bytes(rows, cols) if rows > 16 else 0


class MX4Tensor:
    """A quantised matrix: ``packed`` u8 [rows, 16 ceil(cols/32)] (two codes per
    byte, low nibble first), ``scales`` u8 [rows, ceil(cols/32)] (2^(b-127), 255
    = NaN), and the scales as the tensor cores read them; ``shape``: the shape
    it stands for, leading dimensions included."""

    __slots__ = ("rows", "cols", "shape", "device", "_hold", "_packed", "_scales", "_pp", "_ps", "_pa", "_c")

    def __init__(self, rows, shape, device, hold, packed, scales, atoms, views=(None, None)):
        """``hold``: what owns the memory at the addresses ``packed``, ``scales`` and ``atoms``."""
        self.rows, self.cols, self.shape, self.device = rows, shape[-1], shape, device
        self._hold, self._pp, self._ps, self._pa = hold, packed, scales, atoms
        self._packed, self._scales = views
        self._c = None

    def _view(self, address: int, cols: int) -> torch.Tensor:
        at = address - self._hold.data_ptr()
        return self._hold[at:at + self.rows * cols].view(self.rows, cols)

    @property
    def packed(self) -> torch.Tensor:
        if self._packed is None:
            self._packed = self._view(self._pp, _blocks(self.cols) * 16)
        return self._packed

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._view(self._ps, _blocks(self.cols))
        return self._scales

    @property
    def atoms(self) -> torch.Tensor:
        """[ceil(rows/128) * ceil(cols/128) * 512] bytes (include/deepseeker_b200.h)."""
        if isinstance(self._hold, tuple):
            return self._hold[2]
        at = self._pa - self._hold.data_ptr()
        return self._hold[at:at + _atoms_bytes(self.rows, self.cols)]

    def _ref(self):
        if self._c is None:
            self._c = _abi.DsMx4(self._pp, self._pa, self.rows, self.cols)
        return ctypes.byref(self._c)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the codes stand for, f32 or bf16 (both exact)."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("dtype must be torch.float32 or torch.bfloat16")
        dev = self.device
        out = torch.empty(self.shape, dtype=dtype, device=dev)
        with on_device(dev):
            _abi.check(_abi.lib().ds_mx4_dequantize(self._pp, self._ps, self.rows, self.cols, out.data_ptr(),
                                                    _DTYPES[dtype], raw_stream(dev)),
                       "ds_mx4_dequantize")
        return out


def _check_x(x) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a f32, bf16 or f16 CUDA tensor (or an MX4Tensor where one is taken)")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [..., cols] with at least one column")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("4-bit operators have no backward pass: detach x or use torch.no_grad()")
    if has_tangent(x):
        raise ValueError("4-bit operators have no forward-mode derivatives: x is a dual tensor")


def _matrix(x):
    """x [..., cols] as rows, and their distance in elements."""
    return rows_of(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))


def quantize(x: torch.Tensor) -> MX4Tensor:
    """x [..., cols] -> MX4Tensor.  A block's scale is the smallest power of two
    that brings its largest magnitude to 6 or less (1 for zeros); values round
    to the nearest code, ties to the even one.  A NaN or an infinity makes its
    whole block NaN."""
    _check_x(x)
    rows, ld = _matrix(x)
    n, cols = rows.shape
    nb, dev = _blocks(cols), x.device
    # one buffer: codes, atoms, scales
    at = (n * nb * 16 + 255) // 256 * 256
    sc = at + _atoms_bytes(n, cols)
    buf = torch.empty(sc + n * nb, dtype=torch.uint8, device=dev)
    p = buf.data_ptr()
    with on_device(dev):
        _abi.check(_abi.lib().ds_mx4_quantize(rows.data_ptr(), _DTYPES[x.dtype], n, cols, ld, p, p + sc, p + at,
                                              raw_stream(dev)), "ds_mx4_quantize")
    return MX4Tensor(n, x.shape, dev, buf, p, p + sc, p + at)


def from_packed(packed: torch.Tensor, scales: torch.Tensor, cols: int | None = None) -> MX4Tensor:
    """MX4Tensor over stored codes u8 [rows, 16 ceil(cols/32)] and scales u8
    [rows, ceil(cols/32)] (used in place where contiguous; the scale atoms are
    built once here, so scales that change later need a new MX4Tensor).
    ``cols`` defaults to 32 per scale; the codes behind an uneven end have to
    be 0, as ``quantize`` leaves them: products add them up."""
    for name, t in (("packed", packed), ("scales", scales)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8 or t.dim() != 2:
            raise ValueError(f"{name} must be a 2-D u8 CUDA tensor")
    rows, nb = scales.shape
    cols = nb * BLOCK if cols is None else cols
    if rows < 1 or cols < 1 or _blocks(cols) != nb or packed.shape != (rows, nb * 16) or packed.device != scales.device:
        raise ValueError("packed [rows, 16 ceil(cols/32)] and scales [rows, ceil(cols/32)] expected, on one device")
    packed, scales, dev = packed.contiguous(), scales.contiguous(), packed.device
    if packed.data_ptr() % 16:
        packed = packed.clone()
    atoms = torch.empty(_atoms_bytes(rows, cols), dtype=torch.uint8, device=dev)
    with on_device(dev):
        _abi.check(_abi.lib().ds_mx4_scale_atoms(scales.data_ptr(), rows, cols, atoms.data_ptr(), raw_stream(dev)),
                   "ds_mx4_scale_atoms")
    return MX4Tensor(rows, torch.Size((rows, cols)), dev, (packed, scales, atoms), packed.data_ptr(), scales.data_ptr(),
                     atoms.data_ptr(), (packed, scales))


def _input(x, cols: int, out_dtype):
    """(what keeps it alive, pointer, atoms' pointer, type, rows, row stride, result type) of x, quantised or not."""
    if isinstance(x, MX4Tensor):
        got, dtype = (x, x._pp, x._pa, _abi.DS_U8, x.rows, 0), torch.bfloat16
    else:
        _check_x(x)
        rows, ld = _matrix(x)
        got, dtype = (rows, rows.data_ptr(), None, _DTYPES[x.dtype], rows.shape[0], ld), x.dtype
    if x.shape[-1] != cols:
        raise ValueError(f"x must be [..., {cols}]")
    if out_dtype is None:
        out_dtype = dtype
    if out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be f32, bf16 or f16")
    return *got, out_dtype


def _weight(w, name: str, x) -> None:
    if not isinstance(w, MX4Tensor) or len(w.shape) != 2:
        raise ValueError(f"{name} must be a 2-D MX4Tensor")
    if w.device != getattr(x, "device", None):
        raise ValueError(f"{name} must be on x's device")


def linear(x, w: MX4Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] (a tensor, quantised on the way, or an MX4Tensor) times W^T,
    W [N, K] -> [..., N] in out_dtype (default: x's type; bf16 for an
    MX4Tensor).  Exact up to the f32 accumulation and the final rounding."""
    _weight(w, "w", x)
    hold, px, pa, dt, rows, ld, out_dtype = _input(x, w.cols, out_dtype)
    dev = w.device
    out = torch.empty((*x.shape[:-1], w.rows), dtype=out_dtype, device=dev)
    n = 0 if dt == _abi.DS_U8 else _x_bytes(rows, w.cols)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    with on_device(dev):
        _abi.check(_abi.lib().ds_mx4_linear(px, pa, dt, rows, ld, w._ref(), out.data_ptr(), _DTYPES[out_dtype],
                                            ws.data_ptr() if n else None, n, raw_stream(dev)), "ds_mx4_linear")
    return out


def gated_ffn(x, w1: MX4Tensor, w3: MX4Tensor, w2: MX4Tensor, limit: float | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """(silu(min(x W1^T, L)) * clip(x W3^T, -L, L)) W2^T with x and the product
    of the gate quantised; w1 and w3 [I, H], w2 [H, I].  Clamps as in
    ``deepseeker.gated.gated_ffn``."""
    for name, w in (("w1", w1), ("w3", w3), ("w2", w2)):
        _weight(w, name, x)
    hidden, inter = w1.cols, w1.rows
    if w3.shape != w1.shape or w2.shape != (hidden, inter):
        raise ValueError("w1 [I, H], w3 [I, H], w2 [H, I] expected")
    if limit is not None and not limit > LEAST_LIMIT:
        raise ValueError("limit must be positive in f32, or None for no clamps")
    hold, px, pa, dt, rows, ld, out_dtype = _input(x, hidden, out_dtype)
    dev = w1.device
    same = dt == _DTYPES[out_dtype]   # x is a tensor of the result's type and shape
    out = new_like(x) if same else torch.empty(x.shape, dtype=out_dtype, device=dev)
    n = _workspace_bytes(rows, inter) + (0 if dt == _abi.DS_U8 else _x_bytes(rows, hidden))
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with on_device(dev):
        _abi.check(_abi.lib().ds_mx4_gated_ffn(px, pa, dt, rows, ld, w1._ref(), w3._ref(), w2._ref(), limit or 0.0,
                                               out.data_ptr(), _DTYPES[out_dtype], ws.data_ptr(), n, raw_stream(dev)),
                   "ds_mx4_gated_ffn")
    return out


def status(device: torch.device | None = None) -> int:
    """Error bits of this module's calls on `device` since the last query (2: a
    bounded device wait gave up; outputs are then undefined).  Waits for the stream."""
    err = torch.zeros(1, dtype=torch.int32)
    with torch.cuda.device(device):
        _abi.check(_abi.lib().ds_mx4_status(err.data_ptr(), stream_handle(device)), "ds_mx4_status")
        torch.cuda.current_stream(device).synchronize()
    return int(err[0])
