"""Checks of the dense operators that need no GPU: argument validation in the
C ABI comes before any CUDA call, sizes are the documented ones, and the Python
layer refuses host tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from deepseeker import _abi, _build, gated, mx4


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _abi.lib()


def desc(**kw):
    d = dict(tokens=4, hidden=64, inter=32, dtype=_abi.DS_BF16, limit=0.0, x=256, w1=256, w3=256, w2=256,
             ld_x=64, ld_w1=64, ld_w3=64, ld_w2=32)
    d.update(kw)
    return _abi.DsGatedFfn(**d)


def size(lib, d, keeps=0):
    n = ctypes.c_size_t(0)
    return lib.ds_gated_ffn_workspace_size(ctypes.byref(d), keeps, ctypes.byref(n)), n.value


def test_gated_workspace(lib):
    assert size(lib, desc()) == (_abi.DS_OK, 256)                       # h: 4 x 32 x 2 bytes
    assert size(lib, desc(), keeps=1) == (_abi.DS_OK, 0)
    assert size(lib, desc(inter=33, ld_w2=33)) == (_abi.DS_OK, 64 * 40 * 2 + 512)   # w2 copied, h [4, 40]
    assert size(lib, desc(x=258)) == (_abi.DS_OK, 512 + 256)            # x copied: no 16-byte base
    assert size(lib, desc(ld_x=65), keeps=1) == (_abi.DS_OK, 512)
    n = ctypes.c_size_t(0)
    assert lib.ds_gated_ffn_backward_workspace_size(ctypes.byref(desc()), 256, 64, ctypes.byref(n)) == _abi.DS_OK
    assert n.value == 512                                               # dg and du
    assert lib.ds_gated_ffn_backward_workspace_size(ctypes.byref(desc()), 256, 63, ctypes.byref(n)) == _abi.DS_EINVAL


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=-1), _abi.DS_ERANGE), (dict(tokens=(1 << 22) + 1), _abi.DS_ERANGE), (dict(hidden=0), _abi.DS_ERANGE),
    (dict(inter=(1 << 17) + 1), _abi.DS_ERANGE), (dict(dtype=_abi.DS_F32), _abi.DS_EINVAL),
    (dict(limit=-1.0), _abi.DS_EINVAL), (dict(limit=float("nan")), _abi.DS_EINVAL), (dict(ld_x=63), _abi.DS_EINVAL),
    (dict(ld_w1=63), _abi.DS_EINVAL), (dict(ld_w3=63), _abi.DS_EINVAL), (dict(ld_w2=31), _abi.DS_EINVAL)])
def test_gated_descriptor(lib, kw, status):
    assert size(lib, desc(**kw))[0] == status
    assert lib.ds_last_error_string()


def test_gated_call_arguments(lib):
    y, ws = 1024, 4096
    call = lambda d, y=y, h=None, pre=None, ws=ws, n=1 << 20: lib.ds_gated_ffn(  # noqa: E731
        ctypes.byref(d), y, h, pre, ws, n, None)
    assert call(desc(x=None)) == _abi.DS_EINVAL
    assert call(desc(w2=257)) == _abi.DS_EALIGN
    assert call(desc(), n=255) == _abi.DS_EINVAL
    assert call(desc(), ws=4097) == _abi.DS_EALIGN
    assert call(desc(), y=None) in (_abi.DS_EALIGN, _abi.DS_ECUDA)      # the driver's encoder may be missing here
    assert call(desc(tokens=0)) == _abi.DS_OK
    assert lib.ds_gated_ffn_backward(ctypes.byref(desc()), 256, 256, 256, 63, None, None, None, None, ws, 1 << 20,
                                     None) == _abi.DS_EINVAL
    assert lib.ds_gated_ffn_status(None, None) == _abi.DS_EINVAL


def test_mx4_sizes_and_arguments(lib):
    n = ctypes.c_size_t(0)
    for rows, cols in ((0, 1), (1, 1), (128, 128), (129, 129), (5, 4096)):
        assert lib.ds_mx4_atoms_size(rows, cols, ctypes.byref(n)) == _abi.DS_OK
        assert n.value == -(-rows // 128) * -(-cols // 128) * 512 == mx4._atoms_bytes(rows, cols)
        assert lib.ds_mx4_linear_workspace_size(rows, cols, ctypes.byref(n)) == _abi.DS_OK
        assert n.value == mx4._x_bytes(rows, cols) == (mx4._workspace_bytes(rows, cols) if rows > 16 else 0)
    for rows in (7, 16, 17, 70):                                        # up to 16 rows x needs none, h always
        assert lib.ds_mx4_gated_ffn_workspace_size(rows, 100, 60, ctypes.byref(n)) == _abi.DS_OK
        assert n.value == mx4._x_bytes(rows, 100) + mx4._workspace_bytes(rows, 60)
    assert lib.ds_mx4_atoms_size(1, 0, ctypes.byref(n)) == _abi.DS_EINVAL
    q = lambda *a: lib.ds_mx4_quantize(*a, None)  # noqa: E731
    assert q(256, _abi.DS_U8, 1, 32, 32, 256, 256, 256) == _abi.DS_EINVAL
    assert q(256, _abi.DS_F32, 1, 0, 32, 256, 256, 256) == _abi.DS_ERANGE
    assert q(256, _abi.DS_F32, 2, 32, 31, 256, 256, 256) == _abi.DS_EINVAL
    assert q(None, _abi.DS_F32, 2, 32, 32, 256, 256, 256) == _abi.DS_EINVAL
    assert q(258, _abi.DS_F32, 2, 32, 32, 256, 256, 256) == _abi.DS_EALIGN
    assert q(None, _abi.DS_F32, 0, 32, 32, None, None, None) == _abi.DS_OK
    assert lib.ds_mx4_dequantize(256, 256, 1, 32, 256, _abi.DS_F16, None) == _abi.DS_EINVAL
    assert lib.ds_mx4_scale_atoms(256, 1, 0, 256, None) == _abi.DS_ERANGE
    w, w2 = _abi.DsMx4(256, 256, 64, 96), _abi.DsMx4(256, 256, 96, 64)
    lin = lambda x, xa, dt, rows, ld, w, odt, ws, n: lib.ds_mx4_linear(  # noqa: E731
        x, xa, dt, rows, ld, ctypes.byref(w), 256, odt, ws, n, None)
    assert lin(256, None, _abi.DS_U8, 1, 0, w, _abi.DS_F32, None, 0) == _abi.DS_EINVAL     # codes without atoms
    assert lin(256, None, _abi.DS_F32, 2, 95, w, _abi.DS_F32, 256, 1 << 20) == _abi.DS_EINVAL
    assert lin(256, None, _abi.DS_F32, 1, 96, w, _abi.DS_U8, 256, 1 << 20) == _abi.DS_EINVAL
    assert lin(256, None, _abi.DS_F32, 17, 96, w, _abi.DS_F32, 256, 255) == _abi.DS_EINVAL
    assert lin(256, None, _abi.DS_F32, (1 << 22) + 1, 96, w, _abi.DS_F32, 256, 1 << 40) == _abi.DS_ERANGE
    assert lin(256, None, _abi.DS_F32, 1, 96, _abi.DsMx4(256, None, 64, 96), _abi.DS_F32, 256, 1 << 20) == _abi.DS_EINVAL
    assert lin(256, None, _abi.DS_F32, 1, 96, _abi.DsMx4(264, 256, 64, 96), _abi.DS_F32, 256, 1 << 20) == _abi.DS_EALIGN
    ffn = lambda a, b, c, limit: lib.ds_mx4_gated_ffn(  # noqa: E731
        256, None, _abi.DS_F32, 1, 96, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c), limit, 256, _abi.DS_F32, 256,
        1 << 20, None)
    assert ffn(w, w2, w2, 0.0) == _abi.DS_EINVAL and ffn(w, w, w, 0.0) == _abi.DS_EINVAL
    assert ffn(w, w, w2, -1.0) == _abi.DS_EINVAL


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        gated.gated_ffn(x, w, w, w.t())
    with pytest.raises(ValueError):
        mx4.quantize(x)
    with pytest.raises(ValueError):
        mx4.linear(x, w)
    with pytest.raises(ValueError):
        mx4.from_packed(torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8))
