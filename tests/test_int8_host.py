"""Checks of the 8-bit integer operators that need no GPU: the C ABI looks at its arguments before any CUDA call, and
the Python layer refuses host tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from deepseeker import _abi, _build, int8

BF16, I8, U8 = _abi.DS_BF16, _abi.DS_I8, _abi.DS_U8


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _abi.lib()


def quantize(lib, x=256, dtype=BF16, rows=4, cols=40, ld=40, codes=256, pitch=48, scales=256):
    return lib.ds_int8_quantize(x, dtype, rows, cols, ld, codes, pitch, scales, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=U8), _abi.DS_EINVAL), (dict(dtype=I8), _abi.DS_EINVAL), (dict(rows=-1), _abi.DS_ERANGE),
    (dict(rows=1 << 31), _abi.DS_ERANGE), (dict(cols=0), _abi.DS_ERANGE),
    (dict(cols=1 << 17, ld=1 << 17, pitch=1 << 17), _abi.DS_ERANGE), (dict(ld=39), _abi.DS_EINVAL),
    (dict(pitch=32), _abi.DS_EINVAL), (dict(pitch=40), _abi.DS_EINVAL), (dict(x=None), _abi.DS_EINVAL),
    (dict(scales=None), _abi.DS_EINVAL), (dict(x=257), _abi.DS_EALIGN), (dict(codes=264), _abi.DS_EALIGN),
    (dict(scales=258), _abi.DS_EALIGN)])
def test_quantize_arguments(lib, kw, status):
    assert quantize(lib, **kw) == status and lib.ds_last_error_string()
    assert quantize(lib, rows=0, x=None, codes=None, scales=None) == _abi.DS_OK


def test_dequantize_arguments(lib):
    call = lambda codes=256, pitch=48, scales=256, rows=4, cols=40, out=256, dtype=BF16: lib.ds_int8_dequantize(  # noqa: E731
        codes, pitch, scales, rows, cols, out, dtype, None)
    assert call(dtype=I8) == call(pitch=40) == call(pitch=32) == call(out=None) == _abi.DS_EINVAL
    assert call(rows=-1) == call(cols=0) == call(cols=1 << 17, pitch=1 << 17) == _abi.DS_ERANGE
    assert call(codes=264) == call(out=257) == call(scales=258) == _abi.DS_EALIGN
    assert call(rows=0, codes=None, out=None) == _abi.DS_OK


def linear(lib, x=256, xs=None, dtype=BF16, rows=20, ld=40, out=256, to=BF16, ws=256, n=1 << 20, null=False, **w):
    d = dict(codes=256, scales=256, rows=8, cols=40, pitch=48)
    d.update(w.get("w", {}))
    return lib.ds_int8_linear(x, xs, dtype, rows, ld, None if null else ctypes.byref(_abi.DsInt8(**d)), out, to, ws, n,
                              None)


@pytest.mark.parametrize("kw,status", [
    (dict(null=True), _abi.DS_EINVAL), (dict(w=dict(codes=None)), _abi.DS_EINVAL), (dict(w=dict(rows=0)), _abi.DS_ERANGE),
    (dict(w=dict(rows=(1 << 20) + 1)), _abi.DS_ERANGE), (dict(w=dict(cols=1 << 17, pitch=1 << 17)), _abi.DS_ERANGE),
    (dict(w=dict(pitch=40)), _abi.DS_EINVAL), (dict(w=dict(pitch=32)), _abi.DS_EINVAL),
    (dict(w=dict(codes=264)), _abi.DS_EALIGN), (dict(w=dict(scales=258)), _abi.DS_EALIGN), (dict(dtype=U8), _abi.DS_EINVAL),
    (dict(dtype=I8, ld=48), _abi.DS_EINVAL), (dict(dtype=I8, xs=256, ld=40), _abi.DS_EINVAL),
    (dict(dtype=I8, xs=256, ld=32, rows=1), _abi.DS_EINVAL), (dict(dtype=I8, xs=256, ld=48, x=264), _abi.DS_EALIGN),
    (dict(dtype=I8, xs=258, ld=48), _abi.DS_EALIGN), (dict(rows=-1), _abi.DS_ERANGE),
    (dict(rows=(1 << 22) + 1), _abi.DS_ERANGE), (dict(ld=39), _abi.DS_EINVAL), (dict(to=U8), _abi.DS_EINVAL),
    (dict(x=None), _abi.DS_EINVAL), (dict(x=257), _abi.DS_EALIGN), (dict(n=20 * 48 + 64 + 256 - 1), _abi.DS_EINVAL),
    (dict(ws=None), _abi.DS_EINVAL), (dict(ws=264), _abi.DS_EALIGN), (dict(out=None), _abi.DS_EALIGN),
    (dict(out=257), _abi.DS_EALIGN)])
def test_linear_arguments(lib, kw, status):
    assert linear(lib, **kw) == status and lib.ds_last_error_string()
    assert linear(lib, rows=0, x=None, out=None, ws=None, n=0) == _abi.DS_OK


def test_sizes(lib):
    n = ctypes.c_size_t(0)
    for rows, cols in ((0, 1), (1, 1), (2, 16), (3, 16), (8, 40), (9, 17), (16, 17), (17, 17), (129, 4096)):
        assert lib.ds_int8_linear_workspace_size(rows, cols, ctypes.byref(n)) == _abi.DS_OK
        assert n.value == int8._x_bytes(rows, cols) == (
            int8._workspace_bytes(rows, cols) if rows > 1 else 0)
    assert lib.ds_int8_linear_workspace_size(1, 0, ctypes.byref(n)) == _abi.DS_EINVAL
    assert lib.ds_int8_linear_workspace_size(1, 1, None) == _abi.DS_EINVAL
    assert lib.ds_int8_status(None, None) == _abi.DS_EINVAL


def test_host_tensors_are_refused():
    x = torch.zeros(2, 32)
    for call in (lambda: int8.quantize(x), lambda: int8.linear(x, x),
                 lambda: int8.from_codes(torch.zeros(2, 32, dtype=torch.int8), torch.ones(2))):
        with pytest.raises(ValueError):
            call()
