"""Checks of the layer norm that need no GPU: the C ABI looks at its arguments before any CUDA call, and the Python
layer refuses host tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from deepseeker import _abi, _build, norm


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _abi.lib()


F32, BF16, F16, U8 = _abi.DS_F32, _abi.DS_BF16, _abi.DS_F16, _abi.DS_U8


def forward(lib, x=256, dtype=BF16, rows=4, cols=64, ld=64, w=256, b=256, kind=F32, eps=1e-5, y=256, stats=256):
    return lib.ds_layer_norm(x, dtype, rows, cols, ld, w, b, kind, eps, y, stats, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=U8), _abi.DS_EINVAL), (dict(kind=F16), _abi.DS_EINVAL), (dict(dtype=F32, kind=BF16), _abi.DS_EINVAL),
    (dict(rows=-1), _abi.DS_ERANGE), (dict(rows=1 << 31), _abi.DS_ERANGE), (dict(cols=0), _abi.DS_ERANGE),
    (dict(cols=(1 << 20) + 1, ld=1 << 21), _abi.DS_ERANGE), (dict(ld=63), _abi.DS_EINVAL),
    (dict(eps=-1.0), _abi.DS_EINVAL), (dict(eps=float("nan")), _abi.DS_EINVAL), (dict(eps=float("inf")), _abi.DS_EINVAL), (dict(x=None), _abi.DS_EINVAL),
    (dict(y=None), _abi.DS_EINVAL), (dict(x=257), _abi.DS_EALIGN), (dict(w=258), _abi.DS_EALIGN),
    (dict(stats=260), _abi.DS_EALIGN)])
def test_forward_arguments(lib, kw, status):
    assert forward(lib, **kw) == status and lib.ds_last_error_string()
    assert forward(lib, rows=0, x=None, y=None) == _abi.DS_OK


def backward(lib, x=256, dtype=BF16, rows=4, cols=64, ld=64, w=256, kind=F32, stats=256, dy=256, ld_dy=64, dx=256,
             dw=256, db=256, ws=256, n=1 << 30):
    return lib.ds_layer_norm_backward(x, dtype, rows, cols, ld, w, kind, stats, dy, ld_dy, dx, dw, db, ws, n, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=U8), _abi.DS_EINVAL), (dict(ld_dy=63), _abi.DS_EINVAL), (dict(stats=None), _abi.DS_EINVAL),
    (dict(dy=None), _abi.DS_EINVAL), (dict(n=0), _abi.DS_EINVAL), (dict(ws=None), _abi.DS_EINVAL),
    (dict(ws=264), _abi.DS_EALIGN), (dict(dx=257), _abi.DS_EALIGN), (dict(dw=258), _abi.DS_EALIGN)])
def test_backward_arguments(lib, kw, status):
    assert backward(lib, **kw) == status and lib.ds_last_error_string()


def test_backward_of_nothing(lib):
    assert backward(lib, rows=0, x=None, dy=None, stats=None, dw=None, db=None, ws=None, n=0) == _abi.DS_OK


def test_workspace(lib):
    n = ctypes.c_size_t(0)
    size = lambda r, c: (lib.ds_layer_norm_backward_workspace_size(r, c, ctypes.byref(n)), n.value)  # noqa: E731
    assert size(0, 64) == (_abi.DS_OK, 0)
    assert size(1, 4096) == (_abi.DS_OK, 2 * 4096 * 4)
    for rows, cols in ((5, 1), (100, 711), (8192, 4096), (1 << 30, 8192), (7, 8193), (1 << 30, 1 << 20)):
        ok, bytes_ = size(rows, cols)
        assert ok == _abi.DS_OK and bytes_ % (8 * cols) == 0 and 1 <= bytes_ // (8 * cols) <= min(rows, 148 * 16)
    assert size(1, 0)[0] == size(-1, 4)[0] == _abi.DS_EINVAL
    assert lib.ds_layer_norm_backward_workspace_size(1, 1, None) == _abi.DS_EINVAL


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        norm.layer_norm(x)
    with pytest.raises(ValueError):
        norm.layer_norm(x, torch.ones(8), torch.zeros(8))
