"""Edge arguments of the dense operators that need no GPU."""
from __future__ import annotations

import ctypes

import pytest

from deepseeker import _abi, _build


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _abi.lib()


def test_no_rows_of_codes(lib):
    """A quantised matrix of no rows has no codes and no atoms; its products are empty, as those of no rows of values."""
    w, w2 = _abi.DsMx4(256, 256, 64, 96), _abi.DsMx4(256, 256, 96, 64)
    for dtype in (_abi.DS_U8, _abi.DS_BF16):
        assert lib.ds_mx4_linear(None, None, dtype, 0, 96, ctypes.byref(w), None, _abi.DS_BF16, None, 0, None) == _abi.DS_OK
        assert lib.ds_mx4_gated_ffn(None, None, dtype, 0, 96, ctypes.byref(w), ctypes.byref(w), ctypes.byref(w2), 0.0, None,
                                    _abi.DS_BF16, None, 0, None) == _abi.DS_OK
    # with rows, codes still need their atoms
    assert lib.ds_mx4_linear(256, None, _abi.DS_U8, 1, 96, ctypes.byref(w), 256, _abi.DS_BF16, None, 0, None) == _abi.DS_EINVAL
