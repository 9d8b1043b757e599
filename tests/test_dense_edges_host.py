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


def test_workspace_with_clamps(lib):
    """Row norms of x, W1 and W3, and from 129 tokens on the list of values close to the limit, each on 256 bytes."""
    def size(limit, tokens, keeps):
        d = _abi.DsGatedFfn(tokens, 64, 32, _abi.DS_BF16, limit, 256, 256, 256, 256, 64, 64, 64, 32)
        n = ctypes.c_size_t(0)
        assert lib.ds_gated_ffn_workspace_size(ctypes.byref(d), keeps, ctypes.byref(n)) == _abi.DS_OK
        st = lib.ds_gated_ffn(ctypes.byref(d), 1024, 1024, 1024, 4096, n.value - 1, None) if keeps and n.value else _abi.DS_EINVAL
        assert st == _abi.DS_EINVAL                     # one byte too few
        return n.value

    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    for tokens in (1, 128, 129, 1000):
        more = up(4 * (tokens + 64)) + 256 + (up(8 * (tokens * 32 // 32)) if tokens > 128 else 0)
        assert size(0.0, tokens, 1) == 0 and size(10.0, tokens, 1) == more
        assert size(10.0, tokens, 0) == more + size(0.0, tokens, 0)
