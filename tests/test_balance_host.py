"""Checks of the balance loss that need no GPU: the C ABI looks at its arguments before any CUDA call, and the Python
layer refuses host tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from deepseeker import _abi, _build, balance


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _abi.lib()


def desc(**kw):
    d = dict(logits=256, tokens=8, ld=16, dtype=_abi.DS_F32, experts=16, top_k=2, kind=_abi.DS_ROUTE_SOFTMAX, ids=256,
             valid=None, offsets=None, offsets_i64=0, sequences=1)
    d.update(kw)
    return _abi.DsBalance(**d)


def size(lib, **kw):
    n = ctypes.c_size_t(0)
    return lib.ds_balance_loss_workspace_size(ctypes.byref(desc(**kw)), ctypes.byref(n)), n.value


BAD = [(dict(dtype=_abi.DS_U8), _abi.DS_EINVAL), (dict(kind=_abi.DS_ROUTE_SCORES), _abi.DS_EINVAL),
       (dict(experts=0), _abi.DS_ERANGE), (dict(experts=1025, ld=1025), _abi.DS_ERANGE), (dict(top_k=0), _abi.DS_ERANGE),
       (dict(top_k=33), _abi.DS_ERANGE), (dict(tokens=-1), _abi.DS_ERANGE), (dict(tokens=1 << 30), _abi.DS_ERANGE),
       (dict(tokens=1 << 62), _abi.DS_ERANGE), (dict(sequences=2), _abi.DS_ERANGE),
       (dict(sequences=-1, offsets=256), _abi.DS_ERANGE), (dict(sequences=(1 << 24) + 1, offsets=256), _abi.DS_ERANGE),
       (dict(ld=15), _abi.DS_EINVAL), (dict(logits=None), _abi.DS_EINVAL), (dict(logits=258), _abi.DS_EALIGN),
       (dict(ids=258), _abi.DS_EALIGN), (dict(offsets=258), _abi.DS_EALIGN),
       (dict(offsets=260, offsets_i64=1), _abi.DS_EALIGN)]


@pytest.mark.parametrize("kw,status", BAD)
def test_descriptor(lib, kw, status):
    assert size(lib, **kw)[0] == status and lib.ds_last_error_string()
    d = ctypes.byref(desc(**kw))
    assert lib.ds_balance_loss(d, 256, 256, 256, 256, 1 << 30, None) == status
    assert lib.ds_balance_loss_backward(d, 256, 256, 256, None) == status


def test_workspace_and_outputs(lib):
    assert size(lib) == (_abi.DS_OK, (1 + 1) * (2 * 16 + 1) * 4)          # one block and one sequence
    assert size(lib, offsets=256, sequences=5) == (_abi.DS_OK, (1 + 5) * 33 * 4)
    ok, n = size(lib, tokens=1 << 24, experts=1024, ld=1024)
    assert ok == _abi.DS_OK and n <= (148 * 4 + 1) * 2049 * 4
    d = ctypes.byref(desc())
    for bad in ((None, 256, 256, 256), (256, None, 256, 256), (256, 256, None, 256), (256, 256, 256, None)):
        assert lib.ds_balance_loss(d, *bad, 1 << 20, None) == _abi.DS_EINVAL
    assert lib.ds_balance_loss(d, 256, 256, 256, 256, 200, None) == _abi.DS_EINVAL
    assert lib.ds_balance_loss(d, 258, 256, 256, 256, 1 << 20, None) == _abi.DS_EALIGN
    assert lib.ds_balance_loss(ctypes.byref(desc(ids=None)), 256, 256, 256, 256, 1 << 20, None) == _abi.DS_EINVAL
    assert lib.ds_balance_loss_backward(d, None, 256, 256, None) == _abi.DS_EINVAL
    assert lib.ds_balance_loss_backward(d, 256, 256, 257, None) == _abi.DS_EALIGN
    assert lib.ds_balance_loss_workspace_size(d, None) == _abi.DS_EINVAL
    none = ctypes.byref(desc(sequences=0, offsets=256))
    assert lib.ds_balance_loss(none, None, None, None, None, 0, None) == _abi.DS_OK
    assert lib.ds_balance_loss_backward(ctypes.byref(desc(tokens=0)), None, None, None, None) == _abi.DS_OK


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        balance.balance_loss(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32))
