"""The dense operators' error words are read and cleared in one step: with a
copy and a memset, a call on another stream that gives up between the two would
never be told."""
from __future__ import annotations

import ctypes

import pytest
import torch

from deepseeker import _abi, gated, mx4
from deepseeker._dev import stream_handle

pytestmark = pytest.mark.gpu
KERNEL, MEMCPY, MEMSET = 0, 1, 2   # CUgraphNodeType


def nodes(graph) -> list[int]:
    """Node types of a captured graph."""
    cu = ctypes.CDLL("libcuda.so.1")
    handle, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert cu.cuGraphGetNodes(handle, None, ctypes.byref(n)) == 0
    at = (ctypes.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(handle, at, ctypes.byref(n)) == 0
    kinds = []
    for node in at:
        kind = ctypes.c_int(-1)
        assert cu.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        kinds.append(kind.value)
    return kinds


@pytest.mark.parametrize("name", ["ds_gated_ffn_status", "ds_mx4_status"])
def test_one_step(name, cuda):
    err = torch.full((1,), 77, dtype=torch.int32).pin_memory()
    call = lambda: _abi.call(name, err.data_ptr(), stream_handle(cuda))  # noqa: E731
    call()
    torch.cuda.synchronize()
    assert int(err[0]) == 0
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    kinds = nodes(graph)
    assert kinds.count(KERNEL) == 1 and kinds.count(MEMCPY) == 1 and MEMSET not in kinds
    err.fill_(77)
    graph.replay()
    torch.cuda.synchronize()
    assert int(err[0]) == 0


def test_every_kind_of_memory(cuda):
    """The answer goes to host memory of either kind or to the device."""
    for err in (torch.full((1,), 5, dtype=torch.int32), torch.full((1,), 5, dtype=torch.int32, device=cuda)):
        for name in ("ds_gated_ffn_status", "ds_mx4_status"):
            err.fill_(5)
            _abi.call(name, err.data_ptr(), stream_handle(cuda))
            torch.cuda.synchronize()
            assert int(err[0]) == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert gated.status() == 0 and mx4.status() == 0
