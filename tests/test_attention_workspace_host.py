"""Which workspace a codec decode-attention call gets, eagerly and while a CUDA graph is captured,
without a GPU (the stream, the allocation and the library are stand-ins)."""

import types
import weakref

import pytest
import torch

from flashcodec_b200 import _kernels as K

CUDA = torch.device("cuda", 0)


@pytest.fixture
def lib(monkeypatch):
    lib, zeros = types.SimpleNamespace(capture=0), torch.zeros
    lib.fc_capture_id = lambda stream: lib.capture
    monkeypatch.setattr(K._lib, "load", lambda: lib)
    monkeypatch.setattr(K.torch, "zeros", lambda n, dtype, device: zeros(n, dtype=dtype))
    monkeypatch.setattr(K.torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(K, "_workspaces", {})
    return lib


def test_a_capture_shares_its_workspace_with_no_other_call(lib):
    eager = K.workspace(CUDA, 5000)
    lib.capture = 1
    first = K.workspace(CUDA, 5000)
    assert K.workspace(CUDA, 100) is first
    lib.capture = 2
    second = K.workspace(CUDA, 5000)
    lib.capture = 0
    assert K.workspace(CUDA, 5000) is eager
    assert len({x.data_ptr() for x in (eager, first, second)}) == 3


def test_a_larger_call_leaves_a_captured_workspace_alone(lib):
    lib.capture = 1
    alive = weakref.ref(K.workspace(CUDA, 5000))
    lib.capture = 0
    assert K.workspace(CUDA, 50000).numel() == 50000
    assert alive() is not None
