"""Workspaces of the paged 4-bit cache, without a GPU: which buffer a call gets, eagerly and
while a CUDA graph is captured (the allocations and the library are stand-ins)."""

import ctypes
import weakref

import pytest
import torch

from flashcodec_b200 import _kernels as K


class Library:
    """The size function, and a capture that is under way or not."""

    def __init__(self):
        self.capture = 0

    def fc_capture_id(self, stream):
        return self.capture

    def fc_kv4_select_workspace_size(self, B, Hk, n):
        return 64 + 4 * B * Hk * n

    fc_kv4_attn_workspace_size = fc_kv4_select_workspace_size


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    empty = torch.empty
    monkeypatch.setattr(K._lib, "load", lambda: lib)
    monkeypatch.setattr(K.torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype).fill_(9))
    for held in ("_kv4_workspaces", "_kv4_captured"):
        monkeypatch.setattr(K, held, {})
    return lib


def get(B, stream=7, what="select"):
    return K._kv4_workspace(what, (B, 2, 8), B * 16, 0, stream)


def buffer(B, **kw):
    return get(B, **kw).buffer


def test_a_larger_call_leaves_a_captured_buffer_alone(lib):
    """A graph captured for one sequence, then an eager call and another capture for eight."""
    lib.capture = 1
    ws = get(1)
    address, alive = ws.address, weakref.ref(ws.buffer)
    ws = None
    lib.capture = 0
    assert buffer(8).data_ptr() != address
    assert alive() is not None and get(8).address != address


def test_a_capture_shares_its_buffer_with_no_other_call(lib):
    """What zeroes it is a node of its own graph: nobody else may count on that."""
    eager = buffer(4)
    lib.capture = 1
    first = buffer(4)
    assert buffer(4) is first  # one memset a graph, not one a call
    lib.capture = 2
    second = buffer(4)
    lib.capture = 0
    assert len({x.data_ptr() for x in (eager, first, second)}) == 3
    assert buffer(4) is eager


def test_captures_on_two_streams_have_a_buffer_each(lib):
    """One capture may fork into streams whose calls overlap."""
    lib.capture = 1
    assert buffer(4, stream=7).data_ptr() != buffer(4, stream=8).data_ptr()
    assert buffer(4, what="attn").data_ptr() != buffer(4, what="select").data_ptr()


@pytest.mark.parametrize("capture", [0, 5])
def test_buffers_grow_and_fit(lib, capture):
    lib.capture = capture
    for B in (1, 8, 3):
        ws = get(B)
        assert ws.bytes == ws.buffer.numel() >= lib.fc_kv4_select_workspace_size(B, 2, 8)
        assert ws.address == ws.buffer.data_ptr() and not ws.buffer[:64].any()
    small, large = get(1), get(8)
    assert small is large


def test_no_capture_is_under_way_here():
    from flashcodec_b200 import _lib, build
    build.build()
    assert _lib.load().fc_capture_id(ctypes.c_void_p(0)) == 0
