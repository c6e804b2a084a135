"""What the package keeps is written to in whatever mode it was made in, without a GPU (allocations, the stream and
the library are stand-ins): a tensor made in inference mode could not be written to outside of it."""

import types

import pytest
import torch

from flashcodec_b200 import _kernels as K


@pytest.fixture
def lib(monkeypatch):
    lib = types.SimpleNamespace(fc_capture_id=lambda stream: 0, fc_kv8_attn_workspace_size=lambda *sizes: 4096,
                                fc_kv4_select_workspace_size=lambda *sizes: 256)
    for name in ("zeros", "empty"):
        make = getattr(torch, name)
        monkeypatch.setattr(K.torch, name, lambda n, dtype, device, make=make: make(n, dtype=dtype))
    monkeypatch.setattr(K._lib, "load", lambda: lib)
    monkeypatch.setattr(K.torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=7))
    for held in ("_workspaces", "_prompt_workspaces", "_kv4_workspaces", "_kv4_captured"):
        monkeypatch.setattr(K, held, {})


def test_workspaces(lib):
    with torch.inference_mode():
        decode = K.workspace(torch.device("cuda", 0), 5000)
        prompt = K._prompt_workspace(0, 7, 100000)
        paged = K._kv4_workspace("attn", (1, 1, 8, 2, 64), 64, 0, 7, cache="kv8")
    for ws in (decode, prompt, paged.buffer):
        ws[:256].zero_()
    paged.clear()
    with torch.inference_mode():
        decode.zero_()
