"""Arguments of the paged 4-bit cache's calls, without a GPU: a cache on the CPU whose launches
are stand-ins."""

import weakref

import pytest
import torch

from flashcodec_b200 import PagedInt4Cache
from flashcodec_b200 import _kernels as K

HK, D, PAGE = 2, 64, 16


@pytest.fixture
def cache(monkeypatch):
    cache = object.__new__(PagedInt4Cache)
    cache.device, cache._index, cache._scale = torch.device("cpu"), -1, 1.0  # a CPU tensor's index
    cache.num_kv_heads, cache.head_dim, cache.page_size = HK, D, PAGE
    cache._bounds = cache._exponents = torch.zeros(1)
    return cache


class Temporaries:
    """Tensors that nobody but the call holds."""

    def __init__(self):
        self.refs = []

    def __call__(self, t):
        self.refs.append(weakref.ref(t))
        return t

    def check(self, *args, **kwargs):
        assert all(r() is not None for r in self.refs), "freed before the launch"
        self.launched = True


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("call", ["read", "read_packed", "append", "append_packed", "attend", "select"])
def test_arguments_live_until_the_launch(cache, monkeypatch, call):
    """Outputs and workspaces are allocated within a call: an argument that is freed before could
    be where they are put."""
    tmp = Temporaries()
    for name in ("kv4_read", "kv4_append", "kv4_attn", "kv4_select"):
        monkeypatch.setattr(K, name, tmp.check)
    rows = lambda *lead, heads=HK: tmp(torch.zeros(*lead, heads, D))  # noqa: E731
    table = lambda: tmp(torch.zeros(3, 4, dtype=torch.int32))  # noqa: E731
    if call == "read":
        cache.read(table(), tmp(i32(0, 1, 2)), count=5)
    elif call == "read_packed":
        cache.read(table(), tmp(i32(0, 1, 2)), count=5, cu_seqlens=tmp(i32(0, 1, 3, 5)))
    elif call == "append":
        cache.append(rows(3, 1, heads=4), rows(3, 1), rows(3, 1), table(), tmp(i32(0, 1, 2)),
                     positions=tmp(i32(0, 1, 2)), q_weight=tmp(torch.ones(D)), k_weight=tmp(torch.ones(D)),
                     rotary=tmp(torch.ones(8, D)))
    elif call == "append_packed":
        cache.append(rows(5, heads=4), rows(5), rows(5), table(), tmp(i32(0, 1, 2)),
                     positions=tmp(i32(0, 1, 2, 3, 4)), cu_seqlens=tmp(i32(0, 1, 3, 5)))
    elif call == "attend":
        cache.attend(rows(3, heads=4), table(), tmp(i32(1, 1, 2)), return_lse=True,
                     selected=tmp(torch.zeros(3, HK, 2, dtype=torch.int32)))
    else:
        cache.select(rows(3, heads=4), table(), tmp(i32(1, 1, 2)), 3)
    assert tmp.launched


def test_dual_tensors_are_refused(cache, monkeypatch):
    """A tangent would be dropped: forward-mode differentiation is refused like reverse mode."""
    from torch.autograd import forward_ad
    monkeypatch.setattr(K, "kv4_attn", lambda *args: None)
    q, table, lengths = torch.zeros(3, 4, D), torch.zeros(3, 4, dtype=torch.int32), i32(1, 1, 2)
    with forward_ad.dual_level():
        cache.attend(q, table, lengths)
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for guard in (torch.no_grad(), torch.enable_grad()):
            with guard, pytest.raises(RuntimeError, match="tangent"):
                cache.attend(dual, table, lengths)
        cache.attend(forward_ad.unpack_dual(dual).primal, table, lengths)
    cache.attend(q, table, lengths)
    with pytest.raises(RuntimeError, match="no gradient"):
        cache.attend(q.clone().requires_grad_(), table, lengths)


@pytest.mark.parametrize("name", ["pool", "bounds", "exponents", "status"])
def test_the_caches_tensors_cannot_be_replaced(cache, name):
    """Launches go by their addresses: the kernels would write to what was freed."""
    cache._pool = cache._status = torch.zeros(1)
    held = getattr(cache, name)
    with pytest.raises(AttributeError):
        setattr(cache, name, held.clone())
    getattr(cache, name).fill_(3)
    assert getattr(cache, name) is held and held.item() == 3
