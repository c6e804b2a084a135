"""Paged 4-bit attention where its sums could lose.  Against fp64 over the values held, with the
bounds of test_gpu_kv4.py where none is given."""

import math

import numpy as np
import pytest
import torch

from oracle import kv4
from test_gpu_kv4 import DT, UNIT, fc, i32, near, table_of

pytestmark = pytest.mark.gpu


def held_by(k, v, page=64):
    """A cache of one sequence: (cache, table, keys, values as held)."""
    n, D = k.shape
    table, pages = table_of([n], page)
    cache = fc().PagedInt4Cache(pages, 1, D, page_size=page)
    cache.append(None, k[None, :, None].cuda(), v[None, :, None].cuda(), table, i32([0]))
    return cache, table, *(kv4.values(*kv4.quantise(x.numpy())) for x in (k, v))


# ------------------------------------------------------------------- small values
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vscale", [1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("alike", [False, True])
def test_small_values(dtype, vscale, alike):
    """One strong token among 4096 that together weigh as much, in batches so large that a warp
    takes 1024 of them.  `alike`: the same value everywhere, so that what the weights' roundings
    do to one token they do to all.  (An fp16 output this small is itself a multiple of 2^-24.)"""
    n, D, B = 4096, 128, 450
    g = torch.Generator().manual_seed(12)
    k = torch.zeros(n, D)
    k[1234] = math.log(n) / D ** 0.5
    v = vscale * (torch.randn(1, D, generator=g).expand(n, D) if alike else torch.randn(n, D, generator=g))
    cache, table, hk, hv = held_by(k, v)
    q = torch.ones(B, 2, D, dtype=DT[dtype], device="cuda")
    out = cache.attend(q, table.repeat(B, 1), torch.full((B,), n, dtype=torch.int32, device="cuda"))
    want, _ = kv4.attend(np.ones((2, D)), hk, hv)
    want, top = np.broadcast_to(want, out.shape), np.abs(hv).max()
    if dtype == "fp16":
        err = np.abs(out.double().cpu().numpy() - want)
        lim = 2 * UNIT[dtype] * np.abs(want) + 2.0 ** -13 * top + 2.0 ** -25
        assert (err <= lim).all(), f"{err.max():.3e} over {lim.flat[err.argmax()]:.3e}"
    else:
        near(out, want, dtype, top)
