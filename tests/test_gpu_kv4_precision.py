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


# --------------------------------------------------------------- values with a mean
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("halves", [False, True])
def test_flat_attention_over_values_with_a_mean(dtype, halves):
    """Equal weights over 2^20 tokens, 2^18 of them a warp's, of values around 3, or around 3 and
    then around -3: the sums grow with the mean.  Beside its rounding the output may be off by
      * what sums lose that are cut at each of 256 steps of 16 tokens before they are added up
        in rounded fp32: growing from zero, 256 / 2 ulps (2^-23) of the mean, 2^-16 * 3;
      * the cuts of the codes' offset between two centrings, 2^-16 of a code's step (M / 7);
      * the fp32 sums' roundings, 2^-20 M, as in the test of values without a mean."""
    n, D, B, page, G = 1 << 20, 128, 450, 64, 2
    cache = fc().PagedInt4Cache(n // page, 1, D, page_size=page)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None].contiguous()
    v = torch.randn(1, n, 1, D, generator=torch.Generator("cuda").manual_seed(5), device="cuda") + 3
    if halves:
        v[:, n // 2:] -= 6
    cache.append(None, torch.zeros_like(v), v, table, i32([0]))
    held = cache.read(table, count=n, dtype=torch.float32)[1][0, :, 0].double()
    want, top = held.mean(0).cpu().numpy(), float(held.abs().max())
    out = cache.attend(torch.zeros(B, G, D, dtype=DT[dtype], device="cuda"), table.repeat(B, 1).contiguous(),
                       torch.full((B,), n, dtype=torch.int32, device="cuda"))
    err = np.abs(out.double().cpu().numpy() - want).max((0, 1))
    lim = 2 * UNIT[dtype] * np.abs(want) + 2.0 ** -16 * 3 + 2.0 ** -16 * top / 7 + 2.0 ** -20 * top
    assert (err <= lim).all(), f"{err.max():.2e} over {lim[err.argmax()]:.2e}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,page,G,Sq", [(64, 64, 2, 1), (96, 16, 4, 1), (128, 64, 16, 1), (256, 32, 2, 1),
                                         (128, 128, 2, 3), (192, 64, 3, 1)])
@pytest.mark.parametrize("rise", [-1.0, 1.0])
def test_segments_of_several_spans(dtype, D, page, G, Sq, rise):
    """70001 tokens a sequence in batches so large that a warp takes 17500 of them, with scores that
    rise or fall by 80 on the way: the references of a warp's spans lie far apart."""
    n, B = 70001, 450
    g = torch.Generator().manual_seed(D)
    way = torch.linspace(0, 80 * rise, n)[:, None] / D ** 0.5
    cache, table, hk, hv = held_by(torch.randn(n, D, generator=g) + way, torch.randn(n, D, generator=g), page)
    q = (1 + 0.2 * torch.randn(1, Sq, G, D, generator=g)).to(DT[dtype])
    out, lse = cache.attend(q.cuda().expand(B, Sq, G, D).contiguous(), table.repeat(B, 1),
                            torch.full((B,), n, dtype=torch.int32, device="cuda"), return_lse=True)
    for s in range(Sq):
        m = n - Sq + 1 + s
        want, wl = kv4.attend(q[0, s].float().numpy(), hk[:m], hv[:m])
        near(out[:, s], np.broadcast_to(want, out[:, s].shape), dtype, np.abs(hv).max(), s)
        assert (np.abs(lse[:, s].double().cpu().numpy() - wl) <= 2.0 ** -9 * (1 + np.abs(wl))).all()
    cache.check()


# ------------------------------------------------------------------ ends of the range
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("log2q", [20, 26, 33, 50, 100, 118, 125])
@pytest.mark.parametrize("best", [0.0, 2.0 ** -12, -2.0 ** -12])
def test_queries_and_scores_at_the_ends_of_fp32(dtype, log2q, best):
    """Queries near the largest number: the weights are one and zeros, whether the largest score
    is zero, far above it or far below -1e30 (the other keys' scores are far below it)."""
    n, D = 200, 64
    g = torch.Generator().manual_seed(13)
    q = 2.0 ** log2q * (1 + torch.rand(2, D, generator=g)).to(DT[dtype])
    v = torch.randn(n, D, generator=g)
    k = -(1 + torch.rand(n, 1, generator=g)).expand(n, D) * 2.0 ** -9
    k = k.contiguous()
    k[77] = best
    cache, table, hk, hv = held_by(k, v)
    want, wl = kv4.attend(q.double().numpy(), hk, hv)
    assert (want == hv[77]).all()
    out, lse = cache.attend(q[None].cuda(), table, i32([n]), return_lse=True)
    near(out[0], want, dtype, np.abs(hv).max())
    if log2q < 120 or dtype == "fp32":  # bf16 queries beyond: the logarithm itself is not kept
        assert (np.abs(lse[0].double().cpu().numpy() - wl) <= 2.0 ** -9 * np.abs(wl)).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.0, 1e-30, None])
def test_tiny_queries_and_scales(dtype, scale):
    """Scores that round to zero, next to tokens that the first of two queries does not see."""
    n, D = 77, 64
    g = torch.Generator().manual_seed(14)
    cache, table, hk, hv = held_by(torch.randn(n, D, generator=g), torch.randn(n, D, generator=g))
    q = (1e-25 * torch.randn(1, 2, 2, D, generator=g)).to(DT[dtype])
    out = cache.attend(q.cuda(), table, i32([n]), scale=scale)[0]
    for s in range(2):
        want, _ = kv4.attend(q[0, s].float().numpy(), hk[: n - 1 + s], hv[: n - 1 + s], scale=scale)
        near(out[s], want, dtype, np.abs(hv).max(), s)
