"""Paged 8-bit KV cache: calls that its documentation allows and that lie off the beaten track."""

import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import DT, fc, i32, new_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_values_that_are_no_numbers_and_weigh_nothing(D, dtype):
    """A run that reads as NaN makes the outputs that see it NaN, whether its weights are below fp32 (scores of
    -320 D^1/2 / 8) or not, and wherever it lies among the tokens; outputs that do not see it stay what they were."""
    n, Hk, page = 600, 2, 16
    g = torch.Generator().manual_seed(D)
    table = i32([list(range(38))])
    q = torch.ones(1, 2, 2 * Hk, D, dtype=DT[dtype], device="cuda")
    for run in (0, 3, 10, 11, 36):
        k, v = (torch.randn(1, n, Hk, D, generator=g) for _ in range(2))
        k[:, 16 * run:16 * run + 16] = -40
        out = []
        for x in (0.0, math.nan, math.inf):
            v[0, 16 * run + 9, 0, 7] = x
            cache = new_cache(38, Hk, D, page)
            cache.append(None, k.cuda(), v.cuda(), table, i32([0]))
            out.append([cache.attend(q, table, i32([m])) for m in (n, 16 * run + 17, 16 * run)])
        for m, (fine, nan, inf) in enumerate(zip(*out)):
            if m < 2:
                assert nan[:, :, :2].isnan().all() and inf[:, :, :2].isnan().all() and fine.isfinite().all()
                assert torch.equal(nan[:, :, 2:], fine[:, :, 2:]) and torch.equal(inf[:, :, 2:], fine[:, :, 2:])
            else:  # not seen
                assert torch.equal(nan, fine) and torch.equal(inf, fine) and fine.isfinite().all()


@pytest.mark.parametrize("made_in_inference_mode", [True, False])
@pytest.mark.parametrize("bits", [4, 8])
def test_caches_and_calls_in_inference_mode(bits, made_in_inference_mode):
    """A cache made in inference mode is checked, cleared and restored outside of it, and the other way round."""
    make = fc().PagedInt8Cache if bits == 8 else (lambda *a, **kw: fc().PagedInt4Cache(*a, bounds=True, **kw))
    x = torch.randn(1, 20, 2, 64, device="cuda")
    with torch.inference_mode(made_in_inference_mode):
        cache = make(4, 2, 64, page_size=16)
        cache.append(None, x, x, i32([[0, 1]]), i32([0]))
        cache.append(None, x, x, i32([[0, 9]]), i32([0]))  # a page outside the pool
        want = cache.attend(x[:, 0], i32([[0, 1]]), i32([20]))
        fc().prompt_attention(x[0].half(), x[0].half(), x[0].half(), i32([0, 20]))
    with torch.inference_mode(not made_in_inference_mode):
        with pytest.raises(fc()._lib.FlashCodecError, match="page outside"):
            cache.check()
        cache.check()
        assert fc().attention_status(reset=True).value() == 0
        held = [cache.pool] if bits == 4 else [cache.codes, cache.scales]
        for t in held:
            t.copy_(t.clone())
        assert torch.equal(cache.attend(x[:, 0], i32([[0, 1]]), i32([20])), want)


def test_a_pool_beyond_32_bits():
    """Pages whose codes lie beyond 2^32 bytes are appended to, read and attended to as those at the front."""
    Hk, D, page, n = 8, 128, 64, 150
    num = (9 << 29) // (2 * Hk * page * D) + 8
    cache = fc().PagedInt8Cache(num, Hk, D, page_size=page)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, n, Hk, D, generator=g).cuda() for _ in range(2))
    q = torch.randn(1, 16, D, generator=g).cuda()
    got = []
    for first in (0, num - 3):
        table = i32([[first, first + 2, first + 1]])
        cache.append(None, k, v, table, i32([0]))
        got.append((*cache.read(table, count=n, dtype=torch.float32), cache.attend(q, table, i32([n]))))
    cache.check()
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert (got[0][0] - k).abs().max() <= 2.0 ** -7 * k.abs().max()


def test_calls_on_two_streams_at_once():
    """Steps of two caches and prompts that are cut, issued to two streams in turn, without waiting: each gives what it
    gives alone."""
    work = []
    for i, lens in enumerate(([40, 900, 3], [4000])):
        g = torch.Generator().manual_seed(i)
        B, m = len(lens), max(lens)
        cache = new_cache(B * 64, 2, 128, 64)
        table = torch.arange(B * 64, dtype=torch.int32, device="cuda").view(B, 64)
        k = torch.randn(B, m, 2, 128, generator=g).bfloat16().cuda()
        cache.append(None, k, k, table, i32([0] * B))
        q = torch.randn(B, 8, 128, generator=g).bfloat16().cuda()
        x = torch.randn(20, 8, 128, generator=g).bfloat16().cuda()
        work.append((cache, table, i32(lens), q, (x, k[0], k[0], i32([0, 20]), i32([0, m]))))
    run = lambda w: (w[0].attend(w[3], w[1], w[2]), fc().prompt_attention(*w[4]))  # noqa: E731
    want = [run(w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(100):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append((i, run(work[i])))
    torch.cuda.synchronize()
    for i, out in outs:
        assert all(torch.equal(x, y) for x, y in zip(out, want[i]))
