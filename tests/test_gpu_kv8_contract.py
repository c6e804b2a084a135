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
