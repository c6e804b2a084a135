"""The plan of the paged 4-bit attention: batches whose pieces end, or begin, among the chunks
that stand for a unit's overhead, so that a block plans a unit of which it has no chunk."""

import numpy as np
import pytest
import torch

from oracle import kv4
from test_gpu_kv4 import DT, filled, i32, near

pytestmark = pytest.mark.gpu

SLOTS = 4  # warps of a block


def without_chunks(lens, heads, tokens, overhead, blocks):
    """(block, unit) pairs where a block's piece of the line reaches a unit of `n + overhead` and
    holds none of its n chunks."""
    units = [(-(-n // tokens), b, h) for b, n in enumerate(lens) if n for h in range(heads)]
    line = sum(n + overhead for n, _, _ in units)
    blocks = min(blocks, -(-line // (overhead + SLOTS)))
    found, at = [], 0
    for n, b, h in units:
        for i in range(blocks):
            x, end = line * i // blocks, line * (i + 1) // blocks
            if x < at + n + overhead and end > at and end <= at + overhead:
                found.append((i, b, h))
        at += n + overhead
    return found


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,page,tokens,overhead", [(64, 64, 64, 8), (128, 64, 64, 8), (64, 32, 32, 16),
                                                    (256, 16, 32, 16)])
@pytest.mark.parametrize("seed", [0, 1])
def test_pieces_that_end_in_a_units_overhead(dtype, D, page, tokens, overhead, seed):
    Hk, G = 2, 2
    rng = np.random.default_rng(seed)
    lens = [int(n) for n in np.exp(rng.uniform(0, np.log(1500), 150))] + [0, 1, 1]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for resident in (2, 3, 4):  # whatever number of blocks an SM holds
        assert without_chunks(lens, Hk, tokens, overhead, sms * resident)
    cache, table, held = filled(lens, Hk, D, page, seed=seed)
    q = torch.randn(len(lens), Hk * G, D, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    out = cache.attend(q.cuda(), table, i32(lens))
    for _ in range(20):
        assert torch.equal(cache.attend(q.cuda(), table, i32(lens)), out)
    for b, n in enumerate(lens):
        for h in range(Hk):
            rows = slice(h * G, (h + 1) * G)
            k, v = (x[:, h] for x in held[b])
            want, _ = kv4.attend(q[b, rows].float().numpy(), k, v)
            near(out[b, rows], want, dtype, np.abs(v).max() if n else 1.0, (b, h))
    cache.check()
