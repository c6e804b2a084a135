"""Workspaces of the codec decode attention: calls of different batch sizes on one stream."""

import pytest
import torch

import bench
from test_gpu_attention import DEV, build, check_close, oracle_attention

pytestmark = pytest.mark.gpu


def case(B, Hq, Hk, blocks, seed, mode="jpeg"):
    k, v, q = bench.synth_case(B, Hq, Hk, 8 * blocks + 5, 128, 0.95, seed, device=DEV, dtype=torch.bfloat16)
    return q, *build(mode, dict(keep_freqs=4, quant_bits=8) if mode == "jpeg" else {}, k, v)


def attend(c):
    import flashcodec_b200 as fc
    return fc.codec_decode_attention(*c)


@pytest.mark.parametrize("mode", ["jpeg", "png"])
@pytest.mark.parametrize("Hq,Hk,B", [(32, 8, 10), (32, 2, 24)])
def test_batches_of_different_sizes_share_a_stream(mode, Hq, Hk, B):
    """One long sequence and then more than 64 (sequence, head group)s: what a call leaves behind in
    the workspace is not the next one's arrival counters."""
    few, many = case(1, Hq, Hk, 1500, 1, mode), case(B, Hq, Hk, 400, 2, mode)
    s = torch.cuda.Stream()  # no workspace yet
    s.wait_stream(torch.cuda.current_stream())
    out = None
    with torch.cuda.stream(s):
        for c in (many, few, many, few, many):
            del out
            junk = [torch.full_like(c[0], torch.nan) for _ in range(8)]
            del junk  # what the output's memory held before
            out = attend(c)
            s.synchronize()
            check_close(out, oracle_attention(*c), torch.bfloat16)
