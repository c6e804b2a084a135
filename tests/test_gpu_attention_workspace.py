"""Workspaces of the codec decode attention: calls of different batch sizes on one stream, and
graphs captured on one stream and replayed in any order."""

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


def captured(c, **kw):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, **kw):
        out = attend(c)
    return graph, out


def test_graphs_of_two_sizes_captured_on_one_stream():
    """Replayed in any order, the second one first, and after a larger eager call there."""
    cases = [case(1, 32, 8, 1500, 3), case(4, 32, 8, 700, 4), case(24, 32, 8, 1200, 5)]
    want = [attend(c) for c in cases]  # on the default stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = [captured(c, stream=s) for c in cases[:2]]
    for order in ((1, 0), (0, 1)):
        for i in order:
            graphs[i][1].fill_(torch.nan)
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert torch.equal(graphs[i][1], want[i]), (order, i)
    with torch.cuda.stream(s):
        out = attend(cases[2])
        s.synchronize()
        other = [torch.full((n << 18,), 5, dtype=torch.uint8, device=DEV) for n in range(1, 30)]
        s.synchronize()
    assert torch.equal(out, want[2])
    for i in (1, 0):
        graphs[i][1].fill_(torch.nan)
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1], want[i])
    assert all(bool((x == 5).all()) for x in other)


def test_status_of_captured_calls():
    """A graph that has not run has no status; one that has tells its own, until it is reset."""
    import flashcodec_b200 as fc
    from flashcodec_b200 import _kernels as K
    c = case(1, 32, 8, 1500, 6)
    attend(c)
    dev = c[0].device
    s = torch.cuda.Stream()
    junk = [torch.full((4 << 20,), 77, dtype=torch.uint8, device=DEV) for _ in range(4)]
    del junk
    s.wait_stream(torch.cuda.current_stream())
    graphs = [captured(c, stream=s)[0] for _ in range(2)]
    with torch.cuda.stream(s):
        assert K.attn_status(dev) == 0
        for g in graphs:
            g.replay()
        assert K.attn_status(dev) == 0
        ws = [w for k, w in K._workspaces.items() if k[1] == s.cuda_stream]
        assert len(ws) == 2
        ws[0][:4].view(torch.int32).fill_(9)  # as a launch does whose wait gave up
        assert K.attn_status(dev) == 9 and fc.attention_status(dev, reset=True).value() == 9
        assert fc.attention_status(dev).value() == 0
        ws[1].fill_(77)  # memory that no replay has zeroed
        assert K.attn_status(dev) == 0


def test_captures_do_not_pile_up():
    from flashcodec_b200 import _kernels as K
    c = case(1, 32, 8, 200, 7)
    attend(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(K.KEPT_CAPTURES + 3):
        graph, out = captured(c, stream=s)
    assert sum(k[1] == s.cuda_stream for k in K._workspaces) == K.KEPT_CAPTURES
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(c))
