"""CUDA graphs of the paged 4-bit cache's calls: several graphs, captured on one stream without
a warm-up there, replayed in any order, next to eager calls that need larger workspaces."""

import pytest
import torch

pytestmark = pytest.mark.gpu

D, PAGE, HK, G = 64, 16, 2, 2


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """B sequences in a cache of their own, and a step of select and attend over them."""

    def __init__(self, B, n, seed, d=D):
        import flashcodec_b200 as fc
        g = torch.Generator().manual_seed(seed)
        lens = [n + 37 * b for b in range(B)]
        width = -(-max(lens) // PAGE)
        self.table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).cuda()
        self.cache = fc.PagedInt4Cache(B * width, HK, d, page_size=PAGE, bounds=True)
        k, v = torch.randn(2, B, max(lens), HK, d, generator=g).cuda()
        self.cache.append(None, k, v, self.table, i32([0] * B))
        self.lens, self.q = i32(lens), torch.randn(B, HK * G, d, generator=g).cuda()

    def step(self):
        pages = self.cache.select(self.q, self.table, self.lens, 9)
        return (pages, self.cache.attend(self.q, self.table, self.lens),
                self.cache.attend(self.q, self.table, self.lens, selected=pages))


def captured(batch, **kw):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, **kw):
        out = batch.step()
    return graph, out


def same(got, want):
    return all(torch.equal(x, y) for x, y in zip(got, want))


def test_graphs_of_two_sizes_replayed_in_any_order():
    """Captured one after the other on the same stream, which has run nothing before; the second
    one is replayed first."""
    small, large = Batch(2, 3000, 1), Batch(9, 2000, 2)
    want = [[x.clone() for x in b.step()] for b in (small, large)]  # on the default stream
    s = torch.cuda.Stream()
    graphs = [captured(b, stream=s) for b in (small, large)]
    for order in ((1, 0), (0, 1), (1, 1, 0)):
        for i in order:
            for x in graphs[i][1]:
                x.fill_(-7)
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert same(graphs[i][1], want[i]), (order, i)


def test_replays_after_a_larger_eager_call_leave_other_memory_alone():
    """Eager calls on the capture's stream outgrow its workspaces (more sequences for select, a
    wider head for attend); what is allocated then is not what the replays write to."""
    small, large, wide = Batch(1, 3000, 3), Batch(9, 2000, 4), Batch(3, 1500, 5, d=128)
    want = [[x.clone() for x in b.step()] for b in (small, large, wide)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        small.step()
        s.synchronize()
    graph, out = captured(small, stream=s)
    with torch.cuda.stream(s):
        for b, w in ((large, want[1]), (wide, want[2])):
            assert same(b.step(), w)
        s.synchronize()
        # whatever the allocator has free of the sizes of such workspaces
        other = [torch.full((n,), 5, dtype=torch.uint8, device="cuda")
                 for n in (1 << 20, 2 << 20, 3 << 20, 5 << 20, 10 << 20, 20 << 20) for _ in range(4)]
        s.synchronize()
    for _ in range(3):
        for x in out:
            x.fill_(-7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want[0])
    assert all(bool((x == 5).all()) for x in other)
    with torch.cuda.stream(s):
        assert same(large.step(), want[1])
    torch.cuda.synchronize()


def test_two_graphs_replayed_on_two_streams():
    a, b = Batch(4, 2500, 6), Batch(5, 2300, 7)
    want = [[x.clone() for x in t.step()] for t in (a, b)]
    graphs = [captured(t) for t in (a, b)]  # on one stream
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert same(out, w)
    for t in (a, b):
        t.cache.check()
