"""What the paged 4-bit cache says of inputs at the edge: groups that are no numbers, positions
outside the rotary table, padded packed batches, rows that are not held, fused buffers."""

import math

import numpy as np
import pytest
import torch

from oracle import kv4
from test_gpu_kv4 import fc, i32, table_of

pytestmark = pytest.mark.gpu


def tokens(n, H, D, seed, lead=()):
    return torch.randn(*lead, n, H, D, generator=torch.Generator().manual_seed(seed)).cuda()


# ----------------------------------------------------------------------- page bounds
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cuts", [[1] * 20, [7, 1, 12], [3, 5, 12], [8, 12]])
@pytest.mark.parametrize("first", [0, 7])
def test_bounds_with_groups_that_are_no_numbers_do_not_depend_on_the_split(what, cuts, first):
    """A key token's group that is NaN counts as zeros, alone in its call or not; the bounds of
    channels of one sign that have none keep the sign."""
    Hk, D, page, n = 2, 64, 32, 20
    k = tokens(n, Hk, D, 1, (1,)).abs() + 0.5
    k[:, :, 1] *= -1
    k[0, first, :, 3], k[0, 8, 0, 40] = what, what
    table, pages = table_of([n], page)
    got = []
    for parts in ([n], cuts):
        cache, at = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True), 0
        cache.pool.zero_()
        for c in parts:
            cache.append(None, k[:, at:at + c], k[:, at:at + c], table, i32([at]))
            at += c
        got.append((cache.pool, cache.bounds, cache.exponents))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    held = kv4.values(*kv4.quantise(k[0].cpu().numpy()))
    for h in range(Hk):
        want, e = kv4.bounds(np.nan_to_num(held[:, h]))
        assert np.array_equal(got[0][1][table[0, 0], h].cpu().numpy(), want)
        assert int(got[0][2][table[0, 0], h]) == e
    assert (want[1, 32:] < 0).all()  # the last head's second group has none


def test_bounds_of_a_page_without_numbers():
    """Bounds of zero; keys of numbers that come later are within them all the same."""
    Hk, D, page = 1, 64, 16
    k = torch.full((1, 4, Hk, D), math.nan, device="cuda")
    k[0, 2:] = tokens(2, Hk, D, 2) + 5
    table, pages = table_of([4], page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
    for at in (0, 2):
        cache.append(None, k[:, at:at + 2], k[:, at:at + 2], table, i32([at]))
        lo, hi = cache.bounds[table[0, 0], 0].double().cpu().numpy()
        unit = 2.0 ** int(cache.exponents[table[0, 0], 0])
        if at == 0:
            assert not lo.any() and not hi.any()
    held = kv4.values(*kv4.quantise(k[0, 2:, 0].cpu().numpy()))
    assert (lo * unit <= held.min(0)).all() and (hi * unit >= held.max(0)).all()


# ------------------------------------------------------------------- rotary positions
def test_a_position_outside_the_rotary_table_takes_its_nearest_row():
    Hk, D, page = 1, 64, 16
    table, pages = table_of([4], page)
    q, k = tokens(4, 2, D, 3, (1,)), tokens(4, Hk, D, 4, (1,))
    tab = fc().rotary_table(3, D)
    got = []
    for pos in ([[-5, 1, 7, 2 ** 31 - 1]], [[0, 1, 2, 2]]):
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
        cache.pool.zero_()
        out = cache.append(q, k, k, table, i32([0]), rotary=tab, positions=i32(pos))
        got.append((out, cache.pool))
        if pos[0][0] < 0:
            with pytest.raises(fc()._lib.FlashCodecError, match="rotary table"):
                cache.check()
        cache.check()
    assert all(torch.equal(x, y) for x, y in zip(*got))


# -------------------------------------------------------------- padded packed batches
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("front,new,T", [(0, [3, 1, 20], 64), (0, [5, 0, 11], 16), (0, [0, 0, 0], 40), (21, [3, 0, 19], 50),
                                         (16, [1, 15, 16], 48), (3, [2, 2, 2], 9), (0, [16, 16, 0], 33)])
def test_rows_of_no_sequence_in_a_packed_batch(dtype, front, new, T):
    """A captured prefill has a fixed number of rows, more than its sequences need: the others'
    queries are zeros, they ask for no position, and reading gives zeros there."""
    Hq, Hk, D, page, ctx = 4, 2, 64, 16, [5, 16, 31]
    cu = np.concatenate([[front], front + np.cumsum(new)]).astype(int)
    q, k, v = (tokens(T, H, D, 5 + i).to(dtype) for i, H in enumerate((Hq, Hk, Hk)))
    table, pages = table_of([a + b for a, b in zip(new, ctx)], page)
    tab = fc().rotary_table(max(a + b for a, b in zip(new, ctx)), D)  # no row beyond what is held
    pools = []
    for padded in (True, False):
        rows = slice(0, T) if padded else slice(front, int(cu[-1]))
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
        cache.pool.zero_()
        at = i32((cu if padded else cu - front).tolist())
        if padded or cu[-1] > front:
            out = cache.append(q[rows], k[rows], v[rows], table, i32(ctx), cu_seqlens=at, rotary=tab,
                               q_weight=torch.ones(D, device="cuda", dtype=dtype))
        else:
            out = q[rows]
        cache.check()
        pools.append((cache.pool, out))
        if padded:
            got = out
            junk = [torch.full((T, Hk, D), math.nan, device="cuda", dtype=dtype) for _ in range(4)]
            del junk  # what an output of this size may be made of
            gk, gv = cache.read(table, i32(ctx), count=T, cu_seqlens=at, dtype=dtype)
            for x in (gk, gv, out):
                assert (x[: front] == 0).all() and (x[int(cu[-1]):] == 0).all()
            mine = slice(front, int(cu[-1]))
            held = kv4.values(*kv4.quantise(v[mine].float().cpu().numpy()))
            assert torch.equal(gv[mine].cpu(), torch.from_numpy(held).to(dtype))
    cache.check()
    assert torch.equal(pools[0][0], pools[1][0])
    assert torch.equal(got[front:int(cu[-1])], pools[1][1])


def test_tokens_that_a_packed_batch_cuts_off_are_reported():
    Hk, D, page, T = 1, 64, 16, 12
    k = tokens(T, Hk, D, 9)
    table, pages = table_of([40, 40], page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
    for cu in ([0, 5, 13], [0, 40, 41], [0, 12, 13]):
        cache.append(None, k, k, table, i32([0, 0]), cu_seqlens=i32(cu))
        with pytest.raises(fc()._lib.FlashCodecError, match="past what"):
            cache.check()
        cache.read(table, count=T, cu_seqlens=i32(cu))
        with pytest.raises(fc()._lib.FlashCodecError, match="past what"):
            cache.check()
    cache.append(None, k, k, table, i32([0, 0]), cu_seqlens=i32([0, 5, 12]))
    cache.check()


# ------------------------------------------------------------------ rows that are not held
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,page", [(64, 16), (96, 32), (128, 64)])
def test_read_gives_zeros_where_nothing_can_be_read(dtype, D, page):
    """Sequences that are skipped (a negative start), positions past the page table, pages outside
    the pool: zeros, and a bit of the status for the last two."""
    Hk, n = 2, 3 * page
    table, pages = table_of([n] * 4, page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
    x = tokens(n, Hk, D, 10, (4,))
    cache.append(None, x, x, table, i32([0] * 4))
    want = torch.from_numpy(kv4.values(*kv4.quantise(x.cpu().numpy()))).to(dtype).cuda()
    junk = [torch.full((4, n, Hk, D), math.nan, device="cuda", dtype=dtype) for _ in range(4)]
    del junk
    for y in cache.read(table, i32([-1, 0, -2 ** 31, 0]), count=n, dtype=dtype):
        assert (y[[0, 2]] == 0).all() and torch.equal(y[[1, 3]], want[[1, 3]])
    cache.check()
    start = page + 5  # past the last page from token n - start on
    for y in cache.read(table, i32([start, 0, 2 ** 31 - 1, 0]), count=n, dtype=dtype):
        assert torch.equal(y[0, : n - start], want[0, start:]) and (y[0, n - start:] == 0).all()
        assert (y[2] == 0).all() and torch.equal(y[[1, 3]], want[[1, 3]])
    with pytest.raises(fc()._lib.FlashCodecError, match="past what"):
        cache.check()
    bad = table.clone()
    bad[1, 1] = pages
    for y in cache.read(bad, None, count=n, dtype=dtype):
        assert (y[1, page:2 * page] == 0).all() and torch.equal(y[1, :page], want[1, :page])
    with pytest.raises(fc()._lib.FlashCodecError, match="page outside"):
        cache.check()
    # packed, with a sequence that is skipped in the middle
    cu = i32([0, 7, 30, 30 + page, 40 + page])
    for y in cache.read(table, i32([3, -1, 0, 1]), count=40 + page, cu_seqlens=cu, dtype=dtype):
        assert torch.equal(y[:7], want[0, 3:10]) and (y[7:30] == 0).all()
        assert torch.equal(y[30:30 + page], want[2, :page]) and torch.equal(y[30 + page:], want[3, 1:11])
    cache.check()


# ------------------------------------------------------------------------ fused buffers
@pytest.mark.parametrize("order", ["bshd", "bhsd", "hbsd", "sbhd"])
@pytest.mark.parametrize("B,S", [(2, 3), (1, 5), (3, 1)])
def test_queries_written_over_themselves_in_a_fused_buffer(order, B, S):
    """One buffer holds the heads of queries, keys and values, in whatever order of its dims."""
    Hq, Hk, D, page = 4, 2, 64, 16
    H = Hq + 2 * Hk
    x = tokens(S, H, D, 11, (B,)).bfloat16()
    perm = ["bshd".index(c) for c in order]
    back = [order.index(c) for c in "bshd"]
    table, pages = table_of([S] * B, page)
    tab = fc().rotary_table(16, D)
    got = []
    for fused in (False, True):
        y = x.permute(perm).contiguous().permute(back)
        assert y.shape == x.shape
        q, k, v = (y if fused else x.clone()).split([Hq, Hk, Hk], 2)
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
        cache.pool.zero_()
        out = cache.append(q, k, v, table, i32([0] * B), rotary=tab, q_out=q if fused else None)
        got.append((out.contiguous(), cache.pool))
        assert torch.equal(y[:, :, Hq:], x[:, :, Hq:])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_fused_buffers_that_overlap_are_still_refused():
    Hq, Hk, D, page, B, S = 4, 2, 64, 16, 2, 3
    table, pages = table_of([S] * B, page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
    for perm in ([0, 1, 2, 3], [0, 2, 1, 3]):
        y = tokens(S, 9, D, 12, (B,)).permute(perm).contiguous().permute(perm)
        q, out, k = y[:, :, :Hq], y[:, :, 1:1 + Hq], y[:, :, 7:9]
        for a, b, c in ((q, k, out), (y[:, :, 5:9], y[:, :, 3:5], q), (q, y[:, :, 3:5], q)):
            with pytest.raises(ValueError, match="overlaps"):
                cache.append(a, b, k.clone(), table, i32([0] * B), q_out=c)
        cache.append(q, k, k.clone(), table, i32([0] * B), q_out=q)
    # two sets of rows of one buffer that lie between each other in no such order
    y = torch.zeros(4096, device="cuda")
    a = y.as_strided((2, 3, 2, D), (300, 70, 1000, 1))
    b = y.as_strided((2, 3, 2, D), (310, 70, 1000, 1), 5)
    with pytest.raises(ValueError, match="overlaps"):
        cache.append(a, b, b.clone(), table, i32([0] * B), q_out=a)


def test_outputs_of_attend_over_the_queries():
    """Over the queries themselves is fine, whatever pieces the work is cut into; partly over them,
    or rows in one place, is refused."""
    Hk, G, D, page, B = 2, 2, 64, 16, 3
    lens = [9000, 0, 700]
    table, pages = table_of(lens, page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
    for b, n in enumerate(lens):
        if n:
            x = tokens(n, Hk, D, 20 + b, (1,))
            cache.append(None, x, x, table[b:b + 1], i32([0]))
    for S in (1, 4, 9):
        y = tokens(S, 6, D, 13, (B,))
        q = y[:, :, : Hk * G]
        want = cache.attend(q.clone(), table, i32(lens))
        for out in (y[:, :, 1:1 + Hk * G], y[:, :, 2:], q[:1].expand(B, -1, -1, -1) if S == 1 else y[:, :1, :4].expand_as(q)):
            with pytest.raises(ValueError, match="overlaps|one place"):
                cache.attend(q, table, i32(lens), out=out)
        with pytest.raises(ValueError, match="one place"):
            cache.attend(q, table, i32(lens), out=torch.empty(1, S, 1, D, device="cuda").expand_as(q))
        with pytest.raises(ValueError, match="one place"):
            cache.append(q, q[:, :, :Hk], q[:, :, :Hk], table, i32([0] * B),
                         q_out=torch.empty(1, S, 4, D, device="cuda").expand_as(q))
        assert cache.attend(q, table, i32(lens), out=q).data_ptr() == y.data_ptr()
        assert torch.equal(q, want)


def test_batches_of_no_sequence():
    """Nothing to do, and packed rows of no sequence come out as zeros."""
    Hq, Hk, D, page = 4, 2, 64, 16
    cache = fc().PagedInt4Cache(3, Hk, D, page_size=page, bounds=True)
    cache.pool.zero_()
    table, none = i32([]).view(0, 5), i32([])
    q, k = tokens(1, Hq, D, 1, (0,)), tokens(1, Hk, D, 1, (0,))
    assert cache.append(q, k, k, table, none).shape == q.shape
    out, lse = cache.attend(q, table, none, return_lse=True)
    assert out.shape == q.shape and lse.shape == q.shape[:-1]
    assert cache.select(q[:, 0], table, none, 2).shape == (0, Hk, 2)
    assert cache.read(table, none, count=3)[0].shape == (0, 3, Hk, D)
    q, k = tokens(21, Hq, D, 2), tokens(21, Hk, D, 3)
    tab = fc().rotary_table(4, D)
    assert (cache.append(q, k, k, table, none, cu_seqlens=i32([0]), rotary=tab) == 0).all()
    cache.append(None, k, k, table, none, cu_seqlens=i32([0]))
    junk = [torch.full((21, Hk, D), math.nan, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    del junk
    assert all((x == 0).all() for x in cache.read(table, none, count=21, cu_seqlens=i32([0])))
    assert not cache.pool.any()
    cache.check()
