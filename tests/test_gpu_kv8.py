"""Paged 8-bit KV cache on the GPU against the CPU oracle (oracle/kv8.py).

Stored codes and scales are compared bit for bit: their arithmetic is defined operation by
operation.  Attention is compared with fp64, within u |out| + c M, u half a step of the output type
relative to a value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), M the largest held |value|, and c for
 * the scores: fp32 sums of exact products, up to 32 additions that cut at 2^-23 of a partial sum
   of at most 8 (base 2, scaled): 2^-15, which the weights carry on;
 * the weights: bf16 queries, one fp16 part, half a step of 11 bits: 2^-11; else two parts, 2^-21.
"""

import math

import numpy as np
import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
SLACK = {"fp32": 2.0 ** -15 + 2.0 ** -21, "bf16": 2.0 ** -15 + 2.0 ** -11, "fp16": 2.0 ** -15 + 2.0 ** -21}


def fc():
    import flashcodec_b200
    return flashcodec_b200


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def table_of(lens, page, spare=3, seed=0):
    need = [max(1, -(-n // page)) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([ids.pop() for _ in range(n)])
    return t.cuda(), sum(need) + spare


def new_cache(pages, Hk, D, page):
    cache = fc().PagedInt8Cache(pages, Hk, D, page_size=page)
    cache.codes.fill_(77)
    cache.scales.fill_(math.nan)  # wherever nothing is written
    return cache


def filled(lens, Hk, D, page, seed=0):
    """A cache of random keys and values, and what it holds: (cache, table, [(k, v)])."""
    g = torch.Generator().manual_seed(seed)
    table, pages = table_of(lens, page, seed=seed)
    cache = new_cache(pages, Hk, D, page)
    held = []
    for b, n in enumerate(lens):
        k, v = torch.randn(n, Hk, D, generator=g), torch.randn(n, Hk, D, generator=g)
        v = v * torch.exp(2 * torch.randn(n // 40 + 1, Hk, 1, generator=g)).repeat_interleave(40, 0)[:n]  # scales that differ
        held.append(tuple(kv8.values(*kv8.quantise(x.numpy())) for x in (k, v)))
        if n:
            cache.append(None, k[None].cuda(), v[None].cuda(), table[b:b + 1], i32([0]))
    return cache, table, held


def stored(cache, table, b, n):
    """Codes (n, Hk, D) and scales (runs, Hk) of sequence b, for K and V."""
    P = cache.page_size
    ids = table[b, : -(-n // P)].long()
    out = []
    for i in range(2):
        c = cache.codes[ids, i].transpose(1, 2).flatten(0, 1)[:n]
        s = cache.scales[ids, i].transpose(1, 2).flatten(0, 1)[: -(-n // 16)]
        out.append((c.cpu().numpy(), s.cpu().numpy()))
    return out


def same_bits(got, want):
    (c, s), (cw, sw) = got, want
    assert np.array_equal(s, sw, equal_nan=True)
    ok = np.repeat(~np.isnan(sw), 16, 0)[: len(c)]
    assert np.array_equal(c[ok], cw[ok])


# ------------------------------------------------------------------- append, read
def turned(x, w, cs, interleaved):
    y = x.float().numpy()
    if w is not None:
        y = kv8.head_norm(y, w.float().numpy(), 1e-6)
    return y if cs is None else kv8.rotate(y, cs, interleaved)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D,rot,interleaved,norm,page", [
    (64, 64, False, True, 16), (64, 16, True, False, 32), (96, 96, False, True, 64), (96, 48, True, True, 16),
    (128, 128, False, True, 64), (128, 64, True, False, 128), (128, 0, False, False, 16), (192, 192, False, False, 32),
    (192, 96, False, True, 64), (256, 256, False, True, 16), (256, 128, True, True, 1024)])
def test_append(D, rot, interleaved, norm, page, dtype):
    """Packed prompts, then single tokens, then two at a time: stored bits, queries, and what read gives."""
    dt, Hk, Hq = DT[dtype], 2, 6
    g = torch.Generator().manual_seed(D + rot)
    steps = [[37, 1, 100, 0], [1, 1, 1, 1], [2, 2, 2, 2], [1, 1, 1, 1]]
    total = np.sum(steps, 0).tolist()
    table, pages = table_of(total, page)
    cache = new_cache(pages, Hk, D, page)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dt) if norm else None for _ in range(2)]
    rotary = fc().rotary_table(200, rot, device="cuda") if rot else None
    tab = rotary.cpu().numpy() if rot else None
    lens = np.zeros(4, int)
    all_k, all_v = [[] for _ in range(4)], [[] for _ in range(4)]
    for i, new in enumerate(steps):
        T = sum(new)
        q, k, v = (torch.randn(T, H, D, generator=g).to(dt) for H in (Hq, Hk, Hk))
        k = (k.float() * torch.exp(torch.randn(T, 1, 1, generator=g))).to(dt)
        pos = np.concatenate([lens[b] + np.arange(n) for b, n in enumerate(new)]).astype(int)
        cs = tab[pos] if rot else None
        args = dict(q_weight=None if w[0] is None else w[0].cuda(), k_weight=None if w[1] is None else w[1].cuda(),
                    rotary=rotary, interleaved=interleaved)
        if i == 0:
            got = cache.append(q.cuda(), k.cuda(), v.cuda(), table, i32(lens.tolist()),
                               cu_seqlens=i32([0, *np.cumsum(new).tolist()]), **args)
        else:
            shape = (4, new[0]) if new[0] > 1 else (4,)
            got = cache.append(*(t.cuda().view(*shape, -1, D) for t in (q, k, v)), table, i32(lens.tolist()), **args)
        want = torch.from_numpy(turned(q, w[0], cs, interleaved)).to(dt)
        assert torch.equal(got.cpu().view(T, Hq, D), want)
        kt = turned(k, w[1], cs, interleaved)
        at = 0
        for b, n in enumerate(new):
            all_k[b].append(kt[at:at + n])
            all_v[b].append(v[at:at + n].float().numpy())
            at += n
        lens += new
        for b in range(4):
            for j, x in enumerate((all_k, all_v)):
                same_bits(stored(cache, table, b, lens[b])[j], kv8.quantise(np.concatenate(x[b])))
    cache.check()
    # the values held, from the middle of a run on
    starts = [5, 0, 17, 2]
    n = [int(t - s) for t, s in zip(total, starts)]
    k, v = cache.read(table, i32(starts), count=sum(n) + 3, cu_seqlens=i32([0, *np.cumsum(n).tolist()]), dtype=dt)
    at = 0
    for b in range(4):
        for got, x in ((k, all_k), (v, all_v)):
            want = kv8.values(*kv8.quantise(np.concatenate(x[b])))[starts[b]:]
            assert torch.equal(got[at:at + n[b]].cpu(), torch.from_numpy(want).to(dt))
        at += n[b]
    assert not k[at:].any() and not v[at:].any()  # rows of no sequence
    cache.check()


@pytest.mark.parametrize("seed", range(3))
def test_splits_store_the_same(seed):
    """One call, a token at a time, and pieces of odd sizes."""
    rng = np.random.default_rng(seed)
    n, Hk, D = 75, 2, 64
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n, Hk, D, generator=g) * torch.exp(4 * torch.randn(n, Hk, 1, generator=g))
    v = torch.randn(n, Hk, D, generator=g) * torch.exp(4 * torch.randn(n, Hk, 1, generator=g))
    k[20:30] = 0
    want = [kv8.quantise(x.numpy()) for x in (k, v)]
    cuts = [[0, n], list(range(n + 1)), [0, *sorted(rng.choice(np.arange(1, n), 9, replace=False).tolist()), n]]
    for cut in cuts:
        table, pages = table_of([n], 32, seed=seed)
        cache = new_cache(pages, Hk, D, 32)
        for a, b in zip(cut, cut[1:]):
            cache.append(None, k[None, a:b].cuda(), v[None, a:b].cuda(), table, i32([a]))
        for got, w in zip(stored(cache, table, 0, n), want):
            same_bits(got, w)


@pytest.mark.parametrize("alternate,interleaved", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (128, 64), (192, 192)])
def test_axes(D, rot, alternate, interleaved, dtype):
    """Positions of time, height and width: in a batch of 2 and packed."""
    dt, Hk, Hq, S = DT[dtype], 2, 4, 21
    g = torch.Generator().manual_seed(D)
    half = rot // 2
    axes = fc().rotary_axes((half - 2 * (half // 3), half // 3, half // 3), alternate)
    rotary = fc().rotary_table(500, rot, device="cuda")
    pos = torch.randint(0, 500, (3, 2, S), generator=g, dtype=torch.int32)
    q, k, v = (torch.randn(2, S, H, D, generator=g).to(dt) for H in (Hq, Hk, Hk))
    tab, ax = rotary.cpu().numpy(), axes.cpu().numpy()
    p = pos.numpy().reshape(3, -1)[ax].T  # (T, pairs)
    pair = np.arange(half)
    cs = np.concatenate([tab[p, pair], tab[p, pair + half]], 1)
    want_q = torch.from_numpy(turned(q.flatten(0, 1), None, cs, interleaved)).to(dt)
    want_k = turned(k.flatten(0, 1), None, cs, interleaved).reshape(2, S, Hk, D)
    for packed in (False, True):
        table, pages = table_of([S, S], 16)
        cache = new_cache(pages, Hk, D, 16)
        if packed:
            got = cache.append(q.flatten(0, 1).cuda(), k.flatten(0, 1).cuda(), v.flatten(0, 1).cuda(), table, i32([0, 0]),
                               cu_seqlens=i32([0, S, 2 * S]), rotary=rotary, interleaved=interleaved,
                               positions=pos.flatten(1).cuda(), axes=axes)
        else:
            got = cache.append(q.cuda(), k.cuda(), v.cuda(), table, i32([0, 0]), rotary=rotary, interleaved=interleaved,
                               positions=pos.cuda(), axes=axes)
        assert torch.equal(got.cpu().view(2 * S, Hq, D), want_q)
        for b in range(2):
            same_bits(stored(cache, table, b, S)[0], kv8.quantise(want_k[b]))
        cache.check()
    # one axis for all is the same as no axes
    table, pages = table_of([S, S], 16)
    outs = []
    for kw in (dict(positions=pos[0].cuda()), dict(positions=pos[:1].cuda().contiguous(), axes=torch.zeros_like(axes)),
               dict(positions=pos[:1].cuda().contiguous(), axes=torch.full_like(axes, 7))):  # an axis that is not: the nearest
        cache = new_cache(pages, Hk, D, 16)
        outs.append((cache.append(q.cuda(), k.cuda(), v.cuda(), table, i32([0, 0]), rotary=rotary, interleaved=interleaved, **kw),
                     cache.scales.clone()))
    for o in outs[1:]:
        assert torch.equal(o[0], outs[0][0]) and torch.equal(o[1].nan_to_num(-1), outs[0][1].nan_to_num(-1))


def test_no_numbers():
    """An infinity or a NaN makes its run of 16 tokens NaN, and no other; a run begun anew forgets it."""
    n, Hk, D = 48, 2, 64
    k = torch.randn(n, Hk, D)
    k[20, 1, 3], k[40, 0, 7] = math.inf, math.nan
    table, pages = table_of([n], 16)
    cache = new_cache(pages, Hk, D, 16)
    cache.append(None, k[None].cuda(), k[None].cuda(), table, i32([0]))
    for got, x in zip(cache.read(table, count=n, dtype=torch.float32), (k, k)):
        bad = torch.zeros(n, Hk, dtype=torch.bool)
        bad[16:32, 1] = bad[32:48, 0] = True
        assert got[0].cpu()[bad].isnan().all() and got[0].cpu()[~bad].isfinite().all()
    q = torch.randn(1, 4, D, device="cuda")
    out = cache.attend(q, table, i32([n]))
    assert out.isnan().all()
    out = cache.attend(q, table, i32([16]))  # what is behind the length is not seen
    assert out.isfinite().all()
    good = torch.randn(1, 16, Hk, D).cuda()
    cache.append(None, good, good, table, i32([16]))
    assert cache.read(table, count=32)[0].isfinite().all()
    # a token added to a run that is NaN stays NaN
    cache.append(None, good[:, :1], good[:, :1], table, i32([41]))
    assert cache.read(table, i32([41]), count=1)[0][0, 0, 0].isnan().all()


def test_strides_and_places():
    """Slices of one buffer, heads before tokens, rows off 16-byte boundaries; queries in place."""
    B, S, Hq, Hk, D = 2, 5, 4, 2, 64
    g = torch.Generator().manual_seed(0)
    table, pages = table_of([S, S], 16)
    rotary = fc().rotary_table(64, D, device="cuda")
    buf = torch.randn(B, S, Hq + 2 * Hk, D, generator=g).bfloat16().cuda()
    q, k, v = buf.split([Hq, Hk, Hk], 2)
    want_cache = new_cache(pages, Hk, D, 16)
    want = want_cache.append(q.contiguous(), k.contiguous(), v.contiguous(), table, i32([0, 0]), rotary=rotary)

    def check(*args, **kw):
        cache = new_cache(pages, Hk, D, 16)
        got = cache.append(*args, table, i32([0, 0]), rotary=rotary, **kw)
        assert torch.equal(got, want)
        for b in range(B):
            for x, y in zip(stored(cache, table, b, S), stored(want_cache, table, b, S)):
                same_bits(x, y)
    check(q, k, v)
    check(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)))
    odd = torch.zeros(B, S, Hq + 2 * Hk, D + 1, dtype=buf.dtype, device="cuda")
    odd[..., :D] = buf
    check(*odd[..., :D].split([Hq, Hk, Hk], 2))
    mine = buf.clone()
    q2, k2, v2 = mine.split([Hq, Hk, Hk], 2)
    check(q2, k2, v2, q_out=q2)


def test_bad_tables_and_lengths():
    """Tokens without a page or a row are skipped, and reported; nothing else changes."""
    Hk, D, page = 2, 64, 16
    cache = new_cache(4, Hk, D, page)
    err = fc()._lib.FlashCodecError
    x = torch.randn(2, 3, Hk, D, device="cuda")
    before = cache.codes.clone(), cache.scales.clone()
    cache.append(None, x, x, i32([[0, 9], [-1, 1]]), i32([17, 2]))  # page 9 and page -1
    with pytest.raises(err, match="page outside"):
        cache.check()
    cache.append(None, x, x, i32([[0, 1], [2, 3]]), i32([32, 2 ** 31 - 2]))  # past the table
    with pytest.raises(err, match="past what the page table"):
        cache.check()
    cache.append(None, x, x, i32([[0, 1], [2, 3]]), i32([-1, -5]))  # not in use
    cache.check()
    assert torch.equal(cache.codes, before[0]) and torch.equal(cache.scales.isnan(), before[1].isnan())
    rotary = fc().rotary_table(8, D, device="cuda")
    q = cache.append(x, x, x, i32([[0, 1], [2, 3]]), i32([0, 7]), rotary=rotary)
    with pytest.raises(err, match="rotary table"):
        cache.check()
    assert q.isfinite().all()
    k, _ = cache.read(i32([[0, 7], [2, -3]]), i32([0, 14]), count=20)
    with pytest.raises(err, match="page outside"):
        cache.check()
    assert not k[0, 16:].any() and not k[1, 2:].any()
    k, _ = cache.read(i32([[0]]), i32([14]), count=4)
    with pytest.raises(err, match="past what"):
        cache.check()
    assert not k[0, 2:].any()
    k, _ = cache.read(i32([[0]]), i32([-1]), count=4)
    assert not k.any()
    cache.check()
    # packed rows: those of no sequence, and more than there are
    y = x.flatten(0, 1)
    got = cache.append(y, y, y, i32([[0], [1]]), i32([0, 0]), cu_seqlens=i32([1, 3, 4]))
    assert not got[0].any() and not got[4:].any() and torch.equal(got[1:4], y[1:4])
    cache.check()
    cache.append(y, y, y, i32([[0], [1]]), i32([0, 0]), cu_seqlens=i32([0, 3, 400]))
    with pytest.raises(err, match="past what"):
        cache.check()
    out = cache.attend(torch.randn(1, 4, D, device="cuda"), i32([[77]]), i32([5]))
    with pytest.raises(err, match="page outside"):
        cache.check()
    out = cache.attend(torch.randn(1, 4, D, device="cuda"), i32([[0]]), i32([500]))
    with pytest.raises(err, match="past what"):
        cache.check()
    assert out.shape == (1, 4, D)


def test_no_sequence_and_no_token():
    cache = new_cache(4, 2, 64, 16)
    none = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 2, 64, device="cuda")
    assert cache.append(x, x, x, none, i32([])).shape == (0, 2, 64)
    assert cache.attend(x, none, i32([])).shape == (0, 2, 64)
    assert cache.read(none, count=3)[0].shape == (0, 3, 2, 64)
    y = torch.ones(3, 2, 64, device="cuda")
    assert not cache.append(y, y, y, none, i32([]), cu_seqlens=i32([0])).any()  # rows of no sequence
    assert cache.append(y[None, :0], y[None, :0], y[None, :0], i32([[0]]), i32([0])).shape == (1, 0, 2, 64)
    assert cache.read(i32([[0]]), count=0)[0].shape == (1, 0, 2, 64)
    cache.check()


# ------------------------------------------------------------------------ attention
def check_attend(lens, Hq, Hk, D, page, dtype, Sq=1, scale=None, seed=0, amp=1.0):
    cache, table, held = filled(lens, Hk, D, page, seed)
    g = torch.Generator().manual_seed(seed + 1)
    lead = (len(lens), Sq) if Sq > 1 else (len(lens),)
    q = (amp * torch.randn(*lead, Hq, D, generator=g)).to(DT[dtype])
    out, lse = cache.attend(q.cuda(), table, i32(lens), scale=scale, return_lse=True)
    cache.check()
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == q.shape[:-1]
    s = D ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        want, wl = kv8.attention(q[b].float().numpy().reshape(Sq, Hq, D), *held[b], s)
        got = out[b].double().cpu().numpy().reshape(Sq, Hq, D)
        top = np.abs(held[b][1]).max() if n else 0.0
        err, lim = np.abs(got - want), HALF_STEP[dtype] * np.abs(want) + SLACK[dtype] * top
        assert np.isfinite(got).all() and (err <= lim).all(), f"{n}: {(err / np.maximum(lim, 1e-30)).max():.2f} of the bound"
        gl = lse[b].double().cpu().numpy().reshape(Sq, Hq)
        none = np.isneginf(wl)
        assert np.isneginf(gl[none]).all()
        assert (np.abs(gl[~none] - wl[~none]) <= 2.0 ** -15 + 2.0 ** -21 * np.abs(wl[~none])).all()
    return cache, table, q


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_attend(D, page, dtype):
    check_attend([1, 15, 16, 17, 31, 33, 0, 130, 513, 700], 8, 2, D, page, dtype)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (8, 8), (14, 2), (9, 1), (16, 1), (40, 2)])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_groups(Hq, Hk, D, dtype):
    check_attend([70, 3, 300], Hq, Hk, D, 32, dtype)


@pytest.mark.parametrize("Sq", [2, 3, 4, 7])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "bf16"), (128, "fp16"), (192, "fp32")])
def test_several_queries(Sq, D, dtype):
    """The newest tokens of sequences, some shorter than their number of queries (rows that see none)."""
    check_attend([1, 2, 5, 40, 257, 900], 8, 2, D, 64, dtype, Sq=Sq)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 3.0])
def test_scales(scale):
    check_attend([100, 333], 4, 2, 64, 16, "fp32", scale=scale, amp=0.2)


@pytest.mark.parametrize("amp", [1e-30, 1e-6, 1e4, 1e30])
def test_sizes_of_queries(amp):
    """Queries of any size: the softmax of the scaled scores is what it is for those of size one."""
    cache, table, held = filled([200, 77], 2, 64, 16)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3))
    want = cache.attend(q.cuda(), table, i32([200, 77]))
    two = 2.0 ** round(math.log2(amp))  # a power of two: the same bits
    got = cache.attend((q * two).cuda(), table, i32([200, 77]), scale=0.125 / two)
    assert torch.equal(got, want)


def test_long_and_many():
    check_attend([20000], 8, 2, 128, 64, "bf16")
    rng = np.random.default_rng(0)
    check_attend([int(n) for n in rng.integers(0, 200, 400)], 2, 1, 64, 16, "bf16")


def test_flat_weights_of_a_long_sequence():
    """Sums of 131072 values with a mean, of equal weights: nothing is cut off on the way."""
    n, D = 131072, 64
    table, pages = table_of([n], 1024)
    cache = fc().PagedInt8Cache(pages, 1, D, page_size=1024)
    v = torch.full((1, n, 1, D), 3.0, device="cuda")
    v[:, n // 2:] = -3.0
    v[:, n // 2:, :, :8] = 3.0
    cache.append(None, torch.zeros_like(v), v, table, i32([0]))
    held = cache.read(table, count=n, dtype=torch.float32)[1][0].double().mean(0)
    for dtype in ("fp32", "bf16"):
        out = cache.attend(torch.randn(1, 2, D, device="cuda").to(DT[dtype]), table, i32([n]))[0]
        err = (out.double() - held).abs().max().item()
        # equal weights of one are exact; sums of a warp's chunks are rounded fp32
        assert err <= HALF_STEP[dtype] * 3.05 + 2.0 ** -15


def test_places_of_queries_and_outputs():
    cache, table, q = check_attend([50, 9], 4, 2, 64, 16, "bf16", Sq=3)
    want = cache.attend(q.cuda(), table, i32([50, 9]))
    buf = torch.zeros(2, 3, 8, 64 + 8, dtype=torch.bfloat16, device="cuda")[..., 1:65]
    view = buf[:, :, 2:6]
    view.copy_(q)
    assert torch.equal(cache.attend(view, table, i32([50, 9])), want)
    assert cache.attend(view, table, i32([50, 9]), out=view) is view and torch.equal(view, want)
    assert not buf[:, :, :2].any() and not buf[:, :, 6:].any()
    for out in (buf[:, :, 3:7], torch.zeros(1, 1, 1, 64, dtype=buf.dtype, device="cuda").expand(2, 3, 4, 64)):
        with pytest.raises(ValueError, match="overlaps|one place"):
            cache.attend(buf[:, :, 2:6], table, i32([50, 9]), out=out)


def test_streams_and_graphs():
    """Captured steps of two sizes replayed in turn next to eager ones; a graph follows lengths and tables."""
    cases = []
    for lens, seed in (([40, 3], 0), ([700] * 9, 1)):
        cache, table, _ = filled(lens, 2, 128, 64, seed)
        n = len(lens)
        q = torch.randn(n, 8, 128, device="cuda").bfloat16()
        cases.append([cache, table, i32(lens), q, cache.attend(q, table, i32(lens))])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [c.attend(q, t, n) for c, t, n, q, _ in cases]
    torch.cuda.synchronize()
    assert all(torch.equal(o, c[4]) for o, c in zip(outs, cases))
    graphs, outs = [], []
    for c, t, n, q, _ in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c.attend(q, t, n))
    for order in ((0, 1), (1, 0), (1, 1)):
        for i in order:
            outs[i].zero_()
            graphs[i].replay()
            c, t, n, q, want = cases[1 - i]
            assert torch.equal(c.attend(q, t, n), want)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], cases[i][4])
    c, t, n, q, _ = cases[1]
    n.copy_(i32([5] * 9))
    want = c.attend(q, t, i32([5] * 9))
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], want)


def test_a_captured_step():
    """Append and attend as one graph, replayed with new tokens, are the eager steps."""
    Hk, Hq, D, page, B = 2, 4, 64, 16, 3
    lens0 = [14, 15, 40]
    rotary = fc().rotary_table(100, D, device="cuda")
    xs = [tuple(torch.randn(B, H, D, device="cuda").bfloat16() for H in (Hq, Hk, Hk)) for _ in range(4)]

    def begin():
        cache, table, _ = filled(lens0, Hk, D, page)
        wide = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
        wide[:, : table.shape[1]] = table
        free = [p for p in range(cache.num_pages) if p not in table.flatten().tolist()]
        for b in range(B):
            wide[b, -(-lens0[b] // page)] = free.pop()
        return cache, wide, i32(lens0)
    want = []
    cache, table, lens = begin()
    for q, k, v in xs:
        y = cache.append(q, k, v, table, lens, rotary=rotary)
        lens = lens + 1
        want.append(cache.attend(y, table, lens))
    cache.check()
    bits = [stored(cache, table, b, lens0[b] + 4) for b in range(B)]
    cache, table, lens = begin()
    slot = [t.clone() for t in xs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cache.append(*slot, table, lens, rotary=rotary)
        lens.add_(1)
        out = cache.attend(y, table, lens)
    for i, x in enumerate(xs):
        for s, t in zip(slot, x):
            s.copy_(t)
        graph.replay()
        assert torch.equal(out, want[i])
    cache.check()
    for b in range(B):
        for x, y in zip(stored(cache, table, b, lens0[b] + 4), bits[b]):
            same_bits(x, y)


def test_a_prompt_in_chunks():
    """The operators as a serving loop uses them: chunks are appended, the prefix is read back and
    attended to together with the chunk, then tokens are decoded; against fp64 over the values held."""
    Hk, Hq, D, page = 2, 8, 128, 64
    prompts, chunk = [150, 70, 333], 100
    table, pages = table_of([n + 4 for n in prompts], page)
    cache = new_cache(pages, Hk, D, page)
    rotary = fc().rotary_table(512, D, device="cuda")
    g = torch.Generator().manual_seed(0)
    lens = [0, 0, 0]
    while lens != prompts:
        new = [min(chunk, p - n) for p, n in zip(prompts, lens)]
        x = [torch.randn(sum(new), H, D, generator=g).bfloat16().cuda() for H in (Hq, Hk, Hk)]
        c = i32([0, *np.cumsum(new).tolist()])
        q = cache.append(*x, table, i32(lens), cu_seqlens=c, rotary=rotary)
        lens = [a + b for a, b in zip(lens, new)]
        ck = i32([0, *np.cumsum(lens).tolist()])
        k, v = cache.read(table, count=sum(lens), cu_seqlens=ck)
        out = fc().prompt_attention(q, k, v, c, ck)
        a = b = 0
        for n, m in zip(new, lens):
            if n:
                want, _ = kv8.attention(q[a:a + n].float().cpu().numpy(), k[b:b + m].float().cpu().numpy(),
                                        v[b:b + m].float().cpu().numpy(), D ** -0.5)
                top = v[b:b + m].abs().max().item()
                err = np.abs(out[a:a + n].double().cpu().numpy() - want)
                assert (err <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -12) * top).all()
            a, b = a + n, b + m
    for _ in range(3):
        x = [torch.randn(3, H, D, generator=g).bfloat16().cuda() for H in (Hq, Hk, Hk)]
        q = cache.append(*x, table, i32(lens), rotary=rotary)
        lens = [n + 1 for n in lens]
        out = cache.attend(q, table, i32(lens))
        for b, n in enumerate(lens):
            k, v = (t[0].cpu().numpy() for t in cache.read(table[b:b + 1], count=n, dtype=torch.float32))
            want, _ = kv8.attention(q[b:b + 1].float().cpu().numpy(), k, v, D ** -0.5)
            err = np.abs(out[b].double().cpu().numpy() - want[0])
            assert (err <= 2.0 ** -8 * np.abs(want[0]) + SLACK["bf16"] * np.abs(v).max()).all()
    cache.check()


@pytest.mark.parametrize("bits", [4, 8])
def test_the_serving_example(bits):
    """Prompts by prompt_attention, steps on either cache: the last dense step differs from the attention
    computed from the values held by bf16's roundings (norms of a head's outputs: half a step, 2^-8, at most)."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "paged_decode.py"
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.run(layers=2, steps=5, prompts=(37, 5, 300), bits=bits) < 2.0 ** -7


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_a_large_value_of_no_weight(dtype):
    """A token whose values are 2^16 times larger and whose weight is nothing costs the others no bits: bounds
    with M the largest |value| that has a weight."""
    n, D = 300, 64
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(n, 1, D, generator=g), torch.randn(n, 1, D, generator=g)
    q = torch.ones(1, 2, D)
    k[40:56] = -40.0  # a run that no query attends to: scores of -320, weights of e^-300
    v[40:56] *= 2.0 ** 16
    table, pages = table_of([n], 16)
    cache = new_cache(pages, 1, D, 16)
    cache.append(None, k[None].cuda(), v[None].cuda(), table, i32([0]))
    held = tuple(kv8.values(*kv8.quantise(x.numpy())) for x in (k, v))
    out = cache.attend(q.to(DT[dtype]).cuda(), table, i32([n]))
    want, _ = kv8.attention(q.numpy(), *held, D ** -0.5)
    rest = np.concatenate([held[1][:40], held[1][56:]])
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= HALF_STEP[dtype] * np.abs(want) + SLACK[dtype] * np.abs(rest).max()).all()
