"""Paged 4-bit KV cache on the GPU against the CPU oracle (oracle/kv4.py).

Stored codes, scales, bounds and selected pages are compared bit for bit: their
arithmetic is defined operation by operation.  Attention is compared with fp64.
Its bounds, with u the unit roundoff of the output type and M the largest held
|value|, are |error| <= 2 u |out| + c M, where c M stands for
 * bf16 queries: weights of 16-bit significands of 11 bits, rounded twice
   (2^-10), and scores whose fp32 sums carry an offset of 1032 per code
   (below 2^-11 of the weights): c = 2^-9;
 * fp16 queries: two 11-bit parts per weight; c = 2^-13 for the scores' fp32 sums;
 * fp32 queries: c = 1e-5, the library's fp32 attention bound.
"""

import math

import numpy as np
import pytest
import torch

from oracle import kv4

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -9, "fp16": 2.0 ** -12}
SLACK = {"fp32": 1e-5, "bf16": 2.0 ** -9, "fp16": 2.0 ** -13}


def fc():
    import flashcodec_b200
    return flashcodec_b200


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def table_of(lens, page, spare=3, seed=0):
    """A shuffled page table for sequences of `lens` tokens, and the pool's size."""
    need = [max(1, -(-n // page)) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([ids.pop() for _ in range(n)])
    return t.cuda(), sum(need) + spare


def filled(lens, Hk, D, page, seed=0, bounds=False, garbage=True):
    """A cache of random keys and values, and what it holds: (cache, table, [(k, v)])."""
    g = torch.Generator().manual_seed(seed)
    table, pages = table_of(lens, page, seed=seed)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=bounds)
    if garbage:
        cache.pool.fill_(255)  # NaN scales wherever nothing is written
    held = []
    for b, n in enumerate(lens):
        k = torch.randn(n, Hk, D, generator=g) * torch.exp(torch.randn(Hk, D, generator=g))
        v = torch.randn(n, Hk, D, generator=g)
        held.append(tuple(kv4.values(*kv4.quantise(x.numpy())) for x in (k, v)))
        if n:
            cache.append(None, k[None].cuda(), v[None].cuda(), table[b:b + 1], i32([0]))
    return cache, table, held


def near(got, want, dtype, top, what=""):
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    lim = 2 * UNIT[dtype] * np.abs(want) + SLACK[dtype] * top
    assert np.isfinite(got).all(), what
    assert (err <= lim).all(), f"{what}: {err.max():.3e} over {lim.flat[err.argmax()]:.3e}"


# ------------------------------------------------------------------- append, read
def turned(x, w, eps, cs, interleaved):
    y = x.float().numpy()
    if w is not None:
        y = kv4.head_norm(y, w.float().numpy(), eps)
    return y if cs is None else kv4.rotate(y, cs.numpy(), interleaved)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,page,R,interleaved,norm,S", [
    (128, 64, 128, False, True, 1), (128, 16, 64, True, True, 5), (64, 32, 16, False, False, 33),
    (64, 16, 64, True, True, 16), (96, 32, 96, False, True, 40), (96, 16, 48, False, False, 2),
    (192, 64, 192, True, True, 19), (256, 128, 128, False, True, 70), (256, 16, 0, False, False, 1),
    (128, 256, 32, False, False, 300)])
def test_append_holds_the_oracles_bits(dtype, D, page, R, interleaved, norm, S):
    Hq, Hk, ctx = 6, 3, [0, 15, page - 1, 2 * page + 5]
    g = torch.Generator().manual_seed(D + S)
    table, pages = table_of([n + S for n in ctx], page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
    cache.pool.fill_(255)
    old = [torch.randn(n, Hk, D, generator=g) for n in ctx]
    for b, x in enumerate(old):
        if len(x):
            cache.append(None, x[None].cuda(), x[None].cuda() * 2, table[b:b + 1], i32([0]))
    q, k, v = (torch.randn(4, S, H, D, generator=g).to(DT[dtype]) for H in (Hq, Hk, Hk))
    v[0, 0, 0, :32] = 0  # a group of zeros
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(DT[dtype]) if norm else None for _ in "qk")
    tab = fc().rotary_table(1000, R) if R else None
    out = cache.append(q.cuda(), k.cuda(), v.cuda(), table, i32(ctx),
                       q_weight=wq.cuda() if norm else None, k_weight=wk.cuda() if norm else None,
                       rotary=tab, interleaved=interleaved)
    for b, n in enumerate(ctx):
        cs = tab[n:n + S].cpu() if R else None
        want = torch.from_numpy(turned(q[b], wq, 1e-6, cs, interleaved)).to(DT[dtype])
        assert torch.equal(out[b].cpu(), want)
        ks = kv4.values(*kv4.quantise(turned(k[b], wk, 1e-6, cs, interleaved)))
        vs = kv4.values(*kv4.quantise(v[b].float().numpy()))
        o = kv4.values(*kv4.quantise(old[b].numpy()))
        ks, vs = np.concatenate([o, ks]), np.concatenate([kv4.values(*kv4.quantise(old[b].numpy() * 2)), vs])
        gk, gv = cache.read(table[b:b + 1], count=n + S, dtype=torch.float32)
        assert np.array_equal(gk[0].cpu().numpy(), ks) and np.array_equal(gv[0].cpu().numpy(), vs)
        for p in range(-(-(n + S) // page)):
            for h in range(Hk):
                bd, e = kv4.bounds(ks[p * page:(p + 1) * page, h])
                i = int(table[b, p])
                assert np.array_equal(cache.bounds[i, h].cpu().numpy(), bd)
                assert int(cache.exponents[i, h]) == e
    cache.check()


def test_append_against_the_formula_in_64_bits():
    """Norm and rotation as written on paper: fp32 rounding of a few operations apart."""
    D, R, S = 128, 64, 9
    g = torch.Generator().manual_seed(3)
    table, pages = table_of([S], 16)
    cache = fc().PagedInt4Cache(pages, 1, D, page_size=16)
    q, k = torch.randn(1, S, 2, D, generator=g), torch.randn(1, S, 1, D, generator=g)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    tab = fc().rotary_table(64, R, base=500.0)
    out = cache.append(q.cuda(), k.cuda(), k.cuda(), table, i32([0]), q_weight=w.cuda(), rotary=tab)
    x = q[0].double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
    a = torch.arange(S)[:, None] * 500.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    z = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * torch.polar(torch.ones_like(a), a)[:, None]
    want = torch.cat([z.real, z.imag, x[..., R:]], -1)
    # 8 roundings in the sum of squares, 4 in the norm, the table and 3 in the rotation, below 24 u
    assert (out[0].cpu().double() - want).abs().max() <= 24 * 2.0 ** -24 * want.abs().max()


@pytest.mark.parametrize("cuts", [[1] * 37, [5, 11, 1, 20], [37], [16, 16, 5]])
def test_stored_bits_do_not_depend_on_the_split(cuts):
    Hk, D, page, n = 2, 64, 32, 37
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(1, n, Hk, D, generator=g).cuda(), torch.randn(1, n, Hk, D, generator=g).cuda()
    table, pages = table_of([n], page)
    w, tab = torch.ones(D, device="cuda"), fc().rotary_table(64, D)
    got = []
    for parts in ([n], cuts):
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
        cache.pool.zero_()
        at = 0
        for c in parts:
            cache.append(None, k[:, at:at + c], v[:, at:at + c], table, i32([at]), k_weight=w, rotary=tab)
            at += c
        got.append((cache.pool, cache.bounds, cache.exponents))
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_append_packed_equals_each_sequence_alone():
    Hq, Hk, D, page = 4, 2, 128, 16
    new, ctx = [1, 0, 40, 3, 17, 0, 1], [0, 9, 5, 15, 16, 3, 31]
    g = torch.Generator().manual_seed(7)
    T = sum(new)
    q, k, v = (torch.randn(T, H, D, generator=g).bfloat16().cuda() for H in (Hq, Hk, Hk))
    cu = np.concatenate([[0], np.cumsum(new)])
    table, pages = table_of([a + b for a, b in zip(new, ctx)], page)
    pos = torch.randperm(T, generator=g).to(torch.int32).cuda()
    tab = fc().rotary_table(T, 32)
    pools = []
    for packed in (True, False):
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
        cache.pool.zero_()
        if packed:
            out = cache.append(q, k, v, table, i32(ctx), cu_seqlens=i32(cu.tolist()), rotary=tab, positions=pos)
        else:
            for b, n in enumerate(new):
                if n:
                    s = slice(int(cu[b]), int(cu[b + 1]))
                    one = cache.append(q[None, s], k[None, s], v[None, s], table[b:b + 1], i32(ctx[b:b + 1]),
                                       rotary=tab, positions=pos[None, s].contiguous())
                    assert torch.equal(one[0], out[s])
        pools.append(cache.pool)
        kk, vv = cache.read(table, i32(ctx), count=T, cu_seqlens=i32(cu.tolist()), dtype=torch.float32)
        assert np.array_equal(vv.cpu().numpy(), kv4.values(*kv4.quantise(v.float().cpu().numpy())))
    assert torch.equal(*pools)


def test_strides_alignment_and_in_place():
    """Rows that are not 16-byte aligned, other orders of the dims, and q written over itself."""
    B, S, Hq, Hk, D, page = 2, 3, 4, 2, 64, 16
    g = torch.Generator().manual_seed(9)
    table, pages = table_of([S] * B, page)
    base = [torch.randn(B, S, H, D, generator=g).bfloat16().cuda() for H in (Hq, Hk, Hk)]
    tab = fc().rotary_table(16, D)
    want = None
    for way in ("plain", "odd", "bhsd", "fused"):
        q, k, v = (x.clone() for x in base)
        if way == "odd":
            q, k, v = (torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
                       for x in base)
        elif way == "bhsd":
            q, k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in base)
        elif way == "fused":
            q, k, v = torch.cat(base, 2).split([Hq, Hk, Hk], 2)
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page)
        cache.pool.zero_()
        out = cache.append(q, k, v, table, i32([0, 0]), rotary=tab, q_out=None if way == "plain" else q)
        got = (out.clone(), cache.pool.clone())
        kk = torch.empty(B, Hk, S, D, dtype=torch.float32, device="cuda").transpose(1, 2)
        if want is None:
            want = got
        assert all(torch.equal(x, y) for x, y in zip(got, want)), way
        del kk


def test_values_that_are_not_numbers_stay_in_their_group():
    Hk, D, page, n = 2, 64, 16, 20
    g = torch.Generator().manual_seed(11)
    k, v = torch.randn(1, n, Hk, D, generator=g), torch.randn(1, n, Hk, D, generator=g)
    v[0, 4, 0, 3], k[0, 7, 1, 40] = math.nan, math.inf
    table, pages = table_of([n], page)
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
    cache.append(None, k.cuda(), v.cuda(), table, i32([0]))
    gk, gv = (x[0].cpu().numpy() for x in cache.read(table, count=n, dtype=torch.float32))
    wk, wv = (kv4.values(*kv4.quantise(x[0].numpy())) for x in (k, v))
    assert np.array_equal(gk, wk, equal_nan=True) and np.array_equal(gv, wv, equal_nan=True)
    assert np.isnan(gv).sum() == 32 and np.isnan(gk).sum() == 32
    # attention: the first head is NaN in the value's group alone, the second everywhere
    out = cache.attend(torch.ones(1, 2, D, device="cuda"), table, i32([n]))[0].cpu()
    assert out[0, :32].isnan().all() and not out[0, 32:].isnan().any() and out[1].isnan().all()
    # ... and not at all for sequences that end before them
    out = cache.attend(torch.ones(1, 2, D, device="cuda"), table, i32([4]))
    assert not out.isnan().any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_values_that_are_not_numbers_do_not_reach_queries_that_do_not_see_them(dtype):
    """The last of 4 drafted tokens is NaN in keys and values; the earlier queries never see it."""
    Hk, G, D, page, n, Sq = 2, 2, 64, 32, 45, 4
    cache, table, held = filled([n - 1], Hk, D, page)
    table = torch.cat([table, table], 1)[:, :2]
    bad = torch.full((1, Hk, D), math.nan, device="cuda")
    cache.append(None, bad, bad, table, i32([n - 1]))
    q = torch.randn(1, Sq, Hk * G, D, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    q[0, 1, 0] = math.nan  # nor does a query that is no number reach its neighbours
    out = cache.attend(q.cuda(), table, i32([n]))[0]
    assert out[3].isnan().all() and out[1, 0].isnan().all()
    for s in range(3):
        for h in range(Hk):
            rows = slice(h * G + (s == 1 and h == 0), (h + 1) * G)
            k, v = (x[: n - Sq + 1 + s, h] for x in held[0])
            want, _ = kv4.attend(q[0, s, rows].float().numpy(), k, v)
            near(out[s, rows], want, dtype, np.abs(v).max(), (s, h))


# ------------------------------------------------------------------------- attend
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,page,Hk,G,Sq", [
    (128, 64, 2, 4, 1), (128, 16, 1, 1, 1), (64, 32, 2, 7, 1), (64, 16, 3, 8, 2), (96, 32, 2, 3, 1),
    (192, 16, 1, 2, 3), (256, 128, 1, 4, 1), (128, 32, 1, 16, 1), (128, 64, 2, 4, 5), (256, 16, 1, 12, 3)])
def test_attend(dtype, D, page, Hk, G, Sq):
    lens = [0, 1, 2, 15, 16, 17, page, page + 1, 3 * page - 1, 700]
    cache, table, held = filled(lens, Hk, D, page, seed=D + G)
    q = torch.randn(len(lens), Sq, Hk * G, D, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    out, lse = cache.attend(q.cuda(), table, i32(lens), return_lse=True)
    if Sq == 1:
        assert torch.equal(cache.attend(q[:, 0].cuda(), table, i32(lens)), out[:, 0])
    for b, n in enumerate(lens):
        k, v = held[b]
        for s in range(Sq):
            seen = max(0, n - (Sq - 1 - s))
            for h in range(Hk):
                rows = slice(h * G, (h + 1) * G)
                want, wl = kv4.attend(q[b, s, rows].float().numpy(), k[:seen, h], v[:seen, h])
                near(out[b, s, rows], want, dtype, np.abs(v[:seen, h]).max() if seen else 1.0, (b, s, h))
                got = lse[b, s, rows].double().cpu().numpy()
                if not seen:
                    assert (got == -np.inf).all()
                else:
                    assert (np.abs(got - wl) <= SLACK[dtype] * (1 + np.abs(wl))).all()
    cache.check()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attend_many_splits(dtype):
    """One long sequence next to short ones: the work of one is spread over many blocks."""
    lens, Hk, G, D = [9000, 3, 130], 2, 4, 128
    cache, table, held = filled(lens, Hk, D, 64, seed=3)
    q = 3 * torch.randn(3, Hk * G, D, generator=torch.Generator().manual_seed(2)).to(DT[dtype])
    out = cache.attend(q.cuda(), table, i32(lens))
    again = cache.attend(q.cuda(), table, i32(lens))
    assert torch.equal(out, again)
    for b in range(3):
        k, v = held[b]
        for h in range(Hk):
            want, _ = kv4.attend(q[b, h * G:(h + 1) * G].float().numpy(), k[:, h], v[:, h])
            near(out[b, h * G:(h + 1) * G], want, dtype, np.abs(v).max(), (b, h))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,G,page", [(128, 2, 64), (64, 2, 32), (128, 12, 64)])
def test_flat_attention_over_long_sequences(dtype, D, G, page):
    """Equal weights over 131072 tokens in a batch so large that a warp takes 32768 of them:
    the output is a mean, 1 / 360 of the values.  Beside its rounding it may be off by what
    the sums lose (2^-16 of a code's step, at most M / 7), by the roundings of the weights
    times scales (2^-11 each, 6 standard deviations of their mean) and by those of the fp32
    sums of the weights (2^-20)."""
    n, B = 131072, 450
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None].contiguous()
    cache = fc().PagedInt4Cache(n // page, 1, D, page_size=page)
    v = torch.randn(1, n, 1, D, generator=torch.Generator().manual_seed(5)).cuda()
    cache.append(None, torch.zeros_like(v), v, table, i32([0]))
    held = cache.read(table, count=n, dtype=torch.float32)[1][0, :, 0].double()
    want, top = held.mean(0).cpu().numpy(), float(held.abs().max())
    out = cache.attend(torch.zeros(B, G, D, dtype=DT[dtype], device="cuda"), table.repeat(B, 1).contiguous(),
                       torch.full((B,), n, dtype=torch.int32, device="cuda"))
    err = np.abs(out.double().cpu().numpy() - want).max((0, 1))
    lim = 2 * UNIT[dtype] * np.abs(want) + 2.0 ** -16 * top / 7 + 6 * 2.0 ** -11 / n ** 0.5 + 2.0 ** -20 * top
    assert (err <= lim).all(), f"{err.max():.2e} over {lim[err.argmax()]:.2e}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kscale,vscale", [(1e-4, 1e-4), (40.0, 1e-3), (1.0, 3e3), (30.0, 1e4)])
def test_attend_ranges(dtype, kscale, vscale):
    """Tiny and huge keys and values: a sharp softmax, scales near both ends of fp16."""
    n, D = 300, 128
    g = torch.Generator().manual_seed(4)
    k, v = kscale * torch.randn(1, n, 1, D, generator=g), torch.randn(1, n, 1, D, generator=g)
    v *= vscale * torch.exp(2 * torch.randn(1, n, 1, 1, generator=g))
    table, pages = table_of([n], 64)
    cache = fc().PagedInt4Cache(pages, 1, D)
    cache.append(None, k.cuda(), v.cuda(), table, i32([0]))
    q = torch.randn(1, 2, D, generator=g).to(DT[dtype])
    out = cache.attend(q.cuda(), table, i32([n]))
    hk, hv = (kv4.values(*kv4.quantise(x[0, :, 0].numpy())) for x in (k, v))
    want, _ = kv4.attend(q[0].float().numpy(), hk, hv)
    top = np.abs(hv).max()
    if dtype == "fp16" and np.abs(want).max() > 65504:
        pytest.skip("the output does not fit fp16")
    near(out[0], want, dtype, top)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,page,Hk,G,Sq", [(128, 64, 2, 16, 1), (64, 32, 4, 4, 5), (96, 16, 2, 9, 1)])
def test_attend_many_rows_over_a_long_table(dtype, D, page, Hk, G, Sq):
    """Tables that could hold 2^21 tokens and heads: two column blocks serve a head's rows."""
    lens = [1, page + 3, 900]
    cache, table, held = filled(lens, Hk, D, page, seed=D)
    long = torch.full((3, (1 << 21) // (3 * Hk * page) + 1), -1, dtype=torch.int32, device="cuda")
    long[:, : table.shape[1]] = table
    q = torch.randn(3, Sq, Hk * G, D, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    out = cache.attend(q.cuda(), long, i32(lens))
    for b, n in enumerate(lens):
        for s in range(Sq):
            seen = max(0, n - (Sq - 1 - s))
            for h in range(Hk):
                rows = slice(h * G, (h + 1) * G)
                k, v = (x[:seen, h] for x in held[b])
                want, _ = kv4.attend(q[b, s, rows].float().numpy(), k, v)
                near(out[b, s, rows], want, dtype, np.abs(v).max() if seen else 1.0, (b, s, h))
    cache.check()


def test_attend_scale_out_strides_and_shared_pages():
    Hk, G, D, page = 2, 2, 64, 16
    cache, table, held = filled([50], Hk, D, page)
    both = table.repeat(2, 1)  # two sequences on the same pages
    q = torch.randn(4, 2, Hk * G, D, generator=torch.Generator().manual_seed(6)).transpose(0, 1).cuda()[:, 0]
    out = torch.full((2, Hk * G, 2 * D), 7.0, device="cuda")
    got = cache.attend(q, both, i32([50, 21]), scale=0.3, out=out[..., :D])
    assert got.data_ptr() == out.data_ptr() and (out[..., D:] == 7).all()
    for b, n in enumerate([50, 21]):
        for h in range(Hk):
            want, _ = kv4.attend(q[b, h * G:(h + 1) * G].cpu().numpy(), held[0][0][:n, h], held[0][1][:n, h],
                                 scale=0.3)
            near(got[b, h * G:(h + 1) * G], want, "fp32", np.abs(held[0][1]).max())


def test_inactive_sequences():
    """A negative length: nothing is stored, the output is zero."""
    Hk, D, page = 1, 64, 16
    cache, table, _ = filled([5, 5], Hk, D, page)
    before = cache.pool.clone()
    x = torch.randn(2, Hk, D, device="cuda")
    cache.append(x, x, x, table, i32([-1, -1]))
    assert torch.equal(cache.pool, before)
    out, lse = cache.attend(x, table, i32([-1, 5]), return_lse=True)
    assert (out[0] == 0).all() and (out[1] != 0).all() and lse[0] == -math.inf
    cache.check()


def test_offsets_past_32_bits():
    """The last pages of a pool over 4 GiB."""
    Hk, D, page = 8, 128, 64
    pages = (9 << 29) // fc().PagedInt4Cache(1, Hk, D).page_bytes
    cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
    assert cache.pool.numel() > 1 << 32
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(1, 100, Hk, D, generator=g), torch.randn(1, 100, Hk, D, generator=g)
    table = i32([[pages - 1, pages - 2]])
    cache.append(None, k.cuda(), v.cuda(), table, i32([0]))
    gk, gv = cache.read(table, count=100, dtype=torch.float32)
    hk, hv = (kv4.values(*kv4.quantise(x[0].numpy())) for x in (k, v))
    assert np.array_equal(gk[0].cpu().numpy(), hk) and np.array_equal(gv[0].cpu().numpy(), hv)
    q = torch.randn(1, Hk, D, generator=g)
    out = cache.attend(q.cuda(), table, i32([100]))
    assert cache.select(q.cuda(), table, i32([100]), 1, sink=0).flatten().tolist() == [1] * Hk
    for h in range(Hk):
        want, _ = kv4.attend(q[0, h:h + 1].numpy(), hk[:, h], hv[:, h])
        near(out[0, h:h + 1], want, "fp32", np.abs(hv).max())
    cache.check()


def test_graph_follows_lengths_and_streams():
    """A captured decode step, replayed while the lengths grow, equals eager calls on another stream."""
    B, Hq, Hk, D, page, steps = 3, 4, 2, 64, 16, 20
    g = torch.Generator().manual_seed(10)
    x = torch.randn(steps, B, Hq + 2 * Hk, D, generator=g).bfloat16().cuda()
    table, pages = table_of([40, 60, 30 + steps], page)
    tab = fc().rotary_table(128, D)

    def step(cache, t, lens):
        q, k, v = t.split([Hq, Hk, Hk], 1)
        q = cache.append(q, k, v, table, lens, rotary=tab)
        lens += 1
        p = cache.select(q, table, lens, 2)
        return cache.attend(q, table, lens), cache.attend(q, table, lens, selected=p)

    outs = []
    for captured in (False, True):
        cache = fc().PagedInt4Cache(pages, Hk, D, page_size=page, bounds=True)
        lens, got, buf = i32([0, 16, 30]), [], torch.empty_like(x[0])
        fill = torch.randn(B, 30, Hk, D, generator=torch.Generator().manual_seed(1)).cuda()
        cache.append(None, fill, fill, table, i32([0, 0, 0]))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            if captured:
                buf.copy_(x[0])
                step(cache, buf, lens.clone())  # the workspaces of this stream
                s.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    o = step(cache, buf, lens)
                for t in range(steps):
                    buf.copy_(x[t])
                    graph.replay()
                    got.append([y.clone() for y in o])
            else:
                for t in range(steps):
                    got.append(step(cache, x[t], lens))
        s.synchronize()
        cache.check()
        outs.append(got)
    for a, b in zip(*outs):
        assert all(torch.equal(y, z) for y, z in zip(a, b))


# ------------------------------------------------------------------------- select
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D,page,Hk,G,count,sink,recent", [
    (128, 16, 2, 4, 8, 1, 1), (64, 32, 1, 1, 1, 0, 1), (64, 16, 3, 7, 5, 0, 0), (256, 16, 1, 8, 6, 2, 3),
    (96, 16, 2, 2, 12, 1, 0), (192, 32, 1, 3, 4, 1, 1), (128, 16, 1, 32, 9, 0, 2)])
def test_select_and_attend_over_the_selection(dtype, D, page, Hk, G, count, sink, recent):
    lens = [0, 5, page * count, page * count + 1, 40 * page - 3, 131 * page]
    cache, table, held = filled(lens, Hk, D, page, seed=D, bounds=True)
    q = torch.randn(len(lens), Hk * G, D, generator=torch.Generator().manual_seed(3)).to(DT[dtype])
    pages = cache.select(q.cuda(), table, i32(lens), count, sink=sink, recent=recent)
    out, lse = cache.attend(q.cuda(), table, i32(lens), selected=pages, return_lse=True)
    for b, n in enumerate(lens):
        k, v = held[b]
        for h in range(Hk):
            x = q[b, h * G:(h + 1) * G].float().numpy()
            m = -(-n // page)
            bd = [kv4.bounds(k[p * page:(p + 1) * page, h]) for p in range(m)]
            want = kv4.select(x, np.array([y[0] for y in bd]).reshape(m, 2, D), [y[1] for y in bd],
                              count, sink, recent)
            assert pages[b, h].tolist() == want + [-1] * (count - len(want)), (b, h)
            seen = np.isin(np.arange(n) // page, want)
            o, wl = kv4.attend(x, k[:, h], v[:, h], seen)
            near(out[b, h * G:(h + 1) * G], o, dtype, np.abs(v[:, h]).max() if n else 1.0, (b, h))
    cache.check()


def test_select_ties_zeros_and_long_tables():
    """Equal pages go by index; a zero query scores everything alike; more pages than one pass holds."""
    D, page, m = 64, 16, 5000
    cache = fc().PagedInt4Cache(3, 1, D, page_size=page, bounds=True)
    x = torch.randn(1, 3 * page, 1, D, generator=torch.Generator().manual_seed(2)).cuda()
    ids = i32([[0, 1, 2]])
    cache.append(None, x, x, ids, i32([0]))
    table = ids.repeat(1, m // 3 + 1)[:, :m].contiguous()
    q = torch.randn(1, 2, D, generator=torch.Generator().manual_seed(3)).cuda()
    bd = [kv4.bounds(kv4.values(*kv4.quantise(x[0, p * page:(p + 1) * page, 0].cpu().numpy()))) for p in range(3)]
    for n, count in ((m, 64), (m, 1700), (m - 1, 4000), (1024, 1000), (1025, 1)):
        got = cache.select(q, table, i32([n * page]), count, sink=0, recent=0)[0, 0].tolist()
        want = kv4.select(q[0].cpu().numpy(), np.array([bd[p % 3][0] for p in range(n)]),
                          [bd[p % 3][1] for p in range(n)], count, 0, 0)
        assert got == want
    got = cache.select(torch.zeros_like(q), table, i32([m * page]), 7, sink=1, recent=2)[0, 0].tolist()
    assert got == [0, 1, 2, 3, 4, m - 2, m - 1]
    cache.check()


def test_calls_of_different_sizes_share_a_workspace():
    """Few long sequences, then many: what a call leaves behind is not the next one's counters."""
    Hk, G, D, page = 4, 2, 64, 16
    few, many = [6000, 5000], [300 + 7 * i for i in range(70)]
    held = [filled(lens, Hk, D, page, seed=s, bounds=True) for s, lens in ((1, few), (2, many))]
    q = [torch.randn(len(lens), Hk * G, D, generator=torch.Generator().manual_seed(4)).cuda() for lens in (few, many)]
    first = None
    for _ in range(2):
        for order in ((0, 1), (1, 0)):
            got = {}
            for i in order:
                (cache, table, _), lens = held[i], i32((few, many)[i])
                pages = cache.select(q[i], table, lens, 9)
                got[i] = (cache.attend(q[i], table, lens), pages, cache.attend(q[i], table, lens, selected=pages))
            first = first or got
            assert all(torch.equal(x, y) for i in (0, 1) for x, y in zip(got[i], first[i]))
    for i, lens in enumerate((few, many)):
        for b in range(0, len(lens), 13):
            k, v = held[i][2][b]
            for h in range(Hk):
                x = q[i][b, h * G:(h + 1) * G].cpu().numpy()
                m = -(-lens[b] // page)
                bd = [kv4.bounds(k[p * page:(p + 1) * page, h]) for p in range(m)]
                want = kv4.select(x, np.array([y[0] for y in bd]), [y[1] for y in bd], 9, 1, 1)
                assert first[i][1][b, h].tolist() == want
                o, _ = kv4.attend(x, k[:, h], v[:, h])
                near(first[i][0][b, h * G:(h + 1) * G], o, "fp32", np.abs(v).max())


def test_selected_in_any_order_and_out_of_range():
    Hk, G, D, page, n = 2, 2, 64, 16, 100
    cache, table, held = filled([n, 0], Hk, D, page)
    q = torch.randn(2, Hk * G, D, generator=torch.Generator().manual_seed(3))
    pick = i32([[[6, -1, 2, 99, 0], [-5, 7, -1, 3, 1000000]], [[0, 1, 2, 3, 4]] * 2])
    out = cache.attend(q.cuda(), table, i32([n, 0]), selected=pick)
    for h, pages in enumerate(([6, 2, 0], [3])):
        seen = np.isin(np.arange(n) // page, pages)
        want, _ = kv4.attend(q[0, h * G:(h + 1) * G].numpy(), held[0][0][:, h], held[0][1][:, h], seen)
        near(out[0, h * G:(h + 1) * G], want, "fp32", np.abs(held[0][1]).max())
    assert (out[1] == 0).all()
    none = cache.attend(q.cuda(), table, i32([n, 0]), selected=torch.full_like(pick, -1))
    assert (none == 0).all()
    empty = cache.attend(q.cuda(), table, i32([n, 0]), selected=pick[..., :0].contiguous())
    assert (empty == 0).all()


# ----------------------------------------------------------------------- refusals
def test_bad_pages_lengths_and_positions_are_reported():
    Hk, D, page = 1, 64, 16
    x = torch.randn(1, 1, D, device="cuda")
    cache = fc().PagedInt4Cache(2, Hk, D, page_size=page, bounds=True)
    err = fc()._lib.FlashCodecError
    cache.append(None, x, x, i32([[7]]), i32([0]))  # a page outside the pool: skipped
    with pytest.raises(err, match="page outside"):
        cache.check()
    cache.check()
    cache.append(None, x, x, i32([[0]]), i32([16]))  # past the table
    with pytest.raises(err, match="past what the page table"):
        cache.check()
    cache.append(x, x, x, i32([[0]]), i32([3]), rotary=fc().rotary_table(2, 64))
    with pytest.raises(err, match="rotary table"):
        cache.check()
    cache.attend(x, i32([[-3]]), i32([5]))
    with pytest.raises(err, match="page outside"):
        cache.check()
    cache.attend(x, i32([[0]]), i32([2 ** 31 - 1]))
    with pytest.raises(err, match="past what the page table"):
        cache.check()
    cache.select(x, i32([[0, 9]]), i32([20]), 1, sink=0)
    with pytest.raises(err, match="page outside"):
        cache.check()
    cache.read(i32([[5]]), count=2)
    with pytest.raises(err, match="page outside"):
        cache.check()
    cache.read(i32([[0]]), i32([10]), count=20)
    with pytest.raises(err, match="past what the page table"):
        cache.check()


def test_refusals():
    Hk, D, page = 2, 64, 16
    cache = fc().PagedInt4Cache(4, Hk, D, page_size=page)
    t, n = i32([[0, 1]]), i32([0])
    x = torch.randn(1, Hk, D, device="cuda")
    q = torch.randn(1, 2 * Hk, D, device="cuda")
    wide = torch.randn(1, 6, D, device="cuda")
    bad = [
        lambda: cache.append(q, x, x.bfloat16(), t, n),
        lambda: cache.append(q, x, x[:, :1], t, n),
        lambda: cache.append(q.bfloat16(), x, x, t, n),
        lambda: cache.append(q, x.int(), x.int(), t, n),
        lambda: cache.append(q, x, x, t.long(), n),
        lambda: cache.append(q, x, x, t, n.long()),
        lambda: cache.append(q, x, x, t, i32([0, 0])),
        lambda: cache.append(q, x, x, t[0], n),
        lambda: cache.append(q, x.transpose(1, 2).contiguous().transpose(1, 2), x, t, n),
        lambda: cache.append(q, x, x, t, n, q_weight=torch.ones(D + 1, device="cuda")),
        lambda: cache.append(q, x, x, t, n, rotary=torch.ones(4, 24, device="cuda")),
        lambda: cache.append(q, x, x, t, n, rotary=torch.ones(4, 32, device="cuda").half()),
        lambda: cache.append(q, x, x, t, n, cu_seqlens=i32([0])),
        lambda: cache.append(q, x, x, t, n, positions=i32([0, 1])),
        lambda: cache.append(q, x, x, t, n, q_out=x),
        lambda: cache.append(x, x, x + 1, t, n, q_out=x),
        lambda: cache.append(wide[:, :4], wide[:, 4:6], x, t, n, q_out=wide[:, 1:5]),
        lambda: cache.append(q, wide[:, 4:6], x, t, n, q_out=wide[:, 1:5]),
        lambda: cache.attend(q[:, :3], t, n),
        lambda: cache.attend(q[..., :32], t, n),
        lambda: cache.attend(q, t, n, selected=i32([[[0]]])),
        lambda: cache.attend(q[:, None].repeat(1, 2, 1, 1), t, n, selected=i32([[[0], [0]]])),
        lambda: cache.attend(q, t, n, out=x),
        lambda: cache.attend(q.int(), t, n),
        lambda: cache.select(q, t, n, 2),
        lambda: cache.read(t),
        lambda: cache.read(t, count=2, dtype=torch.int8),
        lambda: fc().PagedInt4Cache(0, Hk, D),
        lambda: fc().PagedInt4Cache(4, Hk, 80),
        lambda: fc().PagedInt4Cache(4, Hk, D, page_size=24),
        lambda: fc().PagedInt4Cache(4, Hk, D, bounds=True).select(q, t, n, 1, sink=1, recent=1),
        lambda: fc().PagedInt4Cache(4, Hk, D, bounds=True).select(q, t, n, 0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was not refused")
    for f in (lambda: cache.append(q, x.cpu(), x.cpu(), t, n), lambda: cache.attend(q.cpu(), t, n),
              lambda: cache.append(q, x.requires_grad_(), x, t, n)):
        with pytest.raises(RuntimeError):
            f()
    with torch.no_grad():
        cache.append(q, x, x, t, n)
    cache.check()
