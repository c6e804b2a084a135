"""Attention over whole prompts on the GPU against fp64.

Bounds.  A weight is rounded to the type of q (half a step, u = 2^-8 for bf16 and 2^-11 for fp16,
of the weight), so the output is off by u M at most, M the largest |value|; the output's own
rounding is u |out|.  Scores are fp32 sums of D exact products: of sum |q k| up to 200 here, off by
D 2^-24 200 / sqrt(D) < 2^-12 after scaling, which the weights carry on: 2^-12 M.  The log-sum takes
the scores' 2^-12, and 2^-22 of itself for its own arithmetic.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def fc():
    import flashcodec_b200
    return flashcodec_b200


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cu(lens):
    return i32([0, *np.cumsum(lens).tolist()])


def exact(q, k, v, causal=True, scale=None):
    """fp64 (n, Hq, D) and log-sums of one sequence; a query that sees nothing: zeros, -inf."""
    q, k, v = (t.double().cpu().numpy() for t in (q, k, v))
    n, Hq, D = q.shape
    m, Hk = k.shape[:2]
    G = Hq // Hk
    out, lse = np.zeros((n, Hq, D)), np.full((n, Hq), -np.inf)
    for h in range(Hq if m else 0):
        s = q[:, h] @ k[:, h // G].T * (D ** -0.5 if scale is None else scale)
        if causal:
            s[np.arange(m) > np.arange(m - n, m)[:, None]] = -np.inf
        seen = np.isfinite(s.max(-1))
        s = s[seen]
        top = s.max(-1, keepdims=True)
        p = np.exp(s - top)
        z = p.sum(-1, keepdims=True)
        out[seen, h] = p / z @ v[:, h // G]
        lse[seen, h] = (top + np.log(z))[:, 0]
    return out, lse


def near(got, want, dtype, top, what=""):
    got = got.double().cpu().numpy()
    u = HALF_STEP[dtype]
    err, lim = np.abs(got - want), u * np.abs(want) + (u + 2.0 ** -12) * top
    assert np.isfinite(got).all(), what
    assert (err <= lim).all(), f"{what}: {err.max():.3e}, {(err / np.maximum(lim, 1e-30)).max():.2f} of the bound"


def near_lse(got, want):
    got = got.double().cpu().numpy()
    none = np.isneginf(want)
    assert np.isneginf(got[none]).all()
    assert (np.abs(got[~none] - want[~none]) <= 2.0 ** -12 + 2.0 ** -22 * np.abs(want[~none])).all()


def make(lens, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    T, L = sum(n for n, _ in lens), sum(m for _, m in lens)
    q = torch.randn(T, Hq, D, generator=g)
    k = torch.randn(L, Hk, D, generator=g)
    v = torch.randn(L, Hk, D, generator=g)
    return tuple(t.to(DT[dtype]).cuda() for t in (q, k, v))


def check(q, k, v, lens, dtype, causal=True, scale=None, **kw):
    cq, ck = cu([n for n, _ in lens]), cu([m for _, m in lens])
    out, lse = fc().prompt_attention(q, k, v, cq, ck, causal=causal, scale=scale, return_lse=True, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == q.shape[:-1]
    a = b = 0
    for n, m in lens:
        want, wl = exact(q[a:a + n], k[b:b + m], v[b:b + m], causal, scale)
        top = v[b:b + m].abs().max().item() if m else 0.0
        near(out[a:a + n], want, dtype, top, f"{n} of {m}")
        near_lse(lse[a:a + n], wl)
        a, b = a + n, b + m
    assert fc().attention_status().value() == 0
    return out


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(n, D):
    check(*make([(n, n)], 4, 2, D, "bf16", n), [(n, n)], "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_packed(D, dtype):
    lens = [(5, 5), (130, 130), (1, 1), (257, 257), (64, 64), (383, 383)]
    check(*make(lens, 8, 2, D, dtype), lens, dtype)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 3), (7, 1), (14, 2), (24, 3), (33, 1), (128, 1)])
@pytest.mark.parametrize("D", [64, 192])
def test_groups(Hq, Hk, D):
    lens = [(70, 70), (19, 150)]
    check(*make(lens, Hq, Hk, D, "bf16"), lens, "bf16")


@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_other_keys(D, causal):
    """Keys that begin before their queries, fewer keys than queries (rows that see none), and none."""
    lens = [(3, 700), (40, 13), (0, 50), (129, 256), (20, 0), (17, 1), (200, 513), (0, 0)]
    check(*make(lens, 4, 2, D, "fp16"), lens, "fp16", causal=causal)


def test_many_sequences():
    """More sequences than a warp has lanes, and more items than there are blocks."""
    rng = np.random.default_rng(0)
    lens = [(int(n), int(n + m)) for n, m in zip(rng.integers(0, 90, 150), rng.integers(0, 200, 150))]
    check(*make(lens, 4, 2, 64, "bf16"), lens, "bf16")


def test_long():
    lens = [(2000, 2000), (100, 5000)]
    check(*make(lens, 8, 2, 128, "bf16"), lens, "bf16")


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("B,Sq,Sk", [(3, 37, 37), (2, 130, 300), (2, 40, 10), (1, 1, 1)])
def test_batches(B, Sq, Sk, D):
    """(B, S, heads, D), and heads before tokens in memory."""
    g = torch.Generator().manual_seed(B)
    for flip in (False, True):
        q, k, v = (torch.randn(B, H, S, D, generator=g).bfloat16().cuda().transpose(1, 2) if flip else
                   torch.randn(B, S, H, D, generator=g).bfloat16().cuda() for S, H in ((Sq, 6), (Sk, 2), (Sk, 2)))
        out, lse = fc().prompt_attention(q, k, v, return_lse=True)
        for b in range(B):
            want, wl = exact(q[b], k[b], v[b])
            near(out[b], want, "bf16", v[b].abs().max().item())
            near_lse(lse[b], wl)


def test_slices_of_one_buffer():
    """q, k and v side by side, as a fused projection leaves them; the outputs over the queries."""
    n, Hq, Hk, D = 200, 6, 2, 64
    buf = torch.randn(n, Hq + 2 * Hk, D, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    q, k, v = buf.split([Hq, Hk, Hk], 1)
    lens = [150, 50]
    keep = [t.clone() for t in (q, k, v)]
    out = fc().prompt_attention(q, k, v, cu(lens), out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(k, keep[1]) and torch.equal(v, keep[2])
    assert torch.equal(q, fc().prompt_attention(*keep, cu(lens)))


@pytest.mark.parametrize("shift", [1, 4])
def test_rows_off_16_byte_boundaries(shift):
    """What tensor maps cannot walk is copied; outputs are written where they are."""
    n, D = 90, 64
    lens = [(n, n)]
    q, k, v = make(lens, 4, 2, D, "bf16")

    def off(t):
        x = torch.zeros(t.numel() + shift, dtype=t.dtype, device="cuda")
        x[shift:] = t.flatten()
        return x[shift:].view(t.shape)
    out = torch.zeros(n, 4, D + shift, dtype=q.dtype, device="cuda")[..., :D]
    got = fc().prompt_attention(off(q), off(k), off(v), cu([n]), out=out)
    assert torch.equal(got, fc().prompt_attention(q, k, v, cu([n])))
    one = k[:, :1].expand(-1, 2, -1)  # heads in one place
    assert torch.equal(fc().prompt_attention(q, one, one, cu([n])),
                       fc().prompt_attention(q, one.contiguous(), one.contiguous(), cu([n])))


@pytest.mark.parametrize("D", [64, 192])
def test_rows_of_no_sequence(D):
    """A captured batch has a fixed number of rows: those before and behind the sequences get zeros."""
    q, k, v = make([(300, 300)], 4, 2, D, "bf16")
    c = i32([7, 60, 60, 250])
    out = torch.full_like(q, 9.0)
    _, lse = fc().prompt_attention(q, k, v, c, out=out, return_lse=True)
    for a, b in ((7, 60), (60, 250)):
        want, wl = exact(q[a:b], k[a:b], v[a:b])
        near(out[a:b], want, "bf16", v.abs().max().item())
        near_lse(lse[a:b], wl)
    for a, b in ((0, 7), (250, 300)):
        assert not out[a:b].any() and torch.isneginf(lse[a:b]).all()
    out = fc().prompt_attention(q, k, v, i32([0]))  # no sequence at all
    assert not out.any()
    out = fc().prompt_attention(q, k, v, i32([0, 200, 900]), i32([0, 200, 900]))  # cut to the rows there are
    assert torch.equal(out, fc().prompt_attention(q, k, v, i32([0, 200, 300])))
    fc().prompt_attention(q, k, v, i32([-50, 200, 100, 7000]), i32([5, -3, 100000, 2]))  # senseless: in bounds


def test_no_rows():
    q, k, v = make([(0, 40)], 4, 2, 64, "bf16")
    out, lse = fc().prompt_attention(q, k, v, i32([0, 0]), i32([0, 40]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q, k, v = make([(9, 0)], 4, 2, 64, "bf16")
    out, lse = fc().prompt_attention(q, k, v, i32([0, 9]), i32([0, 0]), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_matter(D, bad):
    """No numbers in later tokens, and in the neighbouring sequences."""
    lens = [(140, 140), (60, 60), (90, 200)]
    q, k, v = make(lens, 4, 2, D, "bf16")
    cq, ck = cu([n for n, _ in lens]), cu([m for _, m in lens])
    want = fc().prompt_attention(q, k, v, cq, ck)
    for x in (k, v):
        y = x.clone()
        y[139], y[150, 1], y[199, 0] = bad, bad, bad
        out = fc().prompt_attention(q, *((y, v) if x is k else (k, y)), cq, ck)
        same = torch.ones(290, 4, dtype=torch.bool)
        same[139] = False          # the last token of the first sequence
        same[150:200, 2:] = False  # the heads of KV head 1
        same[199, :2] = False
        assert torch.equal(out[same], want[same])
        assert not out[~same].isfinite().all(-1).any()


@pytest.mark.parametrize("D", [64, 192])
def test_infinite_values_that_are_seen(D):
    """An infinite value makes the outputs that see it infinite; two of unlike signs no number."""
    n = 150
    q, k, v = make([(n, n)], 2, 1, D, "bf16")
    v[100, 0, 5], v[120, 0, 5], v[130, 0, 9] = math.inf, -math.inf, math.nan
    out = fc().prompt_attention(q, k, v, cu([n]))
    assert out[:100, :, 5].isfinite().all() and (out[100:120, :, 5] == math.inf).all()
    assert out[120:, :, 5].isnan().all()
    assert out[:130, :, 9].isfinite().all() and out[130:, :, 9].isnan().all()
    rest = [d for d in range(D) if d not in (5, 9)]
    want, _ = exact(q, k, torch.where(v.isfinite(), v, torch.zeros_like(v)))
    near(out[:, :, rest], want[:, :, rest], "bf16", v[v.isfinite()].abs().max().item())


def test_queries_that_are_no_numbers_stay_alone():
    q, k, v = make([(100, 100)], 4, 2, 64, "bf16")
    want = fc().prompt_attention(q, k, v, cu([100]))
    q[40, 1, 3] = math.nan
    out = fc().prompt_attention(q, k, v, cu([100]))
    same = torch.ones(100, 4, dtype=torch.bool)
    same[40, 1] = False
    assert torch.equal(out[same], want[same]) and out[40, 1].isnan().all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(scale):
    lens = [(150, 150)]
    check(*make(lens, 4, 2, 64, "fp16"), lens, "fp16", scale=scale) if scale != 1.0 else \
        check(*(t * 0.5 for t in make(lens, 4, 2, 64, "fp16")), lens, "fp16", scale=scale)


def test_growing_scores():
    """Maxima that grow from tile to tile, and fall: sums are carried over to the new one."""
    n, D = 700, 64
    q, k, v = make([(n, n)], 2, 1, D, "bf16")
    q = torch.ones_like(q) * q[:, :, :1].sign()
    ramp = torch.linspace(0, 6, n).sin().cuda()[:, None, None]
    k = (torch.ones_like(k) * ramp * 4).bfloat16()
    want, wl = exact(q, k, v)
    out, lse = fc().prompt_attention(q, k, v, cu([n]), return_lse=True)
    # sums of 64 equal products are exact but for the last bit: scores up to 32 * 2^-22 off
    near(out, want, "bf16", v.abs().max().item())
    near_lse(lse, wl)


def test_streams_and_graphs():
    """Two captured calls of different sizes, replayed in either order between eager calls."""
    cases = []
    for lens in ([(50, 50)], [(300, 300), (20, 700)]):
        q, k, v = make(lens, 4, 2, 128, "bf16")
        args = (q, k, v, cu([n for n, _ in lens]), cu([m for _, m in lens]))
        cases.append((args, fc().prompt_attention(*args)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fc().prompt_attention(*args) for args, _ in cases]
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, (_, w) in zip(got, cases))
    graphs, outs = [], []
    for args, _ in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(fc().prompt_attention(*args))
    for order in ((0, 1), (1, 0), (1, 1)):
        for i in order:
            outs[i].zero_()
            graphs[i].replay()
            eager = fc().prompt_attention(*cases[1 - i][0])
            torch.cuda.synchronize()
            assert torch.equal(outs[i], cases[i][1]) and torch.equal(eager, cases[1 - i][1])
    # a graph follows the lengths: the same rows as one sequence less
    args = cases[1][0]
    args[3].copy_(i32([0, 300, 300]))
    graphs[1].replay()
    torch.cuda.synchronize()
    assert not outs[1][300:].any() and torch.equal(outs[1][:300], cases[1][1][:300])


def test_refusals():
    q, k, v = make([(8, 8)], 4, 2, 64, "bf16")
    c = cu([8])
    f = fc().prompt_attention
    bad = [
        ((q.float(), k.float(), v.float(), c), {}, NotImplementedError),
        ((q, k.half(), v, c), {}, ValueError),
        ((q, k, v), {}, ValueError),                              # packed rows without cu_seqlens
        ((q[None], k[None], v[None], c), {}, ValueError),
        ((q[None], k[None], v[None], None, c), {}, ValueError),
        ((q, k, v, c.long()), {}, ValueError),
        ((q, k, v, c, cu([4, 4])), {}, ValueError),
        ((q, k[:5], v[:5], c), {}, ValueError),                   # other keys need cu_seqlens_k
        ((q[:, :3], k, v, c), {}, ValueError),                    # heads
        ((q, k, v[:, :1], c), {}, ValueError),
        ((q[..., :48], k[..., :48], v[..., :48], c), {}, NotImplementedError),
        ((q, k, v, c), {"scale": math.nan}, ValueError),
        ((q, k, v, c), {"out": q.float()}, ValueError),
        ((q, k, v, c), {"out": q[:4]}, ValueError),
        ((q, k, v, c), {"out": q[:1].expand(8, -1, -1)}, ValueError),
        ((q.transpose(1, 2).contiguous().transpose(1, 2)[..., ::2], k[..., ::2], v[..., ::2], c), {}, ValueError),
        ((q.cpu(), k, v, c), {}, RuntimeError),
        ((q, k, v, c.cpu()), {}, RuntimeError),
        ((q.clone().requires_grad_(), k, v, c), {}, RuntimeError),
    ]
    for args, kw, err in bad:
        with pytest.raises(err):
            f(*args, **kw)
    buf = torch.zeros(8, 8, 64, dtype=q.dtype, device="cuda")
    for out, args in ((buf[:, 1:5], (buf[:, :4], k, v)), (buf[:, 2:6], (q, buf[:, 4:6], v)), (buf[:, :4], (q, k, buf[:, 3:5]))):
        with pytest.raises(ValueError, match="overlaps"):
            f(*args, c, out=out)
    big = torch.zeros(8, 129, 64, dtype=q.dtype, device="cuda")
    with pytest.raises(NotImplementedError):
        f(big, k[:, :1], v[:, :1], c)



@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_cut_along_keys(D, dtype):
    """Few queries over many keys: blocks share a query tile's keys and the last one joins the results."""
    lens = [(70, 6000), (3, 2500), (1, 9000), (40, 40), (0, 100)]
    q, k, v = make(lens, 4, 2, D, dtype)
    want = check(q, k, v, lens, dtype)
    args = (q, k, v, cu([n for n, _ in lens]), cu([m for _, m in lens]))
    for _ in range(3):  # whichever block comes last, the same bits
        assert torch.equal(fc().prompt_attention(*args), want)
    check(q, k, v, lens, dtype, causal=False)


def test_cut_rows_that_see_little():
    """Pieces that a row does not see, and rows that see nothing at all."""
    lens = [(2000, 1500), (300, 4000)]
    check(*make(lens, 2, 1, 64, "bf16"), lens, "bf16")


@pytest.mark.parametrize("D", [64, 256])
def test_no_numbers_in_pieces(D):
    """Of a key tile in the middle, and of one that is not seen by all."""
    n, m = 40, 5000
    q, k, v = make([(n, m)], 4, 2, D, "bf16")
    args = (cu([n]), cu([m]))
    want = fc().prompt_attention(q, k, v, *args)
    y = v.clone()
    y[m - 10, 0] = math.nan  # seen by the last 10 queries
    out = fc().prompt_attention(q, k, y, *args)
    assert torch.equal(out[:, 2:], want[:, 2:]) and torch.equal(out[: n - 10, :2], want[: n - 10, :2])
    assert out[n - 10 + 0:, :2].isnan().all()
    y = v.clone()
    y[1000, 1, 7] = math.inf  # seen by all
    out = fc().prompt_attention(q, k, y, *args)
    assert torch.equal(out[:, :2], want[:, :2]) and (out[:, 2:, 7] == math.inf).all()
    same = [d for d in range(D) if d != 7]
    assert torch.equal(out[:, 2:][..., same], want[:, 2:][..., same])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B", [31, 32, 33, 700])
def test_numbers_of_sequences(B, causal):
    """As many as a warp has lanes, one more, and many; empty ones among them; as a batch too."""
    rng = np.random.default_rng(B)
    lens = [(int(n), int(n + m)) for n, m in zip(rng.integers(0, 40, B), rng.integers(0, 60, B))]
    lens[3], lens[7], lens[-1] = (0, 0), (150, 150), (0, 9)
    check(*make(lens, 2, 1, 64, "bf16"), lens, "bf16", causal=causal)
    q, k, v = (torch.randn(B, S, H, 64, device="cuda").bfloat16() for S, H in ((5, 4), (9, 2), (9, 2)))
    out = fc().prompt_attention(q, k, v, causal=causal)
    flat = fc().prompt_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), cu([5] * B), cu([9] * B), causal=causal)
    assert torch.equal(out.flatten(0, 1), flat)
    want, _ = exact(q[-1], k[-1], v[-1], causal)
    near(out[-1], want, "bf16", v[-1].abs().max().item())
