"""Attention over prompts: calls that its documentation allows and that lie off the beaten track.

Bounds are those of test_gpu_prompt.py: a weight is off by half a step u of q's type, scores by 2^-12,
the output by u of itself.
"""

import math

import numpy as np
import pytest
import torch

from test_gpu_prompt import cu, exact, fc, i32, make, near, near_lse

pytestmark = pytest.mark.gpu


def guarded(q, k, v, cq, ck, guard, causal=True):
    """fc_prompt_attn with a workspace of exactly the size that it asks for, and what lies behind it."""
    from flashcodec_b200 import _kernels as K
    from flashcodec_b200 import _lib
    lib, (Tq, Hq, D), (Tk, Hk, _), B = _lib.load(), q.shape, k.shape, len(cq) - 1
    size = lib.fc_prompt_attn_workspace_size(B, Tq, Hq, Hk, D)
    ws = torch.zeros(size + guard, dtype=torch.uint8, device="cuda")
    ws[size:] = 0xa5
    out = torch.full_like(q, math.nan)
    rc = lib.fc_prompt_attn(*K._place(q), *K._place(k), *K._place(v), K.DTYPE_CODE[q.dtype], B, 0, 0, Tq, Tk, Hq, Hk, D,
                            cq.data_ptr(), ck.data_ptr(), causal, D ** -0.5, *K._place(out), None, ws.data_ptr(), size,
                            torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "prompt_attn")
    torch.cuda.synchronize()
    assert (ws[size:] == 0xa5).all() and not ws[:4].any()
    return out


def test_sequences_that_overlap_stay_in_the_workspace():
    """cu_seqlens that fall again: 16 sequences over the same 2000 rows, more items than rows could make.
    The rows are written by each of them: the results are those of one or of another."""
    n, m, D = 2000, 20000, 128
    q, k, v = make([(n, m)], 8, 1, D, "bf16")
    cq = i32([0, *[n, 0] * 16])
    ck = i32([0, m, *[0, 10] * 15, 0])
    out = guarded(q, k, v, cq, ck, 160 << 20).double().cpu().numpy()
    top = v.abs().max().item()
    rows = [0, 1, 700, 1989, 1990, 1999]
    long = exact(q[-1:], k, v)[0]  # (the last row sees all of the long sequence's keys)
    short = exact(q[1990:], k[:10], v[:10])[0]
    lim = 2.0 ** -8 * top + (2.0 ** -8 + 2.0 ** -12) * top
    assert np.isfinite(out).all()
    assert np.minimum(np.abs(out[-1] - long[0]), np.abs(out[-1] - short[-1])).max() <= lim
    for i in rows[:4]:  # nothing seen in the short ones
        want = exact(q[i:i + 1], k[:m - n + i + 1], v[:m - n + i + 1])[0][0]
        assert np.minimum(np.abs(out[i] - want), np.abs(out[i])).max() <= lim


@pytest.mark.parametrize("lead", [0, 7, 1500])
@pytest.mark.parametrize("B,n", [(33, 50), (700, 13)])
def test_many_sequences_behind_rows_of_no_sequence(B, n, lead):
    """More sequences than a warp has lanes, not from row 0 on: in place and beside are the same bits, each
    item being computed once; rows of no sequence get zeros.  (Keys of one tile: no row takes another reference.)"""
    T = lead + B * n + 20
    q, k, v = make([(T, T)], 4, 2, 64, "bf16", B + lead)
    c = i32([lead + n * b for b in range(B + 1)])
    want, lse = fc().prompt_attention(q, k, v, c, return_lse=True)
    assert not want[:lead].any() and not want[-20:].any()
    assert torch.isneginf(lse[:lead]).all() and torch.isneginf(lse[-20:]).all()
    for b in (0, 1, B // 2, B - 1):
        at = slice(lead + b * n, lead + b * n + n)
        near(want[at], exact(q[at], k[at], v[at])[0], "bf16", v[at].abs().max().item())
    assert torch.equal(want[lead:-20], fc().prompt_attention(q[lead:-20], k[lead:-20], v[lead:-20], c - lead))
    for _ in range(3):
        mine = q.clone()
        assert fc().prompt_attention(mine, k, v, c, out=mine) is mine and torch.equal(mine, want)
    assert fc().attention_status().value() == 0


@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("Hq,Hk", [(2, 1), (8, 8)])
def test_no_numbers_in_many_sequences(D, Hq, Hk):
    """Every sequence holds an infinity and a NaN among its values, in tiles that are looked through; empty ones
    lie between them.  Outputs are finite where fp64's are, for every item and whatever is under way beside it."""
    rng = np.random.default_rng(D + Hk)
    B = 700 // Hk
    lens = [int(n) if rng.random() < 0.6 else 0 for n in rng.integers(2, 40, B)]
    c = cu(lens)
    q, k, v = make([(sum(lens), sum(lens))], Hq, Hk, D, "bf16", B)
    a, finite = 0, torch.ones(sum(lens), Hq, D, dtype=torch.bool)
    for n in lens:
        if n:
            i, j = sorted(rng.integers(0, n, 2).tolist())
            d, h, G = int(rng.integers(0, D - 1)), int(rng.integers(0, Hk)), Hq // Hk
            v[a + i, h, d], v[a + j, h, d + 1] = math.inf, math.nan
            finite[a + i:a + n, h * G:h * G + G, d] = False
            finite[a + j:a + n, h * G:h * G + G, d + 1] = False
        a += n
    for _ in range(5):
        out = fc().prompt_attention(q, k, v, c)
        assert torch.equal(out.isfinite().cpu(), finite)
    assert fc().attention_status().value() == 0


@pytest.mark.parametrize("Hq,Hk", [(3, 1), (14, 2), (20, 4)])
@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("many", [False, True])
def test_rows_of_no_query_change_no_bits(D, Hq, Hk, many):
    """Groups that do not divide 128 leave rows of a query tile without a query, and a sequence's last tile holds
    the next one's: with scores that grow, in place and beside, after whatever other calls left behind, the same bits."""
    lens = [(300, 300), (5, 260), (129, 400), (41, 41), (700, 700), (77, 390)] * (6 if many else 1)
    q, k, v = make(lens, Hq, Hk, D, "bf16", Hq)
    k = (k.float() * torch.linspace(0, 8, k.shape[0], device="cuda").sin()[:, None, None] * 4).bfloat16()
    args = cu([n for n, _ in lens]), cu([m for _, m in lens])
    want = fc().prompt_attention(q, k, v, *args)
    for a, b, (n, m) in ((0, 0, lens[0]), (300, 300, lens[1])):
        # (sums of |q k| up to 700 here: scores off by 2^-11, 2^-12 more than near() has, which is 2^-4 of its 2^-8)
        near(want[a:a + n], exact(q[a:a + n], k[b:b + m], v[b:b + m])[0], "bf16", (1 + 2.0 ** -4) * v[b:b + m].abs().max().item())
    for size in (1.0, 300.0, -300.0):
        x = torch.full((4000, 16, D), size, dtype=q.dtype, device="cuda")
        fc().prompt_attention(x, x, x, i32([0, 4000]))  # (other rows of shared memory)
        assert torch.equal(fc().prompt_attention(q, k, v, *args), want)
        mine = q.clone()
        fc().prompt_attention(mine, k, v, *args, out=mine)
        assert torch.equal(mine, want)
    # neighbours of other sizes
    other = q.clone()
    a = 0
    for i, (n, _) in enumerate(lens):
        if i % 2:
            other[a:a + n] *= 64
        a += n
    out = fc().prompt_attention(other, k, v, *args)
    a = 0
    for i, (n, _) in enumerate(lens):
        if i % 2 == 0:
            assert torch.equal(out[a:a + n], want[a:a + n])
        a += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_a_key_that_is_no_number(D, dtype):
    """Wherever it lies in a tile that all rows see, the rows that see it are NaN, log-sums too, and no other."""
    n = 400
    q, k, v = (t.to(dtype) for t in make([(n, n)], 4, 2, D, "bf16"))
    want = fc().prompt_attention(q, k, v, cu([n]), return_lse=True)
    for j in [*range(8), 121, 126, 127, 260, 263]:
        y = k.clone()
        y[j, 0, 3] = math.nan
        got = fc().prompt_attention(q, y, v, cu([n]), return_lse=True)
        for g, w in zip(got, want):
            assert torch.equal(g[:, 2:], w[:, 2:]) and torch.equal(g[:j, :2], w[:j, :2])
            assert g[j:, :2].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_keys_that_weigh_nothing(D, dtype):
    """Keys whose scores are infinite below: no weight, wherever they lie in a tile; others as without them."""
    n = 400
    q, k, v = (t.to(dtype) for t in make([(n, n)], 2, 1, D, "bf16"))
    q[..., 0] = 1.0
    for j in range(8):
        none = torch.zeros(n, dtype=torch.bool)
        none[40 + j:200:8] = True
        y = k.clone()
        y[none, 0, 0] = -math.inf
        out, lse = fc().prompt_attention(q, y, v, cu([n]), return_lse=True)
        rest = ~none
        for i in (300, 399):
            want, wl = exact(q[i:i + 1], k[:i + 1][rest[:i + 1]], v[:i + 1][rest[:i + 1]])
            near(out[i:i + 1], want, "bf16" if dtype is torch.bfloat16 else "fp16", v.abs().max().item())
            near_lse(lse[i:i + 1], wl)


@pytest.mark.parametrize("n,m,Hq,Hk", [(3, 32769, 2, 1), (9216, 32769, 4, 4)])
@pytest.mark.parametrize("at", [0, 20000])
def test_a_tail_of_small_weights(n, m, Hq, Hk, at):
    """32768 keys of 2^-25 the weight of one whose value is zero: fp16 weights keep them, cut along the keys and
    not.  Held 2^7 times larger, each is off by 2^-25 of a sum above 2^6: 2^-31 M a key; scores and exponentials
    (polynomials: 2^-18.5, which is 2^-18 with fp32's own) and the output's rounding, 2^-11, are of the result."""
    D = 64
    q = torch.zeros(n, Hq, D, dtype=torch.float16, device="cuda")
    k = torch.zeros(m, Hk, D, dtype=torch.float16, device="cuda")
    v = torch.ones(m, Hk, D, dtype=torch.float16, device="cuda")
    q[..., 0], k[at, :, 0], v[at] = 8.0, 17.33, 0.0
    tail = (m - 1) * math.exp(-k[at, 0, 0].item())
    out, lse = fc().prompt_attention(q, k, v, cu([n]), cu([m]), causal=False, return_lse=True)
    want = tail / (1 + tail)
    err = (out.double() - want).abs().max().item()
    assert err <= (2.0 ** -11 + 2.0 ** -18) * want + m * 2.0 ** -31, f"{out.flatten()[0].item()} for {want}"
    assert (lse.double() - (k[at, 0, 0].item() + math.log1p(tail))).abs().max() <= 2.0 ** -12
    assert fc().attention_status().value() == 0


def test_a_stream_that_waits_for_a_long_one():
    """100 queries over 2^25 keys (a third of a second, one query tile), and items of two tiles behind it on the
    same block: the second tile's warps wait for longer than any product takes, and do not give up."""
    m, n, B, D = 1 << 25, 200, 300, 64
    lens = [(100, m)] + [(n, n)] * (B - 1)
    k = torch.zeros(m + n * (B - 1), 1, D, dtype=torch.bfloat16, device="cuda")
    q, k[m:], _ = make([(100 + n * (B - 1), n * (B - 1))], 1, 1, D, "bf16")
    out, lse = fc().prompt_attention(q, k, k, cu([a for a, _ in lens]), cu([b for _, b in lens]), return_lse=True)
    assert fc().attention_status(reset=True).value() == 0
    assert not out[:100].any()
    # equal scores of zero: weights of one, whose sum is exact
    seen = torch.arange(m - 99, m + 1, device="cuda").double().log()
    assert (lse[:100, 0].double() - seen).abs().max() <= 2.0 ** -19
    for b in range(1, B, 23):
        a, c = 100 + n * (b - 1), m + n * (b - 1)
        x = k[c:c + n]
        near(out[a:a + n], exact(q[a:a + n], x, x)[0], "bf16", x.abs().max().item())


def test_clearing_the_status_leaves_the_counters_of_graphs():
    """A graph may be under way on another stream when its capture's stream clears the status words."""
    from flashcodec_b200 import _kernels as K
    lens = [(40, 3000)]
    q, k, v = make(lens, 4, 2, 64, "bf16")
    args = (q, k, v, cu([40]), cu([3000]))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fc().prompt_attention(*args)
    with torch.cuda.graph(graph, stream=side):
        fc().prompt_attention(*args)
    graph.replay()
    torch.cuda.synchronize()
    held = {key[2] != 0: ws for key, ws in K._prompt_workspaces.items() if key[1] == side.cuda_stream}
    for ws in held.values():
        ws[256:260] = 7  # as if a row's pieces were on their way
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert fc().attention_status(reset=True).value() == 0
    side.synchronize()
    assert held[True][256:260].tolist() == [7] * 4 and held[False][256:260].tolist() == [0] * 4


def test_a_graph_of_many_sequences():
    """More sequences than a warp has lanes, captured: replays follow cu_seqlens, rows in front included."""
    B, T = 40, 900
    q, k, v = make([(T, T)], 4, 2, 128, "bf16")
    c = i32([20 * b for b in range(B + 1)])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fc().prompt_attention(q, k, v, c)
    rng = np.random.default_rng(0)
    for lead in (0, 300, 0, 5):
        lens = rng.multinomial(T - lead - 30, rng.dirichlet([0.4] * B))
        c.copy_(i32((lead + np.concatenate([[0], np.cumsum(lens)])).tolist()))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fc().prompt_attention(q, k, v, c))
        assert not out[:lead].any() and not out[-30:].any()
        b = int(lens.argmax())
        at = slice(int(c[b]), int(c[b + 1]))
        near(out[at], exact(q[at], k[at], v[at])[0], "bf16", v[at].abs().max().item())
