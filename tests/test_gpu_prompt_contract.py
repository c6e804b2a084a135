"""Attention over prompts: calls that its documentation allows and that lie off the beaten track.

Bounds are those of test_gpu_prompt.py: a weight is off by half a step u of q's type, scores by 2^-12,
the output by u of itself.
"""

import math

import numpy as np
import pytest
import torch

from test_gpu_prompt import check, cu, exact, fc, i32, make, near

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
