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
