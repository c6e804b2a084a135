"""Attention over whole prompts, before decoding goes on from a cache.

Decode steps attend to a compressed cache one token at a time; a prompt's own
attention has many queries for every key and runs here: packed sequences of
different lengths, causal, grouped heads.  With ``cu_seqlens_k`` the keys of a
sequence may begin before its queries: the next chunk of a long prompt, over the
values that a paged cache's ``read`` gives.  One launch (csrc/fc_prompt.cu).
The reference leaves prompts to the model's own attention.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _kernels as K


def _walkable(name, t):
    """t, or a copy where its rows are not on 16-byte boundaries or not apart from one another:
    the kernel walks them by tensor maps."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the head dim must have unit stride")
    step = 16 // t.element_size()
    bad = t.data_ptr() % 16
    for n, st in zip(t.shape[:-1], t.stride()):
        bad = bad or (n > 1 and (st <= 0 or st % step))
    if bad:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def prompt_attention(q, k, v, cu_seqlens=None, cu_seqlens_k=None, *, causal=True, scale=None, out=None,
                     return_lse=False):
    """softmax(scale * q . K^T) . V of every sequence.

    q: packed (T, Hq, D) with ``cu_seqlens``, or (B, S, Hq, D) without; bf16 or
        fp16, any strides with unit stride along D; D 64, 96, 128, 192 or 256.
    k, v: (Tk, Hk, D) or (B, Sk, Hk, D) of q's dtype; Hq a multiple of Hk.
    cu_seqlens: (B + 1,) int32 CUDA tensor, sequence b being rows cu_seqlens[b] to
        cu_seqlens[b + 1].  Rows of no sequence (a captured batch of fixed size)
        get zeros.
    cu_seqlens_k: the same for k and v (default: ``cu_seqlens``).  Both are read
        when the kernel runs, and cut to the rows that there are.
    causal: query i of n sees the keys up to its own, the last query being at the
        last key; else all keys.  A query that sees none gives zeros (and -inf).
    scale: of the scores (default D ** -0.5).
    out: where the outputs go (default: a new tensor; may be q).
    Returns the outputs in q's shape and dtype, and with ``return_lse`` the natural
    log of the softmax sums, q.shape[:-1] fp32.

    Scores, softmax and sums are fp32 (a quarter of the exponentials to 2^-13 with
    bf16, 2^-18 with fp16); weights are rounded to q's dtype before they meet the
    values (fp16: or by 2^-31 of their row's sum).  The products' sums cut, at
    2^-24 of the sum of weight * |value| for every 16 keys: 2^-11 of it at 131072 keys.
    Values beyond 2^128 / (256 * keys) may overflow.  It serves and has no gradient.
    """
    index, grad = q.get_device(), torch.is_grad_enabled()
    dual = getattr(forward_ad, "_current_level", 0) >= 0  # inside a dual level
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("cu_seqlens", cu_seqlens),
                    ("cu_seqlens_k", cu_seqlens_k)):
        if t is None:
            continue
        if t.get_device() != index or index < 0:
            K.require_cuda(q, t)
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
        if grad and t.requires_grad:
            raise RuntimeError("prompt_attention has no gradient: call it under torch.no_grad()")
        if dual and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("prompt_attention has no tangent: pass the primal of a dual tensor")
    packed = cu_seqlens is not None
    shape, keys, dtype = q.shape, k.shape, q.dtype
    if len(shape) != (3 if packed else 4):
        raise ValueError("q must be (T, heads, D) with cu_seqlens or (B, S, heads, D) without "
                         f"(got {tuple(shape)})")
    if len(keys) != len(shape) or keys != v.shape or keys[-1] != shape[-1] or shape[-2] == 0 or keys[-2] == 0 \
            or (not packed and keys[0] != shape[0]):
        raise ValueError(f"k and v must be alike and go with q (got {tuple(keys)}, {tuple(v.shape)} "
                         f"and {tuple(shape)})")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must have one dtype")
    if packed:
        for name, t in (("cu_seqlens", cu_seqlens), ("cu_seqlens_k", cu_seqlens_k)):
            if t is not None and (t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] < 1
                                  or t.shape != cu_seqlens.shape or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous int32 tensor of one entry more than sequences "
                                 f"(got {t.dtype}, {tuple(t.shape)})")
        if cu_seqlens_k is None and keys[0] != shape[0]:
            raise ValueError(f"{keys[0]} keys for {shape[0]} queries need cu_seqlens_k")
    elif cu_seqlens_k is not None:
        raise ValueError("cu_seqlens_k goes with cu_seqlens")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not dtype or out.stride(-1) != 1:
        raise ValueError("out must have the shape and dtype of q, and unit stride along the head dim")
    q, k, v = _walkable("q", q), _walkable("k", k), _walkable("v", v)
    lse = torch.empty(shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    K.prompt_attn(q, k, v, cu_seqlens, cu_seqlens if cu_seqlens_k is None else cu_seqlens_k, bool(causal),
                  q.shape[-1] ** -0.5 if scale is None else float(scale), out, lse)
    return (out, lse) if return_lse else out


__all__ = ["prompt_attention"]
