"""A paged 4-bit KV cache for batches of sequences that come and go.

The codec streams (``cache.py``) hold one batch that grows in step.  A serving
engine instead keeps one pool of pages per layer and a table that says which
pages a sequence owns; sequences join, grow by different amounts and leave.
``PagedInt4Cache`` is that pool for one layer: K and V as 4-bit codes with one
fp16 scale for each token and 32 channels (4.5 bits a value), and the four
operations on it:

* ``append``  -- new tokens in: RMS norm of the query and key heads, rotary
  positions, quantisation and the page write, one launch;
* ``attend``  -- attention of the newest token(s) of every sequence, one launch;
* ``select``  -- the pages of a long context worth attending to, by a bound on
  the scores of the rounded queries; ``attend(..., selected=pages)`` reads only those;
* ``read``    -- the values held, gathered back (the prefix of a prompt's next
  chunk).

    cache = PagedInt4Cache(num_pages, num_kv_heads, head_dim)
    table = rotary_table(131072, head_dim, base=1e6)
    q = cache.append(q, k, v, page_table, lengths, q_weight=wq, k_weight=wk, rotary=table)
    lengths += 1
    out = cache.attend(q, page_table, lengths)

``page_table`` (B, n) and ``lengths`` (B,) are int32 CUDA tensors which the
kernels read when they run: a captured CUDA graph follows their contents.  The
caller owns page allocation; entries past a sequence's pages are never read.
Kernels check pages, lengths and positions against the buffers: tokens without a
page are skipped, positions outside the rotary table take its nearest row, and
either is noted in ``status`` (see ``check``).  The
reference has no paged cache; its notes on 4-bit K/V quantisation
(docs/llama-cpp-kv-quantization.md) are the nearest it has.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _kernels as K
from . import _lib

_STATUS = ((1, "a page outside the pool"),
           (2, "a length or position past what the page table holds, or cu_seqlens past the rows given"),
           (4, "a position outside the rotary table"))


def rotary_table(max_positions, rotary_dim, base=10000.0, *, scaling=None, factor=1.0,
                 original_max_positions=None, low_freq_factor=1.0, high_freq_factor=4.0,
                 beta_fast=32.0, beta_slow=1.0, attention_factor=None, device="cuda"):
    """(max_positions, rotary_dim) fp32: the cosines, then the sines, of every
    position's angles ``position * base ** (-2 i / rotary_dim)``, evaluated in
    fp64 and rounded once.  (``append`` takes multiples of 16 as rotary_dim.)

    scaling: how the frequencies are stretched for contexts ``factor`` times
    ``original_max_positions``:
        None      not at all;
        "linear"  positions divided by ``factor``;
        "ntk"     ``base`` times ``factor ** (R / (R - 2))``;
        "llama3"  wavelengths over ``original / low_freq_factor`` divided by
                  ``factor``, those under ``original / high_freq_factor`` kept,
                  a linear ramp between;
        "yarn"    frequencies of fewer than ``beta_slow`` turns over the original
                  context divided by ``factor``, those of more than ``beta_fast``
                  kept, a linear ramp over the channels between; cosines and
                  sines times ``attention_factor`` (0.1 ln factor + 1).
    """
    R = int(rotary_dim)
    if R <= 0 or R % 2 or max_positions <= 0:
        raise ValueError(f"rotary_dim must be even and positive (got {rotary_dim}), "
                         f"max_positions positive (got {max_positions})")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1 (got {factor})")
    if scaling in ("llama3", "yarn") and not original_max_positions:
        raise ValueError(f"scaling {scaling!r} needs original_max_positions")
    if scaling == "ntk":
        base = base * factor ** (R / max(R - 2, 1))
    freq = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    gain = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "llama3":
        turns = original_max_positions * freq / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    elif scaling == "yarn":
        def channel(turns):  # where a frequency makes so many turns over the original context
            return R * math.log(original_max_positions / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(channel(beta_fast)), 0), min(math.ceil(channel(beta_slow)), R - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        gain = attention_factor if attention_factor is not None else \
            (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown rotary scaling {scaling!r}")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (torch.cat([angle.cos(), angle.sin()], 1) * gain).float()


class PagedInt4Cache:
    """One layer's pool of 4-bit K/V pages.

    Args:
        num_pages: pages of the pool.
        num_kv_heads, head_dim: of the model (head_dim 64, 96, 128, 192 or 256).
        page_size: tokens of a page, a power of two from 16 to 1024.
        bounds: keep every page's least and largest key values per channel,
            which ``select`` needs (2 * head_dim + 4 bytes per page and KV head).
        device: a CUDA device.

    Attributes: ``pool`` (num_pages, bytes) uint8; ``bounds`` (num_pages, Hk, 2,
    D) int8 and ``exponents`` (num_pages, Hk) int32, or None; ``status`` int32.
    They cannot be replaced, only written to (a cache restored from a file:
    ``cache.pool.copy_(saved)``).
    """

    def __init__(self, num_pages, num_kv_heads, head_dim, page_size=64, bounds=False,
                 device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("flashcodec_b200 runs on CUDA devices only (got "
                               f"{dev}); there is no CPU implementation")
        if num_pages <= 0 or num_pages > 0x7fffffff:
            raise ValueError(f"num_pages must be positive (got {num_pages})")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        self.num_pages, self.num_kv_heads = int(num_pages), int(num_kv_heads)
        self.head_dim, self.page_size = int(head_dim), int(page_size)
        self.page_bytes = K.kv4_page_bytes(self.num_kv_heads, self.head_dim, self.page_size)
        self._pool = torch.empty(self.num_pages, self.page_bytes, dtype=torch.uint8, device=dev)
        self._bounds = self._exponents = None
        if bounds:
            self._bounds = torch.zeros(self.num_pages, self.num_kv_heads, 2, self.head_dim,
                                       dtype=torch.int8, device=dev)
            self._exponents = torch.zeros(self.num_pages, self.num_kv_heads, dtype=torch.int32,
                                          device=dev)
        self._status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._index, self._scale, self._lib = dev.index, self.head_dim ** -0.5, _lib.load()
        self._status_ptr = self._status.data_ptr()
        self._pool_args = (self._pool.data_ptr(), self.num_pages, self.num_kv_heads, self.head_dim,
                           self.page_size)
        self._bounds_args = (self._bounds.data_ptr(), self._exponents.data_ptr()) if bounds \
            else (None, None)

    # The calls pass these tensors' addresses, taken once: their contents may be written, they
    # themselves stay.
    pool = property(lambda self: self._pool)
    bounds = property(lambda self: self._bounds)
    exponents = property(lambda self: self._exponents)
    status = property(lambda self: self._status)

    # ------------------------------------------------------------ argument checks
    # (a decode step calls these for every layer: each looks at a tensor's attributes once)
    def _here(self, *tensors):
        """Tensors (or None) on the cache's device, none asking for a gradient or with a tangent."""
        index, grad = self._index, torch.is_grad_enabled()
        dual = getattr(forward_ad, "_current_level", 0) >= 0  # inside a dual level
        for t in tensors:
            if t is None:
                continue
            if t.get_device() != index:
                K.require_cuda(t)
                raise ValueError(f"a tensor is on {t.device}, the cache on {self.device}")
            if grad and t.requires_grad:
                raise RuntimeError("the 4-bit cache holds rounded values and has no gradient: "
                                   "call it under torch.no_grad()")
            if dual and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the 4-bit cache holds rounded values and has no tangent: "
                                   "pass the primal of a dual tensor")

    def _ints(self, name, t, shape):
        if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} "
                             f"(got {t.dtype}, {tuple(t.shape)})")

    def _table(self, page_table):
        """(address, row stride, columns) of a page table, and its rows."""
        s = page_table.shape
        if page_table.dtype is not torch.int32 or len(s) != 2 or s[1] == 0:
            raise ValueError("page_table must be an int32 (B, n) tensor")
        st = page_table.stride()
        if st[1] != 1 and s[1] > 1:
            raise ValueError("page_table must have unit stride along n")
        return s[0], (page_table.data_ptr(), st[0], s[1])

    def _rows(self, name, t, shape=None, packed=False, heads=None):
        """(address, sequence, token and head strides) of (B, S, H, D), (B, H, D) or packed
        (T, H, D) rows."""
        s, st = t.shape, t.stride()
        n = len(s)
        if n not in (3, 4) or (packed and n != 3) or s[-1] != self.head_dim \
                or (heads is not None and s[-2] != heads) or (shape is not None and s != shape):
            want = tuple(shape) if shape is not None else (..., heads or "heads", self.head_dim)
            raise ValueError(f"{name}: expected {want}, got {tuple(s)}")
        if st[-1] != 1:
            raise ValueError(f"{name}: the head dim must have unit stride")
        if n == 4:
            return t.data_ptr(), st[0], st[1], st[2]
        return (t.data_ptr(), 0, st[0], st[1]) if packed else (t.data_ptr(), st[0], 0, st[1])

    # ----------------------------------------------------------------- operations
    def append(self, q, k, v, page_table, lengths, *, cu_seqlens=None, q_weight=None,
               k_weight=None, eps=1e-6, rotary=None, interleaved=False, positions=None,
               q_out=None):
        """Put new tokens at the ends of their sequences; returns the queries.

        q, k, v: (B, S, H, D), (B, H, D) for one token each, or packed (T, H, D)
            with ``cu_seqlens`` (B + 1,) int32; fp32, bf16 or fp16, any strides
            with unit stride along D.  q may be None.  Packed rows of no sequence
            (from cu_seqlens[B] on: a captured batch has a fixed number) are not
            stored, and their queries come out as zeros.
        lengths: (B,) int32, tokens held before the call (unchanged by it); a
            negative one skips the sequence.
        q_weight, k_weight: (D,) weights of a per-head RMS norm (``eps``), or None.
        rotary: ``rotary_table``'s (positions, R) fp32, R a multiple of 16, or
            None; its first R channels turn, in pairs (i, i + R/2), or (2i, 2i+1)
            with ``interleaved``.
        positions: (B, S) or (T,) int32 rows of the table (default: the cache
            positions, lengths + i).
        q_out: where the queries go (default: a new tensor; may be q).

        Arithmetic is fp32 and rounded in a fixed order, so what is stored does
        not depend on how tokens are split into calls.
        """
        self._here(q, k, v, page_table, lengths, cu_seqlens, q_weight, k_weight, rotary, positions,
                   q_out)
        B, table = self._table(page_table)
        packed = cu_seqlens is not None
        k_at = self._rows("k", k, packed=packed, heads=self.num_kv_heads)
        shape, dtype = k.shape, k.dtype
        v_at = self._rows("v", v, shape, packed)
        if v.dtype is not dtype:
            raise ValueError("k and v must have one dtype")
        cu = None
        if packed:
            self._ints("cu_seqlens", cu_seqlens, (B + 1,))
            S, T, cu = 0, shape[0], cu_seqlens.data_ptr()
        else:
            S = shape[1] if len(shape) == 4 else 1
            T = B * S
            if shape[0] != B:
                raise ValueError(f"k has {shape[0]} sequences, the page table {B}")
        self._ints("lengths", lengths, (B,))
        q_at, heads = (None, 0, 0, 0, None, 0, 0, 0), 0
        if q is not None:
            q_at, qs = self._rows("q", q, packed=packed), q.shape
            if qs[:-2] != shape[:-2] or q.dtype is not dtype:
                raise ValueError("q must have the tokens and the dtype of k")
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif q_out.dtype is not dtype:
                raise ValueError("q_out must have the dtype of q")
            heads = qs[-2]
            q_at += self._rows("q_out", q_out, qs, packed)
        elif q_out is not None:
            raise ValueError("q_out goes with q")
        w_at, w_dtype = [None, None], None
        for i, w in enumerate((q_weight, k_weight)):
            if w is None:
                continue
            if w.shape != (self.head_dim,) or w.stride(0) != 1:
                raise ValueError(f"norm weights must be contiguous ({self.head_dim},) tensors")
            if w_dtype is not None and w.dtype is not w_dtype:
                raise ValueError("q_weight and k_weight must have one dtype")
            w_at[i], w_dtype = w.data_ptr(), w.dtype
        turn = (None, 0, 0)
        if rotary is not None:
            if rotary.dtype is not torch.float32 or rotary.dim() != 2 or not rotary.is_contiguous():
                raise ValueError("rotary must be a contiguous fp32 (positions, R) tensor")
            turn = (rotary.data_ptr(), *rotary.shape)
        pos = None
        if positions is not None:
            self._ints("positions", positions, shape[:-2] if positions.dim() == 2 else (T,))
            pos = positions.data_ptr()
        K.kv4_append(self, (*q_at, heads, *k_at, *v_at), dtype, B, S, T, cu, lengths.data_ptr(),
                     pos, w_at, w_dtype, eps, turn, bool(interleaved), table)
        return q_out

    def attend(self, q, page_table, lengths, *, scale=None, selected=None, out=None,
               return_lse=False):
        """Attention of every sequence's newest tokens over what the cache holds.

        q: (B, Hq, D), or (B, Sq, Hq, D) for the last Sq tokens of each sequence
            (query i sees lengths - Sq + 1 + i tokens); Hq a multiple of the KV heads.
        lengths: (B,) int32, tokens held, the queries' own among them.
        scale: of the scores (default D ** -0.5).
        selected: (B, Hk, n) int32 from ``select`` (one query per sequence): only
            the tokens of these pages, each named once, count.
        out: where the outputs go (default: a new tensor; may be q).
        Returns the outputs in q's shape and dtype, and with ``return_lse`` the
        natural log of the softmax sums, q.shape[:-1] fp32.  A query that sees no
        token gives zeros (and -inf).
        """
        self._here(q, page_table, lengths, selected, out)
        B, table = self._table(page_table)
        q_at, shape = self._rows("q", q), q.shape
        if shape[0] != B:
            raise ValueError(f"q has {shape[0]} sequences, the page table {B}")
        self._ints("lengths", lengths, (B,))
        if selected is not None:
            if len(shape) == 4 and shape[1] != 1:
                raise ValueError("selected pages go with one query per sequence")
            self._ints("selected", selected, (B, self.num_kv_heads, selected.shape[-1]))
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.dtype is not q.dtype:
            raise ValueError("out must have the dtype of q")
        lse = torch.empty(shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
        K.kv4_attn(self, q_at, q.dtype, shape, table, lengths.data_ptr(), selected,
                   self._scale if scale is None else float(scale), self._rows("out", out, shape), lse)
        return (out, lse) if return_lse else out

    def select(self, q, page_table, lengths, count, *, sink=1, recent=1):
        """(B, Hk, count) int32: for every KV head the pages to attend to, ascending,
        then -1.

        A page's score bounds the sum over the group's query heads of z . k for
        every key in it, z being the group's queries in whole numbers up to 127 of
        one power of two (with 1024 channels of queries and more, of fewer bits).
        The queries themselves may pass it by half a unit of z times the sum of
        the page's largest |keys|: small channels beside one far larger count for
        little.  What the chosen pages hold of the softmax is not bounded.

        The first ``sink`` and last ``recent`` pages of a sequence are always taken,
        the rest by score (ties: the lower index).  q (B, Hq, D).
        The cache needs ``bounds=True``.
        """
        if self.bounds is None:
            raise ValueError("this cache keeps no page bounds (bounds=True)")
        self._here(q, page_table, lengths)
        B, table = self._table(page_table)
        q_at, shape = self._rows("q", q), q.shape
        if len(shape) != 3 or shape[0] != B:
            raise ValueError(f"q must be ({B}, heads, {self.head_dim}) (got {tuple(shape)})")
        self._ints("lengths", lengths, (B,))
        if count <= 0:
            raise ValueError(f"count must be positive (got {count})")
        pages = torch.empty((B, self.num_kv_heads, count), dtype=torch.int32, device=self.device)
        K.kv4_select(self, q_at, q.dtype, B, shape[1], table, lengths.data_ptr(), count, sink, recent,
                     pages.data_ptr())
        return pages

    def read(self, page_table, starts=None, *, count=None, cu_seqlens=None, dtype=torch.bfloat16):
        """The values held, as (k, v): ``count`` tokens of every sequence from
        position ``starts`` ((B,) int32; None: 0) as (B, count, Hk, D), or, with
        ``cu_seqlens``, cu_seqlens[b + 1] - cu_seqlens[b] of sequence b, ``count``
        in all, packed as (count, Hk, D).  Zeros for sequences with a negative
        start, for packed rows of no sequence, and where no page can be read
        (which ``check`` reports)."""
        self._here(page_table, starts, cu_seqlens)
        B, table = self._table(page_table)
        if count is None or count < 0:
            raise ValueError("read needs the number of tokens (count)")
        # (the tensors stay named: a caller's temporary would be freed, and the outputs be put there)
        at = cu = None
        if starts is not None:
            self._ints("starts", starts, (B,))
            at = starts.data_ptr()
        H, D = self.num_kv_heads, self.head_dim
        if cu_seqlens is not None:
            self._ints("cu_seqlens", cu_seqlens, (B + 1,))
            cu = cu_seqlens.data_ptr()
            shape, S, T = (count, H, D), 0, count
        else:
            shape, S, T = (B, count, H, D), count, B * count
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        K.kv4_read(self, table, at, B, S, T, cu, k.data_ptr(), v.data_ptr(), dtype,
                   (count * H * D, H * D, D))
        return k, v

    def check(self):
        """Raise if a kernel met a bad page, length or position since the last
        check, and clear the word (synchronises)."""
        word = int(self.status.item())
        if word:
            self.status.zero_()
            raise _lib.FlashCodecError(_lib.FC_ERANGE, "paged cache: " + "; ".join(
                text for bit, text in _STATUS if word & bit))


__all__ = ["PagedInt4Cache", "rotary_table"]
