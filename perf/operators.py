"""Cases and plain forms of the paged 4-bit KV cache operators.

The operators: `append` (norm of query and key heads, rotary positions, 4-bit
quantisation and the write into the pages of the cache, in one pass), `read`
(the values the cache holds, gathered back), `attend` (attention of one or a few
new tokens over the cache) and `select` (pages chosen by a bound on their
scores, and the attention over those pages alone).

The cache, in its plain form: codes int8 in -7..7 of shape (pages, page_size,
Hk, D) and one fp16 scale for every 32 channels of a token, for K and V each;
for every page and KV head, int8 bounds (2, D) of its keys with one power of two.
A sequence owns the pages that its row of the page table names.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one chat user's decode step on a 16/8-head model: a single token goes in, latency counts
        {"name": "append_1x1", "op": "append", "dtype": "bf16", "B": 1, "new": 1, "ctx": 517,
         "ragged": False, "Hq": 16, "Hk": 8, "D": 128, "page": 64, "rot": 128, "interleaved": False, "norm": True},
        # the decode step of a full serving batch (64 sequences), each at its own odd length
        {"name": "append_64x1", "op": "append", "dtype": "bf16", "B": 64, "new": 1, "ctx": 1500,
         "ragged": False, "Hq": 16, "Hk": 8, "D": 128, "page": 64, "rot": 128, "interleaved": False, "norm": True},
        # a packed prefill of 7 prompts, some continuing earlier chunks, on a 32/8-head model
        {"name": "append_prefill_8191", "op": "append", "dtype": "bf16", "B": 7, "new": 8191, "ctx": 700,
         "ragged": True, "Hq": 32, "Hk": 8, "D": 128, "page": 64, "rot": 128, "interleaved": False, "norm": True},
        # prefill of a model without head norms that rotates a quarter of a 64-wide head in pairs
        {"name": "append_pairs_fp16_2900", "op": "append", "dtype": "fp16", "B": 3, "new": 2900, "ctx": 40,
         "ragged": True, "Hq": 14, "Hk": 2, "D": 64, "page": 16, "rot": 16, "interleaved": True, "norm": False},
        # decode attention of one chat user: latency
        {"name": "attend_1x517", "op": "attend", "dtype": "bf16", "B": 1, "len": 517, "ragged": False,
         "Sq": 1, "Hq": 16, "Hk": 8, "D": 128, "page": 64},
        # the long-context decode batch: 16 sequences of 32768 tokens, 32/8 heads, one layer
        {"name": "attend_16x32768", "op": "attend", "dtype": "bf16", "B": 16, "len": 32768, "ragged": False,
         "Sq": 1, "Hq": 32, "Hk": 8, "D": 128, "page": 64},
        # continuous batching: 61 sequences from one token to 12000, 7 query heads to a KV head
        {"name": "attend_ragged_fp16", "op": "attend", "dtype": "fp16", "B": 61, "len": 12000, "ragged": True,
         "Sq": 1, "Hq": 14, "Hk": 2, "D": 64, "page": 32},
        # verification of 4 drafted tokens for 24 sequences in the middle of their contexts
        {"name": "attend_verify4", "op": "attend", "dtype": "bf16", "B": 24, "len": 9000, "ragged": True,
         "Sq": 4, "Hq": 32, "Hk": 8, "D": 128, "page": 64},
        # sparse decode at 131072 tokens: 64 of each head's 2048 pages
        {"name": "select_4x131072", "op": "select", "dtype": "bf16", "B": 4, "len": 131072, "ragged": False,
         "count": 64, "Hq": 32, "Hk": 8, "D": 128, "page": 64},
        # sparse decode of a ragged fp16 batch with small pages, some shorter than the selection
        {"name": "select_ragged_fp16", "op": "select", "dtype": "fp16", "B": 19, "len": 20000, "ragged": True,
         "count": 48, "Hq": 16, "Hk": 8, "D": 128, "page": 32},
        # the held prefix of one prompt, for the attention of its next chunk
        {"name": "read_1x900", "op": "read", "dtype": "bf16", "B": 1, "len": 900, "ragged": False,
         "Hk": 8, "D": 128, "page": 64},
        # the same for a batch of long prompts of different lengths
        {"name": "read_4x20000", "op": "read", "dtype": "bf16", "B": 4, "len": 20000, "ragged": True,
         "Hk": 8, "D": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "select", "read"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([64, 96, 128, 128, 256])
    Hk = rng.choice([1, 2, 3, 5, 8])
    G = rng.choice([1, 2, 3, 4, 7, 8])
    c = {"op": op, "dtype": dtype, "Hk": Hk, "D": D, "page": rng.choice([16, 32, 64, 128])}
    row = Hk * D
    if op == "append":
        B = _log(rng, 1, 64)
        ragged = rng.random() < 0.5
        new = max(B, _log(rng, B, 8191)) if ragged else _log(rng, 1, 16)
        G = min(G, max(1, 4096 // row))
        rot = rng.choice([0, D // 2 // 16 * 16, D])
        c.update(B=B, new=new, ctx=_log(rng, 1, 1500), ragged=ragged, Hq=Hk * G, rot=rot,
                 interleaved=rng.random() < 0.5, norm=rng.random() < 0.5)
    elif op == "attend":
        B = _log(rng, 1, 64)
        n = _log(rng, 1, min(32768, 16 * 32768 * 1024 // 4 // (B * row)))
        c.update(B=B, len=n, ragged=rng.random() < 0.7, Sq=rng.choice([1, 1, 1, 2, 4]), Hq=Hk * G)
    elif op == "select":
        B = _log(rng, 1, 24)
        n = _log(rng, 100, min(131072, 4 * 131072 * 1024 // (B * row)))
        c.update(B=B, len=n, ragged=rng.random() < 0.7, count=_log(rng, 4, 64), Hq=Hk * G)
    else:
        B = _log(rng, 1, 16)
        n = _log(rng, 1, min(20000, 4 * 20000 * 1024 // 2 // (B * row)))
        c.update(B=B, len=n, ragged=rng.random() < 0.7)
    return c


def _lengths(B, n, ragged):
    """Tokens of each sequence: all `n`, or spread over 1..n (logarithmically), the last one of n.
    The same for every seed, so that outputs keep their shapes; prepare() shuffles the sequences."""
    if not ragged:
        return torch.full((B,), n, dtype=torch.int64)
    g = torch.Generator().manual_seed(1000 * n + B)
    x = torch.exp(torch.rand(B, generator=g, dtype=torch.float64) * math.log(n)).round().long()
    x[-1] = n
    return x.clamp(1, n)


def _new(case):
    """New tokens of each sequence in an append: `new` each, or `new` in all with one at least for each."""
    B, n = case["B"], case["new"]
    if not case["ragged"]:
        return torch.full((B,), n)
    g = torch.Generator().manual_seed(1000 * n + B)
    cut = torch.randperm(n - 1, generator=g)[: B - 1].sort().values + 1
    return torch.diff(cut, prepend=torch.zeros(1, dtype=cut.dtype), append=torch.tensor([n]))


def work(case):
    op, Hk, D, e = case["op"], case["Hk"], case["D"], BYTES[case["dtype"]]
    held = 2 * Hk * (D // 2 + D // 32 * 2)  # bytes of the cache for one token
    if op == "append":
        T = case["new"] if case["ragged"] else case["new"] * case["B"]
        rows = T * D * e
        n = rows * 2 * case["Hq"] + rows * 2 * Hk  # q in and out, k and v in
        n += T * case["rot"] * 4 + T * held + rows * 2 * Hk  # positions, the cache, the values read back
        return {"bytes": n, "flops": 10 * T * (case["Hq"] + 2 * Hk) * D}
    lens = _lengths(case["B"], case["len"], case["ragged"])
    L = int(lens.sum())
    if op == "read":
        return {"bytes": L * (held + 2 * Hk * D * e), "flops": 2 * L * Hk * D}
    Sq = case.get("Sq", 1)
    n = 2 * case["B"] * Sq * case["Hq"] * D * e + case["B"] * 4
    if op == "select":
        pages = int(((lens + case["page"] - 1) // case["page"]).sum())
        kept = int(lens.clamp(max=case["count"] * case["page"]).sum())
        return {"bytes": n + pages * Hk * (2 * D + 4) + kept * held,
                "flops": 4 * pages * Hk * D + 4 * kept * case["Hq"] * D}
    return {"bytes": n + L * held, "flops": 4 * L * Sq * case["Hq"] * D}


# ------------------------------------------------------- the format, in torch
def _tree(x):
    """Sum over the last axis, neighbours first: the order the operator defines."""
    n = x.shape[-1]
    if n == 1:
        return x[..., 0]
    if n % 2:
        x = torch.cat([x, torch.zeros_like(x[..., :1])], -1)
    return _tree(x[..., 0::2] + x[..., 1::2])


def _quantise(x):
    """fp32 (..., D) -> codes int8 (..., D), scales fp16 (..., D / 32)."""
    g = x.unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1) * (1.0 / 7.0)).clamp(max=65504.0).half()
    f = s.float()
    x = torch.where(f[..., None] > 0, g / f[..., None], torch.zeros_like(g))
    return torch.round(x).clamp(-7, 7).to(torch.int8).flatten(-2), s


def _values(codes, scales):
    return (codes.float().unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def _exponent(amax, least=-40):
    """The smallest integer e >= least with amax <= 127 * 2^e."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 127.0 / 128.0, x - 7, x - 6).clamp(min=least)
    return torch.where(amax > 0, e, torch.full_like(e, least)).to(torch.int32)


def _bounds(codes, scales, valid):
    """codes (n, P, Hk, D), valid (n, P) -> bounds int8 (n, Hk, 2, D), exponents int32 (n, Hk)."""
    x = _values(codes, scales)
    m = valid[:, :, None, None]
    lo = torch.where(m, x, torch.full_like(x, math.inf)).amin(1)
    hi = torch.where(m, x, torch.full_like(x, -math.inf)).amax(1)
    e = _exponent(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    f = torch.exp2(-e.float())[..., None]
    return torch.stack([torch.floor(lo * f), torch.ceil(hi * f)], 2).to(torch.int8), e


# ------------------------------------------------------------------ the inputs
def _pages(case, lens, g, dev):
    """(page table (B, n) int32 with -1 where a sequence has no page, number of pages)."""
    P = case["page"]
    need = (lens + P - 1) // P
    total = int(need.sum()) + 2
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    width = int(need.max())
    col = torch.arange(width)
    at = (torch.cumsum(need, 0) - need)[:, None] + col
    table = ids[at.clamp(max=total - 1).to(dev)]
    table[(col[None] >= need[:, None]).to(dev)] = -1
    return table, total


def _tokens(n, Hk, D, g, dev, keys):
    """Keys or values: channels of different spread, neighbours alike, a few key channels far larger."""
    s = torch.exp(0.5 * torch.randn(Hk, D, generator=g, device=dev))
    if keys:
        s[:, :4] *= 10.0
    slow = torch.randn(n // 48 + 1, Hk, D, generator=g, device=dev)
    x = slow.repeat_interleave(48, 0)[:n] * 0.8
    x += 0.6 * torch.randn(n, Hk, D, generator=g, device=dev)
    return x * s


def _make(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, B, Hk, D, P, dt = case["op"], case["B"], case["Hk"], case["D"], case["page"], DTYPES[case["dtype"]]
    s = dict(case)
    mix = torch.randperm(B, generator=torch.Generator().manual_seed(int(seed)))
    if op == "append":
        new = _new(case)[mix]
        shape = (case["new"],) if case["ragged"] else (B, case["new"])
        if case["ragged"]:
            s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(dev, torch.int32)
        held = _lengths(B, case["ctx"], B > 1)[mix]
        cap = held + new
        for name, H in (("q", case["Hq"]), ("k", Hk), ("v", Hk)):
            s[name] = torch.randn(*shape, H, D, generator=g, device=dev).to(dt)
        s["k"] = (s["k"].float() * torch.exp(0.5 * torch.randn(Hk, D, generator=g, device=dev))).to(dt)
        if case["norm"]:
            s["qw"] = (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dt)
            s["kw"] = (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dt)
        if case["rot"]:
            R = case["rot"]
            f = 1.0 / (10000.0 ** (torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R))
            a = torch.arange(int(cap.max()), device=dev, dtype=torch.float64)[:, None] * f
            s["rotary"] = torch.cat([a.cos(), a.sin()], 1).float()
    else:
        held = cap = _lengths(B, case["len"], case["ragged"])[mix]
        if op in ("attend", "select"):
            lead = (B, case["Sq"]) if case.get("Sq", 1) > 1 else (B,)
            s["q"] = torch.randn(*lead, case["Hq"], D, generator=g, device=dev).to(dt)
        if op == "read" and case["ragged"]:
            s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), held.cumsum(0)]).to(dev, torch.int32)
        s["total"] = int(held.sum())
    s["table"], pages = _pages(case, cap, g, dev)
    s["lens"] = held.to(dev, torch.int32)
    for name in ("k", "v"):
        s[name + "_codes"] = torch.zeros(pages, P, Hk, D, dtype=torch.int8, device=dev)
        s[name + "_scales"] = torch.zeros(pages, P, Hk, D // 32, dtype=torch.float16, device=dev)
    s["bounds"] = torch.zeros(pages, Hk, 2, D, dtype=torch.int8, device=dev)
    s["exps"] = torch.zeros(pages, Hk, dtype=torch.int32, device=dev)
    for b, n in enumerate(held.tolist()):
        ids = s["table"][b, : (n + P - 1) // P].long()
        valid = (torch.arange(len(ids) * P, device=dev) < n).view(-1, P)
        for name in ("k", "v"):
            codes, scales = _quantise(_tokens(len(ids) * P, Hk, D, g, dev, name == "k"))
            s[name + "_codes"][ids] = codes.view(-1, P, Hk, D) * valid[:, :, None, None]
            s[name + "_scales"][ids] = scales.view(-1, P, Hk, D // 32) * valid[:, :, None, None]
        if op in ("append", "select"):
            s["bounds"][ids], s["exps"][ids] = _bounds(s["k_codes"][ids], s["k_scales"][ids], valid)
    return s


def prepare(case, seed):
    s = _make(case, seed)
    if not own:
        return s
    import flashcodec_b200 as fc

    P, dev = case["page"], s["lens"].device
    cache = fc.PagedInt4Cache(s["k_codes"].shape[0], case["Hk"], case["D"], page_size=P,
                              bounds=case["op"] in ("append", "select"), device=dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    for b, n in enumerate(s["lens"].tolist()):  # the same content, appended as values
        ids = s["table"][b, : (n + P - 1) // P].long()
        k = _values(s["k_codes"][ids], s["k_scales"][ids]).flatten(0, 1)[None, :n]
        v = _values(s["v_codes"][ids], s["v_scales"][ids]).flatten(0, 1)[None, :n]
        cache.append(None, k, v, s["table"][b:b + 1], zero)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "bounds", "exps"):
        del s[name]
    s["cache"] = cache
    return s


# ------------------------------------------------------------- the plain forms
def _head_norm(x, w, eps=1e-6):
    r = 1.0 / torch.sqrt(_tree(x * x) * (1.0 / x.shape[-1]) + eps)
    return x * r[..., None] * w.float()


def _rotate(x, cs, interleaved):
    R = cs.shape[-1]
    c, s = cs[:, None, : R // 2], cs[:, None, R // 2:]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2: R]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., R:]], -1)


def _places(s, T, B):
    """Of T new tokens: the sequence, the position, the page and the row in it."""
    dev = s["lens"].device
    i = torch.arange(T, device=dev)
    if "cu" in s:
        cu = s["cu"].long()
        b = torch.searchsorted(cu[1:], i, right=True)
        pos = i - cu[b]
    else:
        b = i // (T // B)
        pos = i % (T // B)
    if s["op"] == "append":
        pos = pos + s["lens"].long()[b]
    return b, pos, s["table"].long()[b, pos // s["page"]], pos % s["page"]


def _plain_append(s):
    B, P = s["B"], s["page"]
    q, k, v = (s[n].float().flatten(0, -3) for n in ("q", "k", "v"))
    b, pos, page, row = _places(s, k.shape[0], B)
    if s["norm"]:
        q, k = _head_norm(q, s["qw"]), _head_norm(k, s["kw"])
    if s["rot"]:
        cs = s["rotary"][pos]
        q, k = _rotate(q, cs, s["interleaved"]), _rotate(k, cs, s["interleaved"])
    out = {"q": q.to(s["q"].dtype).view(s["q"].shape)}
    s["k_codes"][page, row], s["k_scales"][page, row] = _quantise(k)
    s["v_codes"][page, row], s["v_scales"][page, row] = _quantise(v)
    # the pages that got tokens, with what they held before
    end = torch.zeros(s["k_codes"].shape[0], dtype=torch.int64, device=q.device)
    end = end.scatter_reduce(0, page, row + 1, "amax")
    ids = end.nonzero()[:, 0]
    valid = torch.arange(P, device=q.device) < end[ids, None]
    s["bounds"][ids], s["exps"][ids] = _bounds(s["k_codes"][ids], s["k_scales"][ids], valid)
    for n in ("k", "v"):
        x = _values(s[n + "_codes"][page, row], s[n + "_scales"][page, row])
        out[n] = x.to(s["q"].dtype).view(s["k"].shape)
    return out | {"bounds": s["bounds"], "exps": s["exps"]}


def _plain_read(s):
    B, dt = s["B"], DTYPES[s["dtype"]]
    _, _, page, row = _places(s, s["total"], B)
    shape = (s["total"],) if "cu" in s else (B, s["total"] // B)
    return {n: _values(s[n + "_codes"][page, row], s[n + "_scales"][page, row]).to(dt).view(
        *shape, s["Hk"], s["D"]) for n in ("k", "v")}


def _softmax_product(q, k, v, visible):
    """q (B, S, Hk, G, D), k and v (B, Hk, L, D), visible (B, Hk or 1, S, L) -> (B, S, Hk, G, D)."""
    a = torch.einsum("bshgd,bhld->bhsgl", q * q.shape[-1] ** -0.5, k)
    a = a.masked_fill(~visible[:, :, :, None], -math.inf)
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(top.isinf(), torch.zeros_like(top), top))
    n = e.sum(-1, keepdim=True)
    e = e / torch.where(n > 0, n, torch.ones_like(n))
    return torch.einsum("bhsgl,bhld->bshgd", e, v)


def _plain_attend(s):
    q = s["q"].float() if s["q"].dim() == 4 else s["q"].float()[:, None]
    B, S, Hq, D = q.shape
    pages = s["table"].long().clamp(min=0)
    k, v = (_values(s[n + "_codes"][pages], s[n + "_scales"][pages]).flatten(1, 2).transpose(1, 2)
            for n in ("k", "v"))
    seen = s["lens"].long()[:, None] - torch.arange(S - 1, -1, -1, device=q.device)
    visible = torch.arange(k.shape[2], device=q.device) < seen[:, :, None]
    out = _softmax_product(q.view(B, S, s["Hk"], -1, D), k, v, visible[:, None])
    return out.reshape(s["q"].shape).to(s["q"].dtype)


def _plain_select(s):
    q, Hk, P, count = s["q"].float(), s["Hk"], s["page"], s["count"]
    B, Hq, D = q.shape
    x = q.view(B, Hk, Hq // Hk, D)
    # the query in whole numbers of a power of two shared by the group's heads
    e = _exponent(x.abs().amax((2, 3)), -100) + max(0, math.ceil(math.log2(Hq // Hk * D / 1024)))
    z = torch.round(x * torch.exp2(-e.float())[:, :, None, None])
    up, down = z.clamp(min=0).sum(2), z.clamp(max=0).sum(2)
    pages = s["table"].long().clamp(min=0)
    bound = s["bounds"][pages].float()  # (B, pages, Hk, 2, D)
    score = torch.einsum("bhd,bphd->bhp", down, bound[:, :, :, 0])
    score = score + torch.einsum("bhd,bphd->bhp", up, bound[:, :, :, 1])  # whole numbers under 2^24
    score = score * torch.exp2(s["exps"][pages].float()).transpose(1, 2)
    n = (s["lens"].long() + P - 1) // P
    at = torch.arange(pages.shape[1], device=q.device)
    score = score.masked_fill((at < 1) | (at >= n[:, None, None] - 1), math.inf)  # the first and the last page stay
    score = score.masked_fill(at >= n[:, None, None], -math.inf)
    top = torch.sort(score, dim=-1, descending=True, stable=True)
    top = torch.where(top.values > -math.inf, top.indices, torch.full_like(top.indices, pages.shape[1]))
    top = top[..., :count].sort(-1).values
    held = top < pages.shape[1]
    at = top.clamp(max=pages.shape[1] - 1)  # (B, Hk, count)
    ids = torch.gather(pages[:, None].expand(-1, Hk, -1), 2, at)
    head = torch.arange(Hk, device=q.device)[:, None]
    k, v = (_values(s[w + "_codes"].transpose(1, 2)[ids, head], s[w + "_scales"].transpose(1, 2)[ids, head])
            .flatten(2, 3) for w in ("k", "v"))
    pos = at[..., None] * P + torch.arange(P, device=q.device)
    visible = ((pos < s["lens"].long()[:, None, None, None]) & held[..., None]).flatten(2)
    out = _softmax_product(x[:, None], k, v, visible[:, :, None])
    chosen = torch.where(held, top, torch.full_like(top, -1)).to(torch.int32)
    if chosen.shape[2] < count:
        chosen = torch.cat([chosen, chosen.new_full((B, Hk, count - chosen.shape[2]), -1)], -1)
    return {"out": out.reshape(B, Hq, D).to(s["q"].dtype), "pages": chosen}


def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend,
                "select": _plain_select}[s["op"]](s)
    cache = s["cache"]
    if s["op"] == "append":
        q = cache.append(s["q"], s["k"], s["v"], s["table"], s["lens"], cu_seqlens=s.get("cu"),
                         q_weight=s.get("qw"), k_weight=s.get("kw"), rotary=s.get("rotary"),
                         interleaved=s["interleaved"])
        k, v = cache.read(s["table"], s["lens"], cu_seqlens=s.get("cu"), dtype=s["q"].dtype,
                          count=s["new"])
        return {"q": q, "k": k, "v": v, "bounds": cache.bounds, "exps": cache.exponents}
    if s["op"] == "read":
        k, v = cache.read(s["table"], None, cu_seqlens=s.get("cu"), dtype=DTYPES[s["dtype"]],
                          count=s["total"] if "cu" in s else s["total"] // s["B"])
        return {"k": k, "v": v}
    if s["op"] == "attend":
        return cache.attend(s["q"], s["table"], s["lens"])
    pages = cache.select(s["q"], s["table"], s["lens"], s["count"], sink=1, recent=1)
    return {"out": cache.attend(s["q"], s["table"], s["lens"], selected=pages), "pages": pages}


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = _make(case, seed)
    P, D, Hk = case["page"], case["D"], case["Hk"]
    lens = s["lens"].tolist()

    def held(name, b, lo, hi):  # (hi - lo, Hk, D) of sequence b, in 64 bits
        ids = s["table"][b, : (hi + P - 1) // P].long()
        c = s[name + "_codes"][ids].flatten(0, 1)[lo:hi].double()
        f = s[name + "_scales"][ids].flatten(0, 1)[lo:hi].double()
        return (c.view(hi - lo, Hk, D // 32, 32) * f[..., None]).view(hi - lo, Hk, D)

    if case["op"] == "read":
        x = {n: torch.cat([held(n, b, 0, m) for b, m in enumerate(lens)]) for n in ("k", "v")}
        return x if "cu" in s else {n: y.view(case["B"], -1, Hk, D) for n, y in x.items()}

    if case["op"] == "append":
        B = case["B"]
        cu = s["cu"].tolist() if "cu" in s else [b * case["new"] for b in range(B + 1)]

        def turned(x, w, b, on):  # tokens of one sequence: normed and rotated
            x = x.double()
            if case["norm"] and on:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
            R = case["rot"]
            if R and on:
                t = s["rotary"][lens[b]: lens[b] + len(x)].double()
                z = torch.complex(t[:, : R // 2], t[:, R // 2:])[:, None]
                if case["interleaved"]:
                    y = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * z
                    y = torch.view_as_real(y).reshape(*x.shape[:-1], R)
                else:
                    y = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * z
                    y = torch.cat([y.real, y.imag], -1)
                x = torch.cat([y, x[..., R:]], -1)
            return x

        def kept(x):  # the values that 4 bits hold for x
            y = x.view(*x.shape[:-1], D // 32, 32)
            f = (y.abs().amax(-1, keepdim=True) / 7).half().double()
            c = torch.where(f > 0, y / torch.where(f > 0, f, torch.ones_like(f)), torch.zeros_like(y))
            return (c.round().clamp(-7, 7) * f).view_as(x)

        out = {}
        for n, w in (("q", "qw"), ("k", "kw"), ("v", None)):
            flat = s[n].flatten(0, -3)
            rows = [turned(flat[cu[b]: cu[b + 1]], s.get(w), b, n != "v") for b in range(B)]
            rows = torch.cat(rows)
            out[n] = (rows if n == "q" else kept(rows)).view(s[n].shape)
        return out | {"bounds": None, "exps": None}

    G = case["Hq"] // Hk
    q = s["q"].double()
    q = q if q.dim() == 4 else q[:, None]
    out = torch.zeros_like(q)
    chosen = []
    for b, n in enumerate(lens):
        k, v = held("k", b, 0, n), held("v", b, 0, n)
        S = q.shape[1]
        if case["op"] == "select":
            m = -(-n // P)
            ids = s["table"][b, :m].long()
            lo, hi = s["bounds"][ids].double().unbind(2)  # (m, Hk, D)
            unit = torch.exp2(s["exps"][ids].double())
            keep = torch.zeros(Hk, m, dtype=torch.bool, device=q.device)
            for h in range(Hk):
                x = q[b, 0, h * G: (h + 1) * G]
                top = float(x.abs().max())
                e = -100
                if top > 0:
                    f, e = math.frexp(top)
                    e = max(-100, e - 7 if f <= 127 / 128 else e - 6)
                e += max(0, math.ceil(math.log2(G * D / 1024)))
                z = torch.round(x * 2.0 ** -e)
                best = torch.maximum(z[:, None] * lo[None, :, h], z[:, None] * hi[None, :, h]).sum((0, 2)) * unit[:, h]
                order = sorted(range(m), key=lambda p, t=best.tolist(): (not (p == 0 or p == m - 1), -t[p], p))
                keep[h, torch.tensor(order[: case["count"]], device=q.device)] = True
            chosen.append([torch.nonzero(keep[h])[:, 0].tolist() for h in range(Hk)])
            see = keep.repeat_interleave(P, 1)[:, :n]
        for t in range(S):
            m = n - (S - 1 - t)
            if m <= 0:
                continue
            a = torch.einsum("hgd,lhd->hgl", q[b, t].view(Hk, G, D), k[:m]) / math.sqrt(D)
            if case["op"] == "select":
                a = a.masked_fill(~see[:, None, :m], -math.inf)
            out[b, t] = torch.einsum("hgl,lhd->hgd", torch.softmax(a, -1), v[:m]).reshape(-1, D)
    out = out.view(s["q"].shape)
    if case["op"] == "attend":
        return out
    full = [[p + [-1] * (case["count"] - len(p)) for p in row] for row in chosen]
    return {"out": out, "pages": torch.tensor(full, dtype=torch.int32, device=q.device)}
