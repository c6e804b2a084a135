"""Cases and plain forms of the paged 8-bit KV cache and of attention over whole prompts.

The operators: `append` (norm of query and key heads, rotary positions of one or
several axes, 8-bit quantisation and the write into the pages, in one pass),
`read` (the values the cache holds, gathered back), `attend` (attention of one
or a few new tokens over the cache) and `prompt` (causal attention of packed
prompts, or of chunks of prompts whose keys begin earlier).

The cache: int8 codes (pages, 2, Hk, page_size, D), keys and values, and one fp32
scale, a power of two, for every 16 tokens of a head, (pages, 2, Hk, page_size / 16).
A code stands for (code + 1/2) * scale.  A sequence owns the pages that its row
of the page table names.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 16  # tokens of a scale


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one chat user's decode step on a 16/8-head model: a single token goes in, latency counts
        {"name": "append_1x1", "op": "append", "dtype": "bf16", "B": 1, "new": 1, "ctx": 517, "ragged": False,
         "Hq": 16, "Hk": 8, "D": 128, "page": 64, "rot": 128, "interleaved": False, "norm": True, "axes": 1},
        # the decode step of a full serving batch on a model that rotates a quarter of a 64-wide head in pairs
        {"name": "append_64x1_fp16", "op": "append", "dtype": "fp16", "B": 64, "new": 1, "ctx": 1500, "ragged": False,
         "Hq": 14, "Hk": 2, "D": 64, "page": 16, "rot": 16, "interleaved": True, "norm": False, "axes": 1},
        # a packed prefill of 7 prompts of text and images (time, height and width), some continuing earlier chunks
        {"name": "append_axes_8191", "op": "append", "dtype": "bf16", "B": 7, "new": 8191, "ctx": 700, "ragged": True,
         "Hq": 32, "Hk": 8, "D": 128, "page": 64, "rot": 128, "interleaved": False, "norm": True, "axes": 3},
        # the held prefix of one prompt, for the attention of its next chunk
        {"name": "read_1x900", "op": "read", "dtype": "bf16", "B": 1, "len": 900, "ragged": False,
         "Hk": 8, "D": 128, "page": 64},
        # the same for a batch of long prompts of different lengths
        {"name": "read_4x20000", "op": "read", "dtype": "bf16", "B": 4, "len": 20000, "ragged": True,
         "Hk": 8, "D": 128, "page": 64},
        # decode attention of one chat user: latency
        {"name": "attend_1x517", "op": "attend", "dtype": "bf16", "B": 1, "len": 517, "ragged": False,
         "Sq": 1, "Hq": 16, "Hk": 8, "D": 128, "page": 64},
        # continuous batching: 61 sequences from one token to 12000, 7 query heads to a KV head
        {"name": "attend_ragged_fp16", "op": "attend", "dtype": "fp16", "B": 61, "len": 12000, "ragged": True,
         "Sq": 1, "Hq": 14, "Hk": 2, "D": 64, "page": 32},
        # the long-context decode batch: 16 sequences of 32768 tokens, 32/8 heads, one layer
        {"name": "attend_16x32768", "op": "attend", "dtype": "bf16", "B": 16, "len": 32768, "ragged": False,
         "Sq": 1, "Hq": 32, "Hk": 8, "D": 128, "page": 64},
        # one chat user's prompt on a 16/8-head model: latency
        {"name": "prompt_1x517", "op": "prompt", "dtype": "bf16", "B": 1, "new": 517, "ctx": 0, "ragged": False,
         "Hq": 16, "Hk": 8, "D": 128},
        # chunks of 512 tokens in all, of 3 prompts with up to 30000 tokens before them, 7 query heads to a KV head
        {"name": "prompt_chunks_fp16", "op": "prompt", "dtype": "fp16", "B": 3, "new": 512, "ctx": 30000, "ragged": True,
         "Hq": 14, "Hk": 2, "D": 64},
        # a packed prefill of 7 prompts of different lengths on a 32/8-head model
        {"name": "prompt_packed_8191", "op": "prompt", "dtype": "bf16", "B": 7, "new": 8191, "ctx": 0, "ragged": True,
         "Hq": 32, "Hk": 8, "D": 128},
        # one long document
        {"name": "prompt_1x16384", "op": "prompt", "dtype": "bf16", "B": 1, "new": 16384, "ctx": 0, "ragged": False,
         "Hq": 32, "Hk": 8, "D": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "prompt"])
    D = rng.choice([64, 96, 128, 128, 192, 256])
    Hk = rng.choice([1, 2, 3, 5, 8])
    G = rng.choice([1, 2, 3, 4, 7, 8])
    c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "Hk": Hk, "D": D}
    row = Hk * D
    if op == "prompt":
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
        B = _log(rng, 1, 24)
        ragged = rng.random() < 0.7
        new = _log(rng, max(B, 16), 16384)
        if not ragged:
            new = max(1, new // B)
        G = min(G, max(1, 8192 // row))
        Hq = Hk * G
        # queries * keys * heads * dims stay below those of the largest listed case
        most = 16384 * 8192 * 32 * 128 / (Hq * D)
        ctx = rng.choice([0, 0, _log(rng, 1, 30000)])
        ctx = int(min(ctx, max(0, most / (new if ragged else new * B) - new)))
        c.update(B=B, new=new, ctx=ctx, ragged=ragged, Hq=Hq)
        return c
    c["page"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        B = _log(rng, 1, 64)
        ragged = rng.random() < 0.5
        new = max(B, _log(rng, B, 8191)) if ragged else _log(rng, 1, 16)
        G = min(G, max(1, 4096 // row))
        rot = rng.choice([0, D // 2 // 16 * 16, D])
        c.update(B=B, new=new, ctx=_log(rng, 1, 1500), ragged=ragged, Hq=Hk * G, rot=rot,
                 interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, axes=rng.choice([1, 3]) if rot else 1)
    elif op == "attend":
        B = _log(rng, 1, 64)
        n = _log(rng, 1, min(32768, 16 * 32768 * 1024 // 4 // (B * row)))
        c.update(B=B, len=n, ragged=rng.random() < 0.7, Sq=rng.choice([1, 1, 1, 2, 4]), Hq=Hk * G)
    else:
        B = _log(rng, 1, 16)
        n = _log(rng, 1, min(20000, 4 * 20000 * 1024 // 2 // (B * row)))
        c.update(B=B, len=n, ragged=rng.random() < 0.7)
    return c


def _lengths(B, n, ragged):
    """Tokens of each sequence: all `n`, or spread over 1..n (logarithmically), the last one of n.
    The same for every seed, so that outputs keep their shapes; prepare() shuffles the sequences."""
    if not ragged or n == 0:
        return torch.full((B,), n, dtype=torch.int64)
    g = torch.Generator().manual_seed(1000 * n + B)
    x = torch.exp(torch.rand(B, generator=g, dtype=torch.float64) * math.log(n)).round().long()
    x[-1] = n
    return x.clamp(1, n)


def _new(case):
    """New tokens of each sequence: `new` each, or `new` in all with one at least for each."""
    B, n = case["B"], case["new"]
    if not case["ragged"]:
        return torch.full((B,), n)
    g = torch.Generator().manual_seed(1000 * n + B)
    cut = torch.randperm(n - 1, generator=g)[: B - 1].sort().values + 1
    return torch.diff(cut, prepend=torch.zeros(1, dtype=cut.dtype), append=torch.tensor([n]))


def _cu(n, dev):
    return torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(dev, torch.int32)


def work(case):
    op, Hk, D, e = case["op"], case["Hk"], case["D"], BYTES[case["dtype"]]
    held = 2 * Hk * (D + 4 / BLOCK)  # bytes of the cache for one token
    if op == "prompt":
        new, ctx = _new(case), _lengths(case["B"], case["ctx"], case["B"] > 1)
        T, L = int(new.sum()), int((new + ctx).sum())
        pairs = int((new * ctx + new * (new + 1) // 2).sum())
        return {"bytes": (2 * T * case["Hq"] + 2 * L * Hk) * D * e, "flops": 4 * pairs * case["Hq"] * D}
    if op == "append":
        T = case["new"] if case["ragged"] else case["new"] * case["B"]
        rows = T * D * e
        n = rows * 2 * case["Hq"] + rows * 2 * Hk  # q in and out, k and v in
        n += T * case["rot"] * 4 + T * held + rows * 2 * Hk  # positions, the cache, the values read back
        return {"bytes": int(n), "flops": 10 * T * (case["Hq"] + 2 * Hk) * D}
    L = int(_lengths(case["B"], case["len"], case["ragged"]).sum())
    if op == "read":
        return {"bytes": int(L * (held + 2 * Hk * D * e)), "flops": 2 * L * Hk * D}
    Sq = case["Sq"]
    n = 2 * case["B"] * Sq * case["Hq"] * D * e + case["B"] * 4
    return {"bytes": int(n + L * held), "flops": 4 * L * Sq * case["Hq"] * D}


# ------------------------------------------------------- the format, in torch
def _tree(x):
    """Sum over the last axis, neighbours first: the order the operator defines."""
    n = x.shape[-1]
    if n == 1:
        return x[..., 0]
    if n % 2:
        x = torch.cat([x, torch.zeros_like(x[..., :1])], -1)
    return _tree(x[..., 0::2] + x[..., 1::2])


def _scale(amax):
    """The smallest power of two s >= 2^-126 with amax < 128 s; 0 for zero."""
    e = (torch.frexp(amax).exponent - 7).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax))


def _codes(x, s):
    """floor(x / s) of fp32 x, 0 where s is 0 (in 64 bits: quotients under 2^-149 keep their sign)."""
    f = torch.where(s > 0, s, torch.ones_like(s)).double()
    return torch.floor(x.double() / f).to(torch.int8)


def _values(codes, s):
    return (codes.float() + 0.5) * s


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
    """Keys or values: channels of different spread, neighbours alike, a few key channels larger."""
    s = torch.exp(0.5 * torch.randn(Hk, D, generator=g, device=dev))
    if keys:
        s[:, :4] *= 5.0
    slow = torch.randn(n // 48 + 1, Hk, D, generator=g, device=dev)
    x = slow.repeat_interleave(48, 0)[:n] * 0.8
    x += 0.6 * torch.randn(n, Hk, D, generator=g, device=dev)
    return x * s


def _positions(case, held, new, dev):
    """(3, T) int32: runs of text, whose axes agree, and every other 64 tokens an image of 8 x 8."""
    at = torch.cat([h + torch.arange(n) for h, n in zip(held.tolist(), new.tolist())])
    i = at % 64
    first = at - i
    image = at // 64 % 2 == 1
    axes = [torch.where(image, first + x, at) for x in (torch.zeros_like(i), i // 8, i % 8)]
    return torch.stack(axes).to(dev, torch.int32)


def _sections(case):
    half = case["rot"] // 2
    return (half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8)


def _make(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, B, Hk, D, dt = case["op"], case["B"], case["Hk"], case["D"], DTYPES[case["dtype"]]
    s = dict(case)
    mix = torch.randperm(B, generator=torch.Generator().manual_seed(int(seed)))
    if op == "prompt":
        new = _new(case)[mix]
        ctx = _lengths(B, case["ctx"], B > 1)[mix]
        s["n_q"], s["n_k"] = new.tolist(), (new + ctx).tolist()
        s["cu_q"], s["cu_k"] = _cu(new, dev), _cu(new + ctx, dev)
        T, L = int(new.sum()), int((new + ctx).sum())
        s["q"] = torch.randn(T, case["Hq"], D, generator=g, device=dev).to(dt)
        s["k"] = _tokens(L, Hk, D, g, dev, True).to(dt)
        s["v"] = _tokens(L, Hk, D, g, dev, False).to(dt)
        return s
    P = case["page"]
    if op == "append":
        new = _new(case)[mix]
        held = _lengths(B, case["ctx"], B > 1)[mix]
        cap = held + new
        shape = (case["new"],) if case["ragged"] else (B, case["new"])
        T = int(new.sum())
        s["new_cu"] = _cu(new, dev)
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
            if case["axes"] > 1:
                s["positions"] = _positions(case, held, new, dev).view(3, *shape)
                s["axis"] = torch.repeat_interleave(torch.arange(3), torch.tensor(_sections(case))).to(dev, torch.int32)
        # what is read back: the new tokens, and those before them in their block, whose scale may have grown
        s["from"] = (held // BLOCK * BLOCK).to(dev, torch.int32)
        s["back_cu"] = _cu(new + held % BLOCK, dev)
        s["back"] = T + (BLOCK - 1) * B
    else:
        held = cap = _lengths(B, case["len"], case["ragged"])[mix]
        if op == "attend":
            lead = (B, case["Sq"]) if case["Sq"] > 1 else (B,)
            s["q"] = torch.randn(*lead, case["Hq"], D, generator=g, device=dev).to(dt)
        if op == "read" and case["ragged"]:
            s["cu"] = _cu(held, dev)
        s["total"] = int(held.sum())
    s["table"], pages = _pages(case, cap, g, dev)
    s["lens"] = held.to(dev, torch.int32)
    s["codes"] = torch.zeros(pages, 2, Hk, P, D, dtype=torch.int8, device=dev)
    s["scales"] = torch.zeros(pages, 2, Hk, P // BLOCK, device=dev)
    for b, n in enumerate(held.tolist()):
        ids = s["table"][b, : (n + P - 1) // P].long()
        for i in range(2):
            x = _tokens(len(ids) * P, Hk, D, g, dev, i == 0)
            x[n:] = 0
            x = x.view(-1, P // BLOCK, BLOCK, Hk, D).permute(0, 3, 1, 2, 4)  # (pages, Hk, blocks, 16, D)
            f = _scale(x.abs().amax((-1, -2)))
            s["codes"][ids, i] = _codes(x, f[..., None, None]).flatten(2, 3)
            s["scales"][ids, i] = f
    return s


def prepare(case, seed):
    s = _make(case, seed)
    if not own or case["op"] == "prompt":
        return s
    import flashcodec_b200 as fc

    cache = fc.PagedInt8Cache(s["codes"].shape[0], case["Hk"], case["D"], page_size=case["page"],
                              device=s["lens"].device)
    cache.codes.copy_(s.pop("codes"))
    cache.scales.copy_(s.pop("scales"))
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


def _places(s, cu, start, T):
    """Of T packed rows: whether they are of a sequence, their position, page and row in it."""
    i = torch.arange(T, device=cu.device)
    on = i < cu[-1]
    cu = cu.long()
    b = torch.searchsorted(cu[1:], i, right=True).clamp(max=s["B"] - 1)
    pos = torch.where(on, i - cu[b] + start.long()[b], torch.zeros_like(i))
    return on, pos, s["table"].long()[b, pos // s["page"]], pos % s["page"]


def _held(s, on, page, row, dtype):
    """The values of K and V at packed places, (T, Hk, D), zeros for rows of no sequence."""
    out = []
    for i in range(2):
        x = _values(s["codes"][page, i, :, row], s["scales"][page, i, :, row // BLOCK][..., None])
        out.append(torch.where(on[:, None, None], x, torch.zeros_like(x)).to(dtype))
    return out


def _plain_append(s):
    P, Hk = s["page"], s["Hk"]
    q, k, v = (s[n].float().flatten(0, -3) for n in ("q", "k", "v"))
    _, pos, page, row = _places(s, s["new_cu"], s["lens"], k.shape[0])
    if s["norm"]:
        q, k = _head_norm(q, s["qw"]), _head_norm(k, s["kw"])
    if s["rot"]:
        if s["axes"] > 1:
            p = s["positions"].flatten(1).long()[s["axis"].long()].t()  # (T, R / 2): the row of every pair
            pair = torch.arange(s["rot"] // 2, device=q.device)
            cs = torch.cat([s["rotary"][p, pair], s["rotary"][p, pair + s["rot"] // 2]], 1)
        else:
            cs = s["rotary"][pos]
        q, k = _rotate(q, cs, s["interleaved"]), _rotate(k, cs, s["interleaved"])
    blocks = page * (P // BLOCK) + row // BLOCK  # of the pool
    n = s["scales"].shape[0] * (P // BLOCK)
    touched = torch.zeros(n, dtype=torch.bool, device=q.device).index_fill(0, blocks, True)
    # blocks that held tokens before: those of the first new row of a sequence, where it is not a block's first
    first = torch.full((n,), P, device=q.device).scatter_reduce(0, blocks, row % BLOCK, "amin")
    for i, x in enumerate((k, v)):
        top = torch.zeros(n, Hk, device=q.device)
        top = top.scatter_reduce(0, blocks[:, None].expand(-1, Hk), x.abs().amax(-1), "amax")
        old = s["scales"][:, i].transpose(1, 2).reshape(n, Hk)
        old = torch.where((touched & (first > 0))[:, None], old, torch.zeros_like(old))
        new = torch.maximum(old, _scale(top))
        ids = touched.nonzero()[:, 0]
        at = (ids // (P // BLOCK), ids % (P // BLOCK))
        codes = s["codes"][:, i].unflatten(2, (-1, BLOCK))  # (pages, Hk, blocks, 16, D), a view
        ratio = torch.where(new > 0, old / torch.where(new > 0, new, torch.ones_like(new)), torch.zeros_like(new))
        codes[at[0], :, at[1]] = torch.floor(codes[at[0], :, at[1]].float() * ratio[ids][..., None, None]).to(torch.int8)
        s["scales"][:, i][at[0], :, at[1]] = new[ids]
        s["codes"][page, i, :, row] = _codes(x, new[blocks][..., None])
    on, _, page, row = _places(s, s["back_cu"], s["from"], s["back"])
    k, v = _held(s, on, page, row, s["q"].dtype)
    return {"q": q.to(s["q"].dtype).view(s["q"].shape), "k": k, "v": v}


def _plain_read(s):
    B, dt = s["B"], DTYPES[s["dtype"]]
    zero = torch.zeros_like(s["lens"])
    cu = s["cu"] if "cu" in s else torch.arange(B + 1, device=zero.device) * (s["total"] // B)
    on, _, page, row = _places(s, cu, zero, s["total"])
    shape = (s["total"],) if "cu" in s else (B, s["total"] // B)
    return dict(zip(("k", "v"), (x.view(*shape, s["Hk"], s["D"]) for x in _held(s, on, page, row, dt))))


def _softmax_product(q, k, v, visible):
    """q (S, Hk, G, D), k and v (L, Hk, D), visible (S, L) -> (S, Hk, G, D)."""
    a = torch.einsum("shgd,lhd->hsgl", q * q.shape[-1] ** -0.5, k)
    a = a.masked_fill(~visible[:, None], -math.inf)
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(top.isinf(), torch.zeros_like(top), top))
    n = e.sum(-1, keepdim=True)
    e = e / torch.where(n > 0, n, torch.ones_like(n))
    return torch.einsum("hsgl,lhd->shgd", e, v)


def _plain_attend(s):
    q = s["q"].float() if s["q"].dim() == 4 else s["q"].float()[:, None]
    B, S, Hq, D = q.shape
    out = torch.empty_like(q)
    for b in range(B):  # the table has no more columns than the longest sequence needs
        pages = s["table"][b].long().clamp(min=0)
        k, v = (_values(s["codes"][pages, i].unflatten(2, (-1, BLOCK)), s["scales"][pages, i][..., None, None])
                .flatten(2, 3).transpose(1, 2).flatten(0, 1) for i in range(2))
        seen = s["lens"][b].long() - torch.arange(S - 1, -1, -1, device=q.device)
        visible = torch.arange(k.shape[0], device=q.device) < seen[:, None]
        out[b] = _softmax_product(q[b].view(S, s["Hk"], -1, D), k, v, visible).reshape(S, Hq, D)
    return out.view(s["q"].shape).to(s["q"].dtype)


def _plain_prompt(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    Hq, Hk, D = s["Hq"], s["Hk"], s["D"]
    out = torch.empty_like(q)
    a = b = 0
    for n, m in zip(s["n_q"], s["n_k"]):
        step = max(1, 2 ** 30 // (Hq * m))  # rows of scores at once: 4 GB
        for i in range(0, n, step):
            j = min(n, i + step)
            seen = m - n + 1 + torch.arange(i, j, device=q.device)
            visible = torch.arange(m, device=q.device) < seen[:, None]
            out[a + i: a + j] = _softmax_product(q[a + i: a + j].view(j - i, Hk, -1, D), k[b: b + m], v[b: b + m],
                                                 visible).reshape(j - i, Hq, D)
        a, b = a + n, b + m
    return out.to(s["q"].dtype)


def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend,
                "prompt": _plain_prompt}[s["op"]](s)
    if s["op"] == "prompt":
        import flashcodec_b200 as fc

        return fc.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"] if s["ctx"] else None)
    cache = s["cache"]
    if s["op"] == "append":
        q = cache.append(s["q"], s["k"], s["v"], s["table"], s["lens"],
                         cu_seqlens=s["new_cu"] if s["ragged"] else None, q_weight=s.get("qw"),
                         k_weight=s.get("kw"), rotary=s.get("rotary"), interleaved=s["interleaved"],
                         positions=s.get("positions"), axes=s.get("axis"))
        k, v = cache.read(s["table"], s["from"], cu_seqlens=s["back_cu"], dtype=s["q"].dtype, count=s["back"])
        return {"q": q, "k": k, "v": v}
    if s["op"] == "read":
        k, v = cache.read(s["table"], None, cu_seqlens=s.get("cu"), dtype=DTYPES[s["dtype"]],
                          count=s["total"] if "cu" in s else s["total"] // s["B"])
        return {"k": k, "v": v}
    return cache.attend(s["q"], s["table"], s["lens"])


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = _make(case, seed)
    D, Hk, G = case["D"], case["Hk"], case.get("Hq", 0) // case["Hk"]

    def attention(q, k, v, first):
        """q (n, Hq, D) at positions first .. over k, v (m, Hk, D): query i sees first + i + 1 keys."""
        n, m = q.shape[0], k.shape[0]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        step = max(1, 2 ** 28 // (Hk * G * m))
        for i in range(0, n, step):
            j = min(n, i + step)
            x = q[i:j].double().view(j - i, Hk, G, D)
            w = torch.einsum("nhgd,mhd->nhgm", x, k.double()) / math.sqrt(D)
            at = torch.arange(first + i, first + j, device=q.device)
            w = w.masked_fill(torch.arange(m, device=q.device) > at[:, None, None, None], -math.inf)
            w = torch.softmax(w, -1).nan_to_num(0.0)
            out[i:j] = torch.einsum("nhgm,mhd->nhgd", w, v.double()).reshape(j - i, -1, D)
        return out

    if case["op"] == "prompt":
        parts, a, b = [], 0, 0
        for n, m in zip(s["n_q"], s["n_k"]):
            parts.append(attention(s["q"][a: a + n], s["k"][b: b + m], s["v"][b: b + m], m - n))
            a, b = a + n, b + m
        return torch.cat(parts)

    P = case["page"]
    lens = s["lens"].tolist()

    def held(i, b, lo, hi):  # (hi - lo, Hk, D) of sequence b, in 64 bits
        ids = s["table"][b, : (hi + P - 1) // P].long()
        c = s["codes"][ids, i].double() + 0.5  # (pages, Hk, P, D)
        f = s["scales"][ids, i].double().repeat_interleave(BLOCK, -1)
        return (c * f[..., None]).transpose(1, 2).reshape(-1, Hk, D)[lo:hi]

    if case["op"] == "read":
        x = {n: torch.cat([held(i, b, 0, m) for b, m in enumerate(lens)]) for i, n in enumerate("kv")}
        return x if "cu" in s else {n: y.view(case["B"], -1, Hk, D) for n, y in x.items()}

    if case["op"] == "attend":
        q = s["q"] if s["q"].dim() == 4 else s["q"][:, None]
        out = [attention(q[b], held(0, b, 0, n), held(1, b, 0, n), n - q.shape[1]) for b, n in enumerate(lens)]
        return torch.stack(out).view(s["q"].shape)

    cu = s["new_cu"].tolist()
    R = case["rot"]

    def turned(x, w, b):  # heads of one sequence's new tokens, normed and rotated
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
        if not R:
            return x
        n = x.shape[0]
        if case["axes"] > 1:
            p = s["positions"].flatten(1)[:, cu[b]: cu[b + 1]].long()
            t = torch.stack([s["rotary"][p[int(ax)]][:, [i, R // 2 + i]] for i, ax in enumerate(s["axis"].tolist())], 1)
        else:
            t = s["rotary"][lens[b]: lens[b] + n].view(n, 2, R // 2).transpose(1, 2)
        z = torch.view_as_complex(t.double().contiguous())[:, None]
        if case["interleaved"]:
            y = torch.view_as_real(torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * z).reshape(*x.shape[:-1], R)
        else:
            y = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * z
            y = torch.cat([y.real, y.imag], -1)
        return torch.cat([y, x[..., R:]], -1)

    q, kv = [], {"k": [], "v": []}
    for b, n in enumerate(lens):
        part = {name: s[name].flatten(0, -3)[cu[b]: cu[b + 1]] for name in ("q", "k", "v")}
        q.append(turned(part["q"], s.get("qw"), b))
        lo = n // BLOCK * BLOCK
        for i, name in enumerate("kv"):
            x = turned(part["k"], s.get("kw"), b) if name == "k" else part["v"].double()
            old = held(i, b, lo, n)
            x = torch.cat([old, x])
            for t in range(0, len(x), BLOCK):  # a block: its scale, and the middles of the steps that hold x
                y = x[t: t + BLOCK]
                top = y.abs().amax((0, 2))
                if t == 0 and n > lo:  # held tokens were at least this large before they were rounded
                    row = s["table"][b, lo // P].long()
                    unit = torch.maximum(s["scales"][row, i, :, lo % P // BLOCK].double(), _scale(top.float()).double())
                else:
                    unit = _scale(top.float()).double()
                f = torch.where(unit > 0, unit, torch.ones_like(unit))[None, :, None]
                x[t: t + BLOCK] = torch.where(unit[None, :, None] > 0, (torch.floor(y / f) + 0.5) * f, torch.zeros_like(y))
            kv[name].append(x)
    out = {"q": torch.cat(q).view(s["q"].shape)}
    for name, parts in kv.items():
        x = torch.cat(parts)
        out[name] = torch.cat([x, x.new_zeros(s["back"] - len(x), Hk, D)])
    return out
