"""Continuous batching on the paged KV caches.

Sequences of different lengths share one pool of pages per layer; they join with a
prompt, grow by a token a step and leave their pages to the next one.  The layers
are attention blocks with random weights (query and key norms, rotary positions,
grouped heads): enough to run the operations as a serving loop does.

    append            prompts packed into one call, then one token per sequence and step
    read              the held keys and values of a prompt, for the prompt's own attention
    prompt_attention  that attention, all prompts in one call
    attend            every step's attention, over the pages
    select            from `sparse_from` tokens on, the pages to attend to (4 bits)

    python examples/paged_decode.py [--bits 4] [--layers 4] [--steps 32] [--sparse-from 512]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from flashcodec_b200 import PagedInt4Cache, PagedInt8Cache, prompt_attention, rotary_table  # noqa: E402


class Pages:
    """Free pages of a pool and the table of the sequences that hold some."""

    def __init__(self, num_pages, rows, width, page_size, device):
        self.page_size, self.free = page_size, list(range(num_pages - 1, -1, -1))
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.held = [[] for _ in range(rows)]

    def hold(self, row, tokens):
        """Give a sequence the pages that `tokens` tokens need."""
        need = -(-tokens // self.page_size)
        while len(self.held[row]) < need:
            self.table[row, len(self.held[row])] = self.free[-1]
            self.held[row].append(self.free.pop())

    def leave(self, row):
        self.free += reversed(self.held[row])
        self.held[row] = []


class Layer:
    def __init__(self, hq, hk, d, pages, page_size, device, gen, bits):
        w = hq * d
        self.hq, self.hk, self.d = hq, hk, d
        self.qkv = torch.randn((hq + 2 * hk) * d, w, generator=gen, device=device).bfloat16() * w ** -0.5
        self.out = torch.randn(w, w, generator=gen, device=device).bfloat16() * w ** -0.5
        self.q_norm = torch.ones(d, device=device, dtype=torch.bfloat16)
        self.k_norm = torch.ones(d, device=device, dtype=torch.bfloat16)
        if bits == 4:
            self.cache = PagedInt4Cache(pages, hk, d, page_size=page_size, bounds=True, device=device)
        else:
            self.cache = PagedInt8Cache(pages, hk, d, page_size=page_size, device=device)

    def heads(self, x):
        y = (x @ self.qkv.t()).unflatten(-1, (-1, self.d))
        return y.split([self.hq, self.hk, self.hk], -2)

    def put(self, x, table, lengths, rotary, cu=None):
        q, k, v = self.heads(x)
        return self.cache.append(q, k, v, table, lengths, cu_seqlens=cu, q_weight=self.q_norm,
                                 k_weight=self.k_norm, rotary=rotary)

    def prompt(self, q, table, cu, starts):
        """Causal attention of packed prompts over what the cache holds of them."""
        k, v = self.cache.read(table, starts, count=q.shape[0], cu_seqlens=cu, dtype=q.dtype)
        return prompt_attention(q, k, v, cu)


@torch.no_grad()
def run(layers=4, steps=32, prompts=(37, 5, 700, 129), hq=16, hk=8, d=128, page_size=64,
        sparse_from=512, count=6, seed=0, bits=4):
    """Returns the largest relative difference between a step's attention and the same
    attention computed from the values that the cache holds (dense steps)."""
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, most = len(prompts), max(prompts) + steps + 1
    width = -(-most // page_size)
    num_pages = rows * width
    stack = [Layer(hq, hk, d, num_pages, page_size, dev, gen, bits) for _ in range(layers)]
    pages = Pages(num_pages, rows, width, page_size, dev)
    rotary = rotary_table(most, d, base=1e6, device=dev)

    # the prompts, packed
    new = torch.tensor(prompts)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(dev, torch.int32)
    lengths = torch.zeros(rows, dtype=torch.int32, device=dev)
    for r, n in enumerate(prompts):
        pages.hold(r, n)
    x = torch.randn(int(new.sum()), hq * d, generator=gen, device=dev).bfloat16()
    for layer in stack:
        q = layer.put(x, pages.table, lengths, rotary, cu)
        x = x + layer.prompt(q, pages.table, cu, lengths).flatten(1) @ layer.out.t()
    lengths += new.to(dev, torch.int32)

    x = x[cu[1:].long() - 1]  # the last token of every prompt starts its answer
    worst = 0.0
    for step in range(steps):
        lens = [n + step + 1 for n in prompts]
        for r, n in enumerate(lens):
            pages.hold(r, n)
        sparse = bits == 4 and max(lens) >= sparse_from and step % 2  # every other step, to show both
        after = lengths + 1
        x = torch.nn.functional.normalize(x.float(), dim=-1).mul(x.shape[-1] ** 0.5).bfloat16()
        for i, layer in enumerate(stack):
            q = layer.put(x, pages.table, lengths, rotary)
            chosen = layer.cache.select(q, pages.table, after, count) if sparse else None
            o = layer.cache.attend(q, pages.table, after, **({"selected": chosen} if sparse else {}))
            if step == (steps - 1) // 2 * 2 and i == layers - 1:  # the last dense step
                worst = max(worst, check(layer, q, o, pages.table, lens))
            x = x + o.flatten(1) @ layer.out.t()
        lengths = after
    for layer in stack:
        layer.cache.check()
    for r in range(rows):
        pages.leave(r)
    assert sorted(pages.free) == list(range(num_pages))
    return worst


def check(layer, q, o, table, lens):
    worst = 0.0
    for r, n in enumerate(lens):
        k, v = layer.cache.read(table[r:r + 1], count=n, dtype=torch.float32)
        g = layer.hq // layer.hk
        a = torch.einsum("hgd,nhd->hgn", q[r].float().view(layer.hk, g, -1), k[0]) * layer.d ** -0.5
        want = torch.einsum("hgn,nhd->hgd", a.softmax(-1), v[0]).reshape_as(o[r])
        worst = max(worst, float((o[r].float() - want).norm() / want.norm()))
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--sparse-from", type=int, default=512)
    ap.add_argument("--bits", type=int, choices=(4, 8), default=4)
    args = ap.parse_args()
    err = run(layers=args.layers, steps=args.steps, sparse_from=args.sparse_from, bits=args.bits)
    print(f"{args.layers} layers, {args.steps} steps: attention over the pages differs from the held values' "
          f"by {err:.2e} (relative)")
