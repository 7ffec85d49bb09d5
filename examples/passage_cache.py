"""Answering from retrieved passages whose keys and values are cached.

    python -m examples.passage_cache [--passages 20000] [--requests 32]

Every passage is one page of a paged key-value cache (its keys and values were
computed once, here: drawn at random) and one row of a graph index over
passage embeddings, under the same number.  A request

1. searches the graph with its question's embedding (int32 ids, -1 where
   unfilled),
2. adopts the pages of those ids as the beginning of its own row -- nothing is
   copied, and passages shorter than a page are masked,
3. extends its row and generates tokens: each layer rotates and appends the new
   token's key and value and attends to passages and own tokens together,
4. forks into two continuations half way, and gives its pages back at the end;
   then the cache is compacted.

The model is a toy (attention layers with random weights): what runs here is
the search, the cache and its operators, as a serving program would call them.
"""
from __future__ import annotations

import argparse
import time

import torch

import jasper_b200 as jasper
from jasper_b200 import paged


def arange(n: int, start: int = 0) -> torch.Tensor:
    return torch.arange(start, start + n, dtype=torch.int32, device="cuda")


class Toy:
    """Attention layers with random weights over a paged cache."""

    def __init__(self, cache: paged.PagedCache, heads: int, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cache, self.heads = cache, heads
        self.rotary = paged.Rotary(cache.head_dim, scaling="yarn", factor=4.0, trained_length=8192)
        self.dim = heads * cache.head_dim
        wide = (heads + 2 * cache.n_kv_heads) * cache.head_dim

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * rows ** -0.5).to(cache.dtype)
        self.qkv = [weight(self.dim, wide) for _ in range(cache.n_layers)]
        self.out = [weight(self.dim, self.dim) for _ in range(cache.n_layers)]

    def step(self, x: torch.Tensor, rows: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        """One new token of each row: hidden states in, hidden states out."""
        c, hkv = self.cache, self.cache.n_kv_heads
        c.extend(rows, torch.ones_like(rows))
        for layer in range(c.n_layers):
            q, k, v = (x @ self.qkv[layer]).view(len(rows), -1, c.head_dim).split([self.heads, hkv, hkv], dim=1)
            q = c.append(layer, k, v, rows, q=q, rotary=self.rotary)
            a = c.attend(layer, q, rows, mask=mask)
            x = torch.nn.functional.rms_norm(x + a.reshape(len(rows), -1) @ self.out[layer], (self.dim,))
        return x


def run(n_passages: int = 20_000, n_requests: int = 32, tokens: int = 24, k: int = 10, layers: int = 4, heads: int = 16,
        kv_heads: int = 4, head_dim: int = 64, page_size: int = 32, seed: int = 0, verbose: bool = True) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    embeddings = torch.randn(n_passages, 128, generator=g, device="cuda").half()
    graph = jasper.Graph.build(embeddings, n_neighbors=32)

    # row 0 holds the passages, page i passage i; rows behind it are requests
    spare = 2 * n_requests * (2 + tokens // page_size)
    cache = paged.PagedCache.allocate(layers, n_passages + spare, page_size, kv_heads, head_dim, 1 + 2 * n_requests,
                                      max(n_passages, k + 2 + tokens // page_size))
    cache.extend(arange(1), torch.tensor([n_passages * page_size], dtype=torch.int32, device="cuda"))
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    fill = torch.randint(page_size // 2, page_size + 1, (n_passages,), generator=g, device="cuda")  # tokens of a passage

    model = Toy(cache, heads, seed + 1)
    pick = torch.randint(0, n_passages, (n_requests,), generator=g, device="cuda")
    questions = embeddings[pick] + 0.1 * torch.randn(n_requests, 128, generator=g, device="cuda").half()
    x = torch.randn(n_requests, model.dim, generator=g, device="cuda").to(cache.dtype)

    torch.cuda.synchronize()
    began = time.perf_counter()
    ids, _ = graph.search(questions, k=k, beam_width=64)
    requests = arange(n_requests, 1)
    cache.adopt(requests, ids)
    inside = torch.where(ids >= 0, fill[ids.clamp_min(0).long()], 0)
    mask = (torch.arange(page_size, device="cuda") < inside[..., None]).view(n_requests, k * page_size)
    for _ in range(tokens // 2):
        x = model.step(x, requests, mask)
    # two continuations of every request: the second begins as a copy
    others = arange(n_requests, 1 + n_requests)
    cache.fork(requests, others)
    rows, masks = torch.cat([requests, others]), torch.cat([mask, mask])
    states = torch.cat([x, x])
    same = model.step(states, rows, masks)
    states = same + torch.randn(same.shape, generator=g, device="cuda").to(same.dtype)  # they part here
    for _ in range(tokens // 2 - 1):
        states = model.step(states, rows, masks)
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    cache.check()

    # the first request's continuations go on after all others have left
    keep = torch.stack([requests[0], others[0]])
    q = torch.randn(2, heads, head_dim, generator=g, device="cuda").to(cache.dtype)
    before = cache.attend(0, q, keep, mask=masks[[0, n_requests]])
    cache.free(torch.cat([requests[1:], others[1:]]))
    remap = cache.compact()
    after = cache.attend(0, q, keep, mask=masks[[0, n_requests]])
    cache.check()
    free = int((cache.refs == 0).sum())
    if verbose:
        print(f"{n_requests} requests x {k} passages of {n_passages}, {tokens} tokens each, two continuations: "
              f"{took * 1e3:.1f} ms; {free} of {cache.n_pages} pages free at the end")
    return {"ids": ids, "same": same, "states": states, "before": before, "after": after, "remap": remap, "free": free,
            "cache": cache}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--passages", type=int, default=20_000)
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args()
    run(a.passages, a.requests, a.tokens, verbose=False)  # the first run loads kernels
    run(a.passages, a.requests, a.tokens)
