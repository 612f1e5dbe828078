"""Retrieval, prompts and decoding over one paged key-value cache (needs a B200).

The passages of a small corpus that answer each request best are found by exact
k-NN search; their tokens are the request's prompt.  The prompts enter a paged
cache, every prompt token attends to the pages that it selects, and then the
requests decode one token each per step.  The "model" is one attention layer of
random projections: the point is the order of the calls and their shapes.

    python examples/paged_decode.py [--requests 16] [--steps 8] [--cache e4m3]
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mlxvs_b200 as mv  # noqa: E402


class Layer:
    """Queries, keys and values of tokens, by random projections."""

    def __init__(self, width, heads, group, dim, gen):
        def matrix(out):
            m = torch.randn(width, out, generator=gen, device="cuda")
            return (m / math.sqrt(width)).bfloat16()

        self.heads, self.group, self.dim = heads, group, dim
        self.wq, self.wk, self.wv = (matrix(h * dim) for h in (heads * group, heads, heads))
        self.wo = matrix(width) if width == heads * group * dim else (
            torch.randn(heads * group * dim, width, generator=gen, device="cuda")
            / math.sqrt(heads * group * dim)).bfloat16()

    def project(self, x):
        n = len(x)
        return ((4 * (x @ self.wq)).view(n, self.heads * self.group, self.dim),
                (x @ self.wk).view(n, self.heads, self.dim),
                (x @ self.wv).view(n, self.heads, self.dim))


def run(requests=16, steps=8, passages=4, passage_tokens=300, page=64, pages_seen=8,
        cache="bf16", heads=4, group=8, dim=128, width=1024, seed=0):
    """Runs the loop; returns the share of the full attention's weight that lay
    in the selected pages, per step (the prompt step first)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    corpus = 2000
    embeddings = torch.randn(corpus, 128, generator=gen, device="cuda")
    words = torch.randn(corpus, passage_tokens, width, generator=gen, device="cuda").bfloat16()
    wanted = torch.randint(corpus, (requests,), generator=gen, device="cuda")
    questions = embeddings[wanted] + 0.3 * torch.randn(requests, 128, generator=gen, device="cuda")

    # the passages that answer each request best, exactly
    found, _ = mv.brute_force_knn(embeddings, questions, passages)
    prompts = words[found.long()].view(requests, -1, width)
    length = prompts.shape[1]

    # the cache: pages for every prompt and the tokens to come, and their bounds
    total = requests * (-(-(length + steps) // page)) + 8
    kind = torch.float8_e4m3fn if cache == "e4m3" else torch.bfloat16
    keys = torch.zeros(total, page, heads, dim, dtype=kind, device="cuda")
    values = torch.zeros_like(keys)
    codes = torch.zeros(total, heads, 2, dim, dtype=torch.int8, device="cuda")
    scales = torch.zeros(total, heads, device="cuda")
    table = torch.full((requests, -(-(length + steps) // page)), -1, dtype=torch.int32,
                       device="cuda")
    free = torch.randperm(total, generator=gen, device="cuda").int()
    layer = Layer(width, heads, group, dim, gen)

    def step(x, past, fresh, free):
        """One step of the layer for x [tokens, width], `fresh` of them per request."""
        t = mv.paged_tables(past, fresh, table, free, page, len(x))
        q, k, v = layer.project(x)
        mv.paged_store(k, v, t.slots, keys, values, codes, scales)
        chosen = mv.paged_select(q, codes, scales, table, t.lengths, page, pages_seen,
                                 requests=t.requests)
        out, lse = mv.paged_attention(q, keys, values, table, t.lengths, requests=t.requests,
                                      pages=chosen, return_lse=True)
        return out.reshape(len(x), -1) @ layer.wo, q, lse, t

    def share(q, lse, t):
        _, full = mv.paged_attention(q, keys, values, table, t.lengths, requests=t.requests,
                                     return_lse=True)
        return torch.exp(lse - full).mean().item()

    past = torch.zeros(requests, dtype=torch.int32, device="cuda")
    fresh = torch.full_like(past, length)
    out, q, lse, t = step(prompts.reshape(-1, width), past, fresh, free)
    shares = [share(q, lse, t)]
    past += fresh
    free = free[int(t.used[0]):]
    x = out.view(requests, length, width)[:, -1]
    one = torch.ones_like(past)
    for _ in range(steps):
        out, q, lse, t = step(x, past, one, free)
        shares.append(share(q, lse, t))
        past += one
        free = free[int(t.used[0]):]
        x = torch.nn.functional.normalize(x + out, dim=-1) * math.sqrt(width)
    mv.synchronize()
    return shares


if __name__ == "__main__":
    a = argparse.ArgumentParser()
    a.add_argument("--requests", type=int, default=16)
    a.add_argument("--steps", type=int, default=8)
    a.add_argument("--pages", type=int, default=8, help="pages that a token attends to")
    a.add_argument("--cache", choices=["bf16", "e4m3"], default="bf16")
    args = a.parse_args()
    got = run(requests=args.requests, steps=args.steps, pages_seen=args.pages, cache=args.cache)
    print("share of the attention's weight in the selected pages:")
    print("  prompts  %.3f" % got[0])
    for i, s in enumerate(got[1:]):
        print("  token %2d %.3f" % (i + 1, s))
