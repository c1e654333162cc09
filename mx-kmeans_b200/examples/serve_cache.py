"""A serving loop over the paged MX cache: prompts in chunks beside decoding
sequences, all of a step in one call.

    python mx-kmeans_b200/examples/serve_cache.py [--bits 8] [--steps 24]

Random keys, values and queries stand in for a model's projections.  Every step
stores the new tokens' rows (mxk.cache_write) and attends over what is cached
(mxk.cache_attention); pages are handed out as sequences grow.  At the end the
cache is read back (mxk.cache_read) and the last step's attention is recomputed from
it in float64.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mxk  # noqa: E402


class Sequence:
    def __init__(self, prompt):
        self.prompt, self.cached, self.pages = prompt, 0, []

    def take(self, chunk):
        """New tokens of the next step: a piece of the prompt, then one at a time."""
        return min(chunk, self.prompt - self.cached) if self.cached < self.prompt else 1


def main(bits=8, steps=24, prompts=(5, 130, 700, 64, 333), chunk=128, heads=16, kv_heads=4, dim=128, page=32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype = "cuda", torch.bfloat16
    pages = sum(-(-(p + steps) // page) for p in prompts)
    cache = mxk.PagedCache.empty(pages, page, kv_heads, dim, bits)
    free = list(range(pages))[::-1]
    seqs = [Sequence(p) for p in prompts]
    width = max(-(-(p + steps) // page) for p in prompts)
    table = torch.zeros(len(seqs), width, dtype=torch.int32)
    for _ in range(steps):
        new = [s.take(chunk) for s in seqs]
        slots = []
        for i, (s, n) in enumerate(zip(seqs, new)):
            while len(s.pages) * page < s.cached + n:
                table[i, len(s.pages)] = free[-1]
                s.pages.append(free.pop())
            slots += [s.pages[t // page] * page + t % page for t in range(s.cached, s.cached + n)]
            s.cached += n
        total = sum(new)
        q, k, v = (torch.randn(total, h, dim, generator=gen, device=dev, dtype=dtype) for h in (heads, kv_heads, kv_heads))
        cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=dev)
        lens = torch.tensor([s.cached for s in seqs], dtype=torch.int32, device=dev)
        out = torch.empty_like(q)
        mxk.cache_write(cache, k, v, torch.tensor(slots, device=dev))
        mxk.cache_attention(cache, q, cu, table.to(dev), lens, out, max_q=max(new), max_kv=max(s.cached for s in seqs))

    # the last step once more, from the values that the cache stands for
    worst, row = 0.0, 0
    for s, n in zip(seqs, new):
        slots = torch.tensor([s.pages[t // page] * page + t % page for t in range(s.cached)], device=dev)
        k, v = (torch.empty(s.cached, kv_heads, dim, device=dev) for _ in range(2))
        mxk.cache_read(cache, slots, k, v)
        k, v = (x.double().repeat_interleave(heads // kv_heads, 1) for x in (k, v))
        scores = torch.einsum("nhd,thd->hnt", q[row:row + n].double(), k) * dim ** -0.5
        seen = torch.arange(s.cached, device=dev) <= torch.arange(s.cached - n, s.cached, device=dev)[:, None]
        want = torch.einsum("hnt,thd->nhd", torch.softmax(scores.masked_fill(~seen, -torch.inf), -1), v)
        worst = max(worst, float((out[row:row + n].double() - want).norm() / want.norm()))
        row += n
    print(f"{steps} steps, {bits}-bit cache, {sum(s.cached for s in seqs)} tokens in {len(seqs)} sequences: "
          f"attention differs from float64 on the cached values by {worst:.1e} (relative, 2-norm)")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--bits", type=int, default=8, choices=(4, 6, 8))
    ap.add_argument("--steps", type=int, default=24)
    main(**vars(ap.parse_args()))
