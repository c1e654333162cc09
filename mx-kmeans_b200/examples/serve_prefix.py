"""The attention of one layer for a batch of conversations behind a common instruction.

    python mx-kmeans_b200/examples/serve_prefix.py [--bits 8] [--steps 16] [--batch 48]

The layer's weights are E4M3 with a scale per 128 x 128 block (mxk.quantize_fp8, once).  Every
step takes the new tokens through the projection (mxk.linear_fp8), rotates and stores them
(mxk.cache_append), attends with the instruction read once for the whole batch
(mxk.cache_attention_shared) and through the output projection.  Decoding steps replay one
captured graph.  At the end the last step's attention is recomputed in float64 from what the
cache holds (mxk.cache_read).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mxk  # noqa: E402


def quantised(n, k, gen):
    """Random weights [n, k] as E4M3 values and scales."""
    w = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.bfloat16) * k ** -0.5
    values = torch.empty(n, k, dtype=torch.uint8, device="cuda")
    scales = torch.empty(-(-n // 128), -(-k // 128), device="cuda")
    mxk.quantize_fp8(w, values, scales, block_rows=128)
    return values, scales


def main(bits=8, steps=16, batch=48, prompt=4000, heads=16, kv_heads=4, dim=128, hidden=2048, page=32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, longest = torch.bfloat16, prompt + steps
    w_in, w_out = quantised((heads + 2 * kv_heads) * dim, hidden, gen), quantised(hidden, heads * dim, gen)
    turns = torch.arange(longest, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
    cos_sin = torch.cat([turns.cos(), turns.sin()], 1).float()

    # whole pages of the instruction are common, what follows is each conversation's own
    common, width = prompt // page, -(-longest // page)
    own = width - common
    cache = mxk.PagedCache.empty(common + batch * own, page, kv_heads, dim, bits)
    table = torch.empty(batch, width, dtype=torch.int32, device="cuda")
    table[:, :common] = torch.arange(common)
    table[:, common:] = common + torch.arange(batch * own).view(batch, own)

    def project(x):
        qkv = torch.empty(x.shape[0], heads + 2 * kv_heads, dim, dtype=dtype, device="cuda")
        mxk.linear_fp8(x, *w_in, qkv.view(x.shape[0], -1))
        return qkv.split([heads, kv_heads, kv_heads], 1)

    # the instruction, once; its last tokens, which share no page, into every conversation's
    q, k, v = project(torch.randn(prompt, hidden, generator=gen, device="cuda", dtype=dtype))
    at = torch.arange(prompt, device="cuda")
    rest = at[common * page:]
    mxk.cache_append(cache, None, k[:common * page], v[:common * page], at[:common * page], cos_sin, at[:common * page])
    if len(rest):
        slots = (table[:, common, None].long() * page + rest % page).view(-1)
        k, v = (t[common * page:].repeat(batch, 1, 1) for t in (k, v))
        mxk.cache_append(cache, None, k, v, rest.repeat(batch), cos_sin, slots)

    cu_q = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    cu_groups = torch.tensor([0, batch], dtype=torch.int32, device="cuda")
    shared = torch.tensor([common * page], dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
    positions, slots = (torch.empty(batch, dtype=torch.int64, device="cuda") for _ in range(2))
    x = torch.empty(batch, hidden, dtype=dtype, device="cuda")
    y, out = torch.empty_like(x), torch.empty(batch, heads, dim, dtype=dtype, device="cuda")
    last = {}

    def step():
        q, k, v = project(x)
        mxk.cache_append(cache, q, k, v, positions, cos_sin, slots)  # queries in place
        mxk.cache_attention_shared(cache, q, cu_q, table, lens, cu_groups, shared, out, max_q=1, max_kv=longest,
                                   max_prefix=common * page)
        mxk.linear_fp8(out.view(batch, -1), *w_out, y)
        last["q"] = q

    graph = torch.cuda.CUDAGraph()
    for t in range(prompt, longest):
        x.copy_(torch.randn(batch, hidden, generator=gen, device="cuda", dtype=dtype))
        lens.fill_(t + 1), positions.fill_(t)
        slots.copy_(table[:, t // page].long() * page + t % page)
        if t == prompt:
            step()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step()
        else:
            graph.replay()
    torch.cuda.synchronize()

    worst = 0.0
    for i in range(batch):
        where = table[i].long().repeat_interleave(page) * page + torch.arange(page, device="cuda").repeat(width)
        k, v = (torch.empty(longest, kv_heads, dim, device="cuda") for _ in range(2))
        mxk.cache_read(cache, where[:longest].contiguous(), k, v)
        k, v = (t.double().repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        s = torch.einsum("hd,thd->ht", last["q"][i].double(), k) * dim ** -0.5
        want = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v)
        worst = max(worst, float((out[i].double() - want).norm() / want.norm()))
    print(f"{steps} steps of {batch} conversations behind {prompt} tokens, {bits}-bit cache: attention differs from "
          f"float64 on the cached values by {worst:.1e} (relative, 2-norm)")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--bits", type=int, default=8, choices=(4, 6, 8))
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--batch", type=int, default=48)
    main(**vars(ap.parse_args()))
