"""A layer's calls as the first ones of a process, captured; and from two threads at once."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
from test_cache_append_gpu import make
from test_cache_attention_gpu import check
from test_cache_attention_shared_gpu import build, wide_bounds

pytestmark = pytest.mark.gpu

FIRST = """
import sys
sys.path[:0] = ["mx-kmeans_b200"]
import torch, mxk
seqs, prefix, new = {sizes}
cache = mxk.PagedCache.empty(prefix // 64 + seqs, 64, 8, 128, 8)
for t in (cache.k_values, cache.v_values, cache.k_scales, cache.v_scales):
    t.fill_(0x38)
i32 = dict(dtype=torch.int32, device="cuda")
table = torch.cat([torch.arange(prefix // 64).expand(seqs, -1), prefix // 64 + torch.arange(seqs)[:, None]], 1).to(**i32).contiguous()
q, k, v = (torch.ones(seqs * new, h, 128, device="cuda", dtype=torch.bfloat16) for h in (32, 8, 8))
cos_sin = torch.cat([torch.ones(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda")], 1)
at = torch.zeros(seqs * new, dtype=torch.int64, device="cuda")
slots = (prefix + 64 * torch.arange(seqs, device="cuda")[:, None] + torch.arange(new, device="cuda")).view(-1)
cu, kv = torch.arange(seqs + 1, **i32) * new, torch.full((seqs,), prefix + new, **i32)
groups, lens = torch.tensor([0, seqs], **i32), torch.tensor([prefix], **i32)
out = torch.zeros_like(q)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    mxk.cache_append(cache, q, k, v, at, cos_sin, slots)
    mxk.cache_attention_shared(cache, q, cu, table, kv, groups, lens, out, max_q=new, max_kv=prefix + new, max_prefix=prefix)
graph.replay()
torch.cuda.synchronize()
# every cached value is 2^(56 - 127), or 1 in the new tokens, with the same scores, or larger ones there
first = out.view(seqs, new, 32, 128)[:, 0].float()
assert torch.isfinite(out).all() and (first == first[0, 0, 0]).all() and first[0, 0, 0] > 0.9
"""


@pytest.mark.parametrize("sizes", [(64, 8192, 1), (4, 256, 1), (32, 4096, 30)])
def test_first_calls_of_a_process_may_be_captured(torch_cuda, sizes):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.format(sizes=sizes)], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_threads(torch_cuda, mxk):
    """Each with its own stream, cache and outputs."""
    torch = torch_cuda
    made, errors = [], []
    for seed, n, bits in ((1, 60, 8), (2, 40, 4)):
        b = build(torch, mxk, np.random.default_rng(seed), [(256, 256, [(1, 1 + 11 * i % 300) for i in range(n)])], 16, 4, 128, 32, bits,
                  "bfloat16")
        made.append((b, *wide_bounds(torch, b), make(torch, mxk, 300, 8, 2, 64, 16, bits, "float16", 64, seed)))
    torch.cuda.synchronize()
    outs = [[], []]

    def work(i):
        try:
            stream = torch.cuda.Stream()
            b, table, tokens, most, (cache, q, k, v, slots, positions, cos_sin) = made[i]
            with torch.cuda.stream(stream):
                for _ in range(30):
                    out, turned = torch.empty_like(b["q"]), torch.empty_like(q)
                    mxk.cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=turned)
                    mxk.cache_attention_shared(b["cache"], b["q"], b["cu"], table, b["kv"], b["groups"], b["prefixes"], out, max_q=1,
                                               max_kv=tokens, max_prefix=most)
                    outs[i].append((out, turned))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for (b, *_), got in zip(made, outs):
        check(torch, b, got[0][0], None)
        assert all(torch.equal(out, got[0][0]) and torch.equal(turned, got[0][1]) for out, turned in got)
