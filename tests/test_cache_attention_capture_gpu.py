"""Attention over the paged MX cache captured into graphs, in processes that have not
called it before, and of several kernels."""
import os
import subprocess
import sys

import numpy as np
import pytest
from test_cache_attention_gpu import attend, build, check

pytestmark = pytest.mark.gpu

FRESH = """
import sys
import numpy as np
import torch
sys.path[:0] = sys.argv[1:3]
import mxk
from test_cache_attention_gpu import attend, build, check

g = np.random.default_rng(51)
if sys.argv[3] == "decode":  # a call that needs the kernel for few rows only
    b = build(torch, mxk, g, [1], [50], 4, 2, 64, 16, 8, "bfloat16")
    attend(torch, mxk, b)
b = build(torch, mxk, g, [int(sys.argv[4]), 1], [1300, 40], 4, 2, 64, 16, 8, "bfloat16")
out = torch.zeros_like(b["q"])
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=int(sys.argv[4]), max_kv=1300)
graph.replay()
torch.cuda.synchronize()
check(torch, b, out, None)
print("captured and right")
"""


@pytest.mark.parametrize("first", ["decode", "nothing"])
@pytest.mark.parametrize("n", [90, 700])
def test_first_call_with_many_rows_is_captured(torch_cuda, mxk, first, n):
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FRESH, os.path.dirname(mxk.__file__), here, first, str(n)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured and right" in r.stdout, r.stderr[-2000:]


def test_several_kernels_in_a_graph(torch_cuda, mxk):
    """Sequences for every kernel, replayed as lengths and row ranges move within the
    bounds: allocations lie between launches that overlap."""
    torch, g = torch_cuda, np.random.default_rng(52)
    q_lens, kv_lens = [1, 300, 60, 5, 400], [500, 700, 300, 90, 1000]
    b = build(torch, mxk, g, q_lens, kv_lens, 4, 2, 128, 32, 8, "bfloat16")
    out = torch.empty_like(b["q"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=400, max_kv=1000)
    every = b["slots"]
    for q, kv in ((q_lens, kv_lens), (q_lens, [400, 650, 61, 5, 999]), ([3, 1, 360, 400, 2], [500, 700, 300, 90, 80]),
                  ([0, 0, 0, 0, 1], [1, 1, 1, 1, 1])):
        b.update(q_lens=q, kv_lens=kv, slots=[s[:l] for s, l in zip(every, kv)])
        b["cu"].copy_(torch.tensor([0] + list(np.cumsum(q)), dtype=torch.int32))
        b["kv"].copy_(torch.tensor(kv, dtype=torch.int32))
        out.fill_(3.0)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        check(torch, b, out, None)
        assert (out[sum(q):] == 3.0).all()


@pytest.mark.parametrize("threads", [False, True])
def test_calls_on_two_streams(torch_cuda, mxk, threads):
    """Calls that overlap on the GPU, from one thread or two, have workspaces of their own."""
    import threading
    torch = torch_cuda
    batches = [build(torch, mxk, np.random.default_rng(s), q, kv, 8, 2, 128, 32, 8, "bfloat16")
               for s, q, kv in ((53, [1, 40, 300], [3000, 900, 800]), (54, [700, 2, 20], [1500, 5000, 700]))]
    want = [attend(torch, mxk, b)[0] for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [[torch.zeros_like(w) for _ in range(20)] for w in want]
    torch.cuda.synchronize()

    def work(i):
        b = batches[i]
        for out in outs[i]:
            mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=max(b["q_lens"]),
                                max_kv=max(b["kv_lens"]), stream=streams[i])
    if threads:
        ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        [t.start() for t in ts]
        [t.join() for t in ts]
    else:
        for j in range(20):
            for i in range(2):
                b = batches[i]
                mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], outs[i][j],
                                    max_q=max(b["q_lens"]), max_kv=max(b["kv_lens"]), stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        for out in outs[i]:
            assert torch.equal(out, want[i])


def test_a_failure_is_reported_once(torch_cuda, mxk):
    """A call that the CUDA runtime refuses (here: waiting for the device while another
    thread captures) fails itself, and not the calls that its thread makes afterwards."""
    import threading
    torch = torch_cuda
    b = build(torch, mxk, np.random.default_rng(55), [3], [50], 4, 2, 64, 16, 8, "bfloat16")
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.full((3,), -1, device="cuda")
    capturing, refused, ended = (threading.Event() for _ in range(3))
    seen = []

    def other():
        capturing.wait(60)
        try:
            mxk.release_workspace()
        except mxk.MxkError:
            seen.append("refused")
        refused.set()
        ended.wait(60)
        mxk.cache_write(b["cache"], k, k, slots)
        seen.append("written")
    thread = threading.Thread(target=other)
    thread.start()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            capturing.set()
            refused.wait(60)
    except RuntimeError:
        pass  # the other thread's call has invalidated the capture
    ended.set()
    thread.join()
    torch.cuda.synchronize()
    assert seen == ["refused", "written"]
