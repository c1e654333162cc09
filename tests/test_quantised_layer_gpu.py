"""The attention of a layer as a server runs it, step by step: projections of quantised
weights (linear_fp8), rotation and storing (cache_append), attention with a shared prefix
(cache_attention_shared), output projection (linear_fp8); against the formulas in 64 bits on the
quantised weights."""
import numpy as np
import pytest

from test_cache_append_gpu import mx_values, rotated, table
from test_gemm_fp8_gpu import expected, scaled

pytestmark = pytest.mark.gpu


def relative(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("heads,kv_heads,dim,hidden", [(8, 2, 64, 512), (4, 4, 128, 640)])
def test_steps_of_a_batch_with_a_common_prompt(torch_cuda, mxk, heads, kv_heads, dim, hidden):
    torch = torch_cuda
    dtype, page, bits, seqs, prompt, steps = torch.bfloat16, 32, 8, 40, 320, 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    width = (heads + 2 * kv_heads) * dim

    def weights(n, k):
        codes, scales = expected(torch, torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5, 128)
        return codes.to(torch.uint8), scales
    w_in, w_out = weights(width, hidden), weights(hidden, heads * dim)
    cos_sin = table(torch, 1024, dim)
    own = -(-(prompt % page + steps) // page) + 1
    pages = prompt // page + seqs * own
    cache = mxk.PagedCache.empty(pages, page, kv_heads, dim, bits)
    rows = torch.full((seqs, prompt // page + own), 0, dtype=torch.int32)
    for i in range(seqs):
        rows[i, :prompt // page] = torch.arange(prompt // page)
        rows[i, prompt // page:] = prompt // page + i * own + torch.arange(own)
    longest = 16384  # (with bounds like these the prompt is worth sharing; the pages behind are not looked at)
    rows = torch.nn.functional.pad(rows, (0, longest // page - rows.shape[1])).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")

    def project(x, w):
        """x [n, k] through w: a new tensor, and the formula in 64 bits."""
        out = torch.empty(x.shape[0], w[0].shape[0], dtype=dtype, device="cuda")
        mxk.linear_fp8(x, *w, out)
        a, s = expected(torch, x, 1)
        return out, scaled(torch, a.to(torch.uint8), s, 1) @ scaled(torch, *w, 128).T

    def append(x, positions, slots):
        q, k, v = x.view(-1, heads + 2 * kv_heads, dim).split([heads, kv_heads, kv_heads], 1)
        before = [t.double().cpu().numpy() for t in (q, k, v)]
        angles = cos_sin[positions].double().cpu().numpy()
        mxk.cache_append(cache, q, k, v, positions, cos_sin, slots)  # queries in place
        return (q, rotated(before[0], angles, False), mx_values(rotated(before[1], angles, False), bits)[0],
                mx_values(before[2], bits)[0])

    # the prompt, once for all
    x = torch.randn(prompt, hidden, generator=gen, device="cuda").to(dtype)
    qkv, want = project(x, w_in)
    assert relative(qkv, want) < 2.0 ** -8
    at = torch.arange(prompt, device="cuda")
    _, _, keys, values = append(qkv, at, at)
    keys, values = [[torch.from_numpy(keys).cuda()] for _ in range(seqs)], [[torch.from_numpy(values).cuda()] for _ in range(seqs)]
    cu_q = torch.arange(seqs + 1, **i32)
    groups, prefixes = torch.tensor([0, seqs], **i32), torch.tensor([prompt], **i32)
    for step in range(steps):
        length = prompt + step + 1
        x = torch.randn(seqs, hidden, generator=gen, device="cuda").to(dtype)
        qkv, want = project(x, w_in)
        assert relative(qkv, want) < 2.0 ** -8
        positions = torch.full((seqs,), length - 1, device="cuda")
        slots = rows[:, (length - 1) // page].long() * page + (length - 1) % page
        q, want_q, k, v = append(qkv, positions, slots)
        assert relative(q, torch.from_numpy(want_q).cuda()) < 2.0 ** -8
        out = torch.empty(seqs, heads, dim, dtype=dtype, device="cuda")
        mxk.cache_attention_shared(cache, q, cu_q, rows, torch.full((seqs,), length, **i32), groups, prefixes, out, max_q=1,
                                   max_kv=longest, max_prefix=longest)
        want = torch.empty(seqs, heads, dim, dtype=torch.float64, device="cuda")
        for i in range(seqs):
            keys[i].append(torch.from_numpy(k[i:i + 1]).cuda()), values[i].append(torch.from_numpy(v[i:i + 1]).cuda())
            ks, vs = (torch.cat(t[i]).repeat_interleave(heads // kv_heads, 1) for t in (keys, values))
            s = torch.einsum("hd,thd->ht", q[i].double(), ks) * dim ** -0.5
            want[i] = torch.einsum("ht,thd->hd", torch.softmax(s, -1), vs)
        # half a step of bfloat16, and of float16 for the weights
        assert relative(out, want) < 2.0 ** -8 + 2.0 ** -11
        y, want = project(out.view(seqs, -1), w_out)
        assert relative(y, want) < 2.0 ** -8


@pytest.mark.parametrize("bits,prompt", [(8, 4000), (6, 2900), (4, 130)])
def test_example_of_conversations_behind_an_instruction(torch_cuda, mxk, bits, prompt):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(mxk.__file__), "examples", "serve_prefix.py")
    spec = importlib.util.spec_from_file_location("serve_prefix", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # half a step of bfloat16 in the output, and of float16 in the weights
    assert example.main(bits=bits, prompt=prompt, steps=6, batch=40) < 2.0 ** -8 + 2.0 ** -11
