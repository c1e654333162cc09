"""Attention over the paged MX cache against the definition in float64.

Tolerance, per output element, from the arithmetic alone: the output's own
rounding (half a unit: 2^-8 of it in bf16, 2^-11 in f16), exp(s) rounded to f16 before the product with v (2^-11 of sum p |v|), an error of each
score of at most `ds` (float32 sums of the products, q rounded to f16 below 2^-25 of
its row's largest: 2^-19 * scale * max_t sum_d |q_d k_td|), which changes every weight
by a factor within exp(+-2 ds), values below 2^-26 of the head's largest magnitude,
and the subnormal step of the output type.
"""
import math

import numpy as np
import pytest
from test_cache_gpu import decode

pytestmark = pytest.mark.gpu


def build(torch, mxk, g, q_lens, kv_lens, heads, kv_heads, dim, page, bits, dtype, scale_k=1.0, scale_v=1.0,
          stale=True, cached=None):
    """A filled cache with a shuffled page table, and q.  Slots no sequence owns hold
    the worst bytes there are (NaN codes and scales)."""
    seqs = len(q_lens)
    width = max(1, max(-(-max(l, 1) // page) for l in kv_lens))
    pages = sum(-(-l // page) for l in kv_lens) + 2
    order = g.permutation(pages)
    table = np.full((seqs, width), pages - 1, np.int32)
    cache = mxk.PagedCache.empty(pages, page, kv_heads, dim, bits)
    for t in (cache.k_values, cache.k_scales, cache.v_values, cache.v_scales):
        t.fill_(0xff if stale else 0)
    at = 0
    rows = []
    for i, l in enumerate(kv_lens):
        m = -(-l // page)
        table[i, :m] = order[at:at + m]
        at += m
        if cached is not None:
            k, v = cached[i]
        else:
            k = (g.standard_normal((l, kv_heads, dim)) * scale_k).astype(np.float32)
            v = (g.standard_normal((l, kv_heads, dim)) * scale_v).astype(np.float32)
            if l:
                k[:, :, :3] *= 6  # a few loud features
        slots = table[i, np.arange(l) // page].astype(np.int64) * page + np.arange(l) % page
        if l:
            mxk.cache_write(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(),
                            torch.from_numpy(slots).cuda())
        rows.append(slots)
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    q = torch.from_numpy(g.standard_normal((int(cu[-1]), heads, dim)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    return dict(cache=cache, table=torch.from_numpy(table).cuda(), cu=torch.from_numpy(cu).cuda(),
                kv=torch.tensor(kv_lens, dtype=torch.int32).cuda(), q=q, slots=rows, q_lens=q_lens, kv_lens=kv_lens)


def attend(torch, mxk, b, lse=True, q=None, out=None, max_q=None, max_kv=None, **kw):
    q = b["q"] if q is None else q
    out = torch.full_like(q, 77.0) if out is None else out
    z = torch.full(q.shape[:2], 55.0, dtype=torch.float32, device="cuda") if lse else None
    mxk.cache_attention(b["cache"], q, b["cu"], b["table"], b["kv"], out, max_q=max_q or max(b["q_lens"]),
                        max_kv=max_kv or max(max(b["kv_lens"]), 1), lse=z, **kw)
    torch.cuda.synchronize()
    return out, z


def cached_rows(torch, b, i):
    """float64 keys and values of sequence i, from the cache's bytes."""
    c, s = b["cache"], b["slots"][i]
    out = []
    for values, scales in ((c.k_values, c.k_scales), (c.v_values, c.v_scales)):
        page, place = s // c.page_size, s % c.page_size
        with np.errstate(invalid="ignore"):
            out.append(decode(values.cpu().numpy()[page, :, place], scales.cpu().numpy()[page, :, place], c.bits))
    return [torch.from_numpy(x.astype(np.float64)).cuda() for x in out]


def check(torch, b, out, lse, scale=None, causal=True, window=0):
    c = b["cache"]
    heads = b["q"].shape[1]
    group = heads // c.kv_heads
    scale = c.head_dim ** -0.5 if scale is None else scale
    u = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -11
    tiny = 0.0 if out.dtype == torch.bfloat16 else 2.0 ** -25
    row = 0
    for i, (n, l) in enumerate(zip(b["q_lens"], b["kv_lens"])):
        k, v = cached_rows(torch, b, i)
        p = l - n + torch.arange(n, device="cuda")
        t = torch.arange(l, device="cuda")
        see = torch.ones(n, l, dtype=torch.bool, device="cuda")
        if causal:
            see &= t[None] <= p[:, None]
        if window:
            see &= t[None] > p[:, None] - window
        some = see.any(-1)
        for h in range(heads):
            q = b["q"][row:row + n, h].double()
            kh, vh = k[:, h // group], v[:, h // group]
            s = torch.where(see, scale * (q @ kh.T), -math.inf)
            z = torch.logsumexp(s, -1) if l else torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
            w = torch.where(see, torch.exp(s - torch.where(some, z, 0.0)[:, None]), 0.0)
            want, size = w @ vh, w @ vh.abs()
            ds = (2.0 ** -19 * abs(scale) * torch.where(see, q.abs() @ kh.abs().T, 0.0).amax(-1)) if l else p * 0.0
            most = vh.abs().max() if l else 0.0
            tol = u * want.abs() + (2.0 ** -11 + 2.0 ** -20 + torch.expm1(2 * ds)[:, None]) * size * (1 + u) + \
                2.0 ** -26 * most + tiny
            got = out[row:row + n, h].double()
            assert not torch.isnan(got).any(), f"sequence {i} head {h}: NaN"
            bad = ~((got - want).abs() <= tol)
            assert not bad.any(), (f"sequence {i} head {h}: {int(bad.sum())} values off, worst "
                                   f"{float(((got - want).abs() - tol).max())}")
            assert (got[~some] == 0).all()
            if lse is not None:
                g = lse[row:row + n, h].double()
                assert (g[~some] == -math.inf).all()
                assert ((g - z).abs()[some] <= (ds + 2.0 ** -20 * (1 + z.abs()))[some]).all()
        row += n


ALL = [(bits, dim, dtype) for bits in (8, 6, 4) for dim in (64, 128) for dtype in ("bfloat16", "float16")]


@pytest.mark.parametrize("bits,dim,dtype", ALL)
def test_single_tokens(torch_cuda, mxk, bits, dim, dtype):
    """One new token per sequence, lengths around the granules and pages, some empty."""
    torch, g = torch_cuda, np.random.default_rng(1)
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 333, 1, 500]
    b = build(torch, mxk, g, [1] * len(kv), kv, 8, 2, dim, 16, bits, dtype)
    check(torch, b, *attend(torch, mxk, b))


@pytest.mark.parametrize("bits,dim,dtype", ALL)
def test_ragged_chunks(torch_cuda, mxk, bits, dim, dtype):
    """Chunks of every size beside single tokens and sequences without queries or keys;
    three queries more than keys leave rows that see nothing."""
    torch, g = torch_cuda, np.random.default_rng(2)
    q_lens = [5, 0, 1, 130, 7, 3, 0, 33, 260]
    kv_lens = [5, 9, 700, 131, 4, 0, 0, 400, 300]
    b = build(torch, mxk, g, q_lens, kv_lens, 6, 2, dim, 48, bits, dtype)
    check(torch, b, *attend(torch, mxk, b))
    check(torch, b, *attend(torch, mxk, b, causal=False), causal=False)


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
@pytest.mark.parametrize("q_len", [1, 3, 150])
def test_window(torch_cuda, mxk, window, q_len):
    torch, g = torch_cuda, np.random.default_rng(window)
    b = build(torch, mxk, g, [q_len, q_len, 1, q_len], [q_len, 777, 300, 1030], 4, 2, 64, 32, 8, "float16")
    check(torch, b, *attend(torch, mxk, b, window=window), window=window)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (16, 1), (24, 1), (40, 2), (5, 5), (32, 8)])
@pytest.mark.parametrize("q_len", [1, 4, 70])
def test_head_groups(torch_cuda, mxk, heads, kv_heads, q_len):
    torch, g = torch_cuda, np.random.default_rng(heads)
    b = build(torch, mxk, g, [q_len, max(1, q_len // 2)], [201, 90], heads, kv_heads, 128, 64, 8, "bfloat16")
    check(torch, b, *attend(torch, mxk, b))


@pytest.mark.parametrize("q_len,kv_len,kv_heads", [(1, 20000, 1), (1, 9973, 3), (40, 9000, 1), (300, 5000, 1)])
@pytest.mark.parametrize("bits", [8, 4])
def test_long_axis_is_split_and_joined(torch_cuda, mxk, q_len, kv_len, kv_heads, bits):
    torch, g = torch_cuda, np.random.default_rng(3)
    b = build(torch, mxk, g, [q_len], [kv_len], 4 * kv_heads, kv_heads, 128, 128, bits, "bfloat16", scale_k=2.0)
    out, lse = attend(torch, mxk, b)
    check(torch, b, out, lse)
    again, lse2 = attend(torch, mxk, b)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "the same call twice differs"


@pytest.mark.parametrize("q_len,kv_len,seqs,heads,kv_heads", [(1, 400, 150, 16, 8), (9, 260, 60, 28, 4),
                                                              (40, 300, 60, 12, 4), (138, 150, 40, 12, 6),
                                                              (100, 700, 30, 32, 8)])
@pytest.mark.parametrize("bits,dim", [(8, 128), (4, 64)])
def test_several_units_per_block(torch_cuda, mxk, q_len, kv_len, seqs, heads, kv_heads, bits, dim):
    """More (sequence, head, row tile) units than the GPU has blocks: every block works
    through several, whole and in part, with row tiles full and nearly empty."""
    torch, g = torch_cuda, np.random.default_rng(16)
    kv = [kv_len - int(x) for x in g.integers(0, kv_len // 2, seqs)]
    q_lens = [min(l, q_len - int(x)) for l, x in zip(kv, g.integers(0, q_len // 3 + 1, seqs))]
    b = build(torch, mxk, g, q_lens, kv, heads, kv_heads, dim, 16, bits, "bfloat16")
    out, lse = attend(torch, mxk, b)
    check(torch, b, out, lse)
    again, lse2 = attend(torch, mxk, b)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("q_len,kv_len,seqs,heads,kv_heads", [(1, 600, 45, 8, 4), (2, 300, 400, 4, 2),
                                                              (1, 90, 700, 4, 2), (16, 600, 10, 16, 4),
                                                              (30, 1800, 10, 16, 4), (90, 700, 12, 16, 4)])
@pytest.mark.parametrize("bits,dim,window", [(8, 128, 0), (4, 64, 0), (6, 64, 70)])
def test_few_tiles_per_block(torch_cuda, mxk, q_len, kv_len, seqs, heads, kv_heads, bits, dim, window):
    """One to a few key tiles for every block: where a block's share ends between a unit's
    start and its first tile, blocks with nothing to do, more sequences than threads."""
    torch, g = torch_cuda, np.random.default_rng(17)
    kv = [kv_len - int(x) for x in g.integers(0, 41, seqs)]
    b = build(torch, mxk, g, [q_len] * seqs, kv, heads, kv_heads, dim, 16, bits, "float16")
    out, lse = attend(torch, mxk, b, window=window)
    check(torch, b, out, lse, window=window)
    again, lse2 = attend(torch, mxk, b, window=window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_many_sequences(torch_cuda, mxk):
    """More sequences than a CTA has threads, many of them empty."""
    torch, g = torch_cuda, np.random.default_rng(4)
    kv = [int(x) for x in g.integers(0, 40, 700)]
    q_lens = [min(l, int(x)) for l, x in zip(kv, g.integers(0, 3, 700))]
    b = build(torch, mxk, g, q_lens, kv, 2, 1, 64, 16, 8, "float16")
    check(torch, b, *attend(torch, mxk, b))


@pytest.mark.parametrize("q_len", [1, 6, 200])
def test_bounds_may_be_loose(torch_cuda, mxk, q_len):
    torch, g = torch_cuda, np.random.default_rng(5)
    b = build(torch, mxk, g, [q_len, 1], [600, 300], 4, 2, 128, 64, 8, "bfloat16")
    tight = attend(torch, mxk, b)
    loose = attend(torch, mxk, b, max_q=q_len + 1000, max_kv=640)
    check(torch, b, *tight)
    check(torch, b, *loose)


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("q_len", [1, 12, 160])
def test_large_and_small_magnitudes(torch_cuda, mxk, bits, q_len):
    """Values whose scale grows and falls by 2^30 along the sequence, keys whose blocks
    differ by 2^20, scores in the hundreds: one token takes nearly all the weight."""
    torch, g = torch_cuda, np.random.default_rng(6)
    l, h, d = 700, 2, 128
    k = g.standard_normal((l, h, d)).astype(np.float32)
    k[:, :, 32:64] *= 2.0 ** -20
    k *= np.exp(g.standard_normal((l, h, 1)) * 2).astype(np.float32)
    v = g.standard_normal((l, h, d)).astype(np.float32)
    v *= np.ldexp(1.0, (15 * np.sin(np.arange(l) / 40)).astype(int))[:, None, None].astype(np.float32)
    v[:, :, 64:96] *= 2.0 ** 8
    b = build(torch, mxk, g, [q_len], [l], 4, h, d, 32, bits, "bfloat16", cached=[(k, v)])
    b["q"].mul_(4)
    check(torch, b, *attend(torch, mxk, b))
    check(torch, b, *attend(torch, mxk, b, scale=-0.5), scale=-0.5)
    check(torch, b, *attend(torch, mxk, b, scale=0.0), scale=0.0)


@pytest.mark.parametrize("q_len", [1, 16, 140])
def test_extreme_queries(torch_cuda, mxk, q_len):
    """Rows of zeros, rows far below and above f16's range."""
    torch, g = torch_cuda, np.random.default_rng(7)
    b = build(torch, mxk, g, [q_len], [300], 4, 2, 64, 16, 8, "bfloat16")
    f = torch.tensor([0.0, 1e-30, 3e-39, 1e8], device="cuda")
    b["q"] = (b["q"].float() * f[None, :, None]).to(torch.bfloat16)
    check(torch, b, *attend(torch, mxk, b, scale=1e-6), scale=1e-6)


@pytest.mark.parametrize("q_len", [4, 33, 300])
def test_nan_reaches_only_rows_that_see_it(torch_cuda, mxk, q_len):
    """A NaN key or value in the middle of the chunk: earlier rows keep their results
    bit for bit, later ones become NaN (in the NaN's feature only, for a value)."""
    torch, g = torch_cuda, np.random.default_rng(8)
    l, n = 450, q_len
    b = build(torch, mxk, g, [n], [l], 4, 2, 128, 64, 8, "bfloat16")
    clean, z = attend(torch, mxk, b)
    at = l - n + n // 2
    slot = int(b["slots"][0][at])
    page, place = slot // 64, slot % 64
    keep = int(b["cache"].v_values[page, 1, place, 37])
    b["cache"].v_values[page, 1, place, 37] = 0x7f
    out, z2 = attend(torch, mxk, b)
    assert torch.equal(z, z2)
    assert torch.equal(out[:, :2], clean[:, :2])
    assert torch.equal(out[:n // 2], clean[:n // 2])
    assert torch.isnan(out[n // 2:, 2:, 37]).all()
    rest = torch.arange(128, device="cuda") != 37
    assert torch.equal(out[:, 2:, rest], clean[:, 2:, rest])
    b["cache"].v_values[page, 1, place, 37] = keep
    b["cache"].k_values[page, 1, place, 5] = 0xff
    out, z2 = attend(torch, mxk, b)
    assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[:n // 2], clean[:n // 2])
    assert torch.isnan(out[n // 2:, 2:]).all() and torch.isnan(z2[n // 2:, 2:]).all()
    # a NaN outside a window
    out, _ = attend(torch, mxk, b, window=1)
    assert torch.isnan(out[n // 2, 2:]).all()
    others = torch.arange(n, device="cuda") != n // 2
    assert not torch.isnan(out[others]).any()


def test_nan_and_infinite_queries_stay_in_their_rows(torch_cuda, mxk):
    torch, g = torch_cuda, np.random.default_rng(9)
    for n in (4, 150):
        b = build(torch, mxk, g, [n], [200], 4, 2, 64, 16, 8, "float16")
        clean, _ = attend(torch, mxk, b)
        b["q"][1, 2, 3] = float("nan")
        b["q"][3, 0, 3] = float("inf")
        out, _ = attend(torch, mxk, b)
        assert torch.isnan(out[1, 2]).all() and torch.isnan(out[3, 0]).all()
        keep = torch.ones(n, 4, dtype=torch.bool, device="cuda")
        keep[1, 2] = keep[3, 0] = False
        assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("q_len", [2, 140])
@pytest.mark.parametrize("pad,shift", [(4, 0), (1, 0), (3, 1), (0, 2)])
def test_strided_queries_and_outputs(torch_cuda, mxk, q_len, pad, shift):
    torch, g = torch_cuda, np.random.default_rng(10)
    b = build(torch, mxk, g, [q_len, 1], [300, 40], 6, 2, 64, 16, 8, "float16")
    want, _ = attend(torch, mxk, b)
    t, h, d = b["q"].shape
    wide = torch.zeros(t, h * (d + pad) + shift, dtype=torch.float16, device="cuda")
    q = wide[:, shift:].unflatten(1, (h, d + pad))[:, :, :d]
    q.copy_(b["q"])
    back = torch.full((h, t, d + pad), 9.0, dtype=torch.float16, device="cuda")
    out = back[:, :, :d].transpose(0, 1)
    attend(torch, mxk, b, q=q, out=out)
    assert torch.equal(out, want)
    assert (back[:, :, d:] == 9.0).all()


@pytest.mark.parametrize("q_len", [1, 140])
def test_side_stream_and_graph(torch_cuda, mxk, q_len):
    """On a stream of the caller's, and replayed from a graph after the lengths and
    the cache have moved on."""
    torch, g = torch_cuda, np.random.default_rng(11)
    b = build(torch, mxk, g, [q_len], [900], 8, 2, 128, 64, 8, "bfloat16")
    want, _ = attend(torch, mxk, b)
    side = torch.cuda.Stream()
    out = torch.empty_like(want)

    def call():
        mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=q_len, max_kv=960)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    every = b["slots"][0]
    for length in (900, 880, 901 - q_len):
        b["kv"].fill_(length)
        b["kv_lens"] = [length]
        b["slots"] = [every[:length]]
        graph.replay()
        torch.cuda.synchronize()
        check(torch, b, out, None)


def test_offsets_past_32_bits(torch_cuda, mxk):
    """Pages past 2^31 bytes of the buffers."""
    torch, g = torch_cuda, np.random.default_rng(12)
    pages, page, h, d = 2200, 128, 64, 128
    cache = mxk.PagedCache.empty(pages, page, h, d, 8)
    for n in (1, 40):
        small = build(torch, mxk, g, [n], [200], h, h, d, page, 8, "bfloat16")
        far = torch.tensor([[pages - 1, pages - 5]], dtype=torch.int32, device="cuda")
        for a, s in ((cache.k_values, small["cache"].k_values), (cache.k_scales, small["cache"].k_scales),
                     (cache.v_values, small["cache"].v_values), (cache.v_scales, small["cache"].v_scales)):
            for i in range(2):
                a[far[0, i].long()] = s[small["table"][0, i].long()]
        want, _ = attend(torch, mxk, small)
        got, _ = attend(torch, mxk, dict(small, cache=cache, table=far))
        assert torch.equal(got, want)


def test_wild_page_numbers_and_lengths_stay_inside(torch_cuda, mxk):
    """Page numbers, lengths and row ranges outside their bounds read and write nothing
    outside the buffers; other sequences keep their results."""
    torch, g = torch_cuda, np.random.default_rng(13)
    for n in (1, 90):
        b = build(torch, mxk, g, [n, n], [300, 200], 4, 2, 64, 16, 8, "float16", stale=False)
        want, _ = attend(torch, mxk, b)
        wild = dict(b, table=b["table"].clone(), kv=b["kv"].clone())
        wild["table"][1] = torch.tensor([-5, 2 ** 31 - 1] + [10 ** 6] * (b["table"].shape[1] - 2),
                                        dtype=torch.int32, device="cuda")
        wild["kv"][1] = 2 ** 31 - 1
        out, _ = attend(torch, mxk, wild)
        assert torch.equal(out[:n], want[:n])
        wild["cu"] = torch.tensor([0, n, 10 ** 9], dtype=torch.int32, device="cuda")
        out, _ = attend(torch, mxk, wild)
        assert torch.equal(out[:n], want[:n])


def test_write_then_attend_step(torch_cuda, mxk):
    """A serving loop: every step stores the new tokens' rows and attends; after it the
    results equal those of one chunk over the whole prompt."""
    torch, g = torch_cuda, np.random.default_rng(14)
    h, hk, d, page, total = 4, 2, 64, 16, 70
    q, k, v = (torch.from_numpy(g.standard_normal((total, n, d)).astype(np.float32)).cuda().to(torch.bfloat16)
               for n in (h, hk, hk))
    cache = mxk.PagedCache.empty(8, page, hk, d, 8)
    table = torch.tensor([[5, 0, 7, 2, 3]], dtype=torch.int32, device="cuda")
    at = torch.arange(total, device="cuda")
    slots = table[0, at // page].long() * page + at % page
    steps = torch.empty_like(q)
    done = 0
    for n in (30, 1, 1, 5, 1, 32):
        sl = slice(done, done + n)
        mxk.cache_write(cache, k[sl], v[sl], slots[sl])
        done += n
        mxk.cache_attention(cache, q[sl], torch.tensor([0, n], dtype=torch.int32, device="cuda"), table,
                            torch.tensor([done], dtype=torch.int32, device="cuda"), steps[sl], max_q=n, max_kv=done)
    assert done == total
    b = dict(cache=cache, table=table, cu=torch.tensor([0, total], dtype=torch.int32, device="cuda"),
             kv=torch.tensor([total], dtype=torch.int32, device="cuda"), q=q, slots=[slots.cpu().numpy()],
             q_lens=[total], kv_lens=[total])
    check(torch, b, steps, None)
    check(torch, b, *attend(torch, mxk, b))


def test_binding_refusals(torch_cuda, mxk):
    torch, g = torch_cuda, np.random.default_rng(15)
    b = build(torch, mxk, g, [2], [20], 4, 2, 64, 16, 8, "float16")
    q, out = b["q"], torch.empty_like(b["q"])

    def call(q=q, cu=b["cu"], table=b["table"], kv=b["kv"], out=out, **kw):
        mxk.cache_attention(b["cache"], q, cu, table, kv, out, **{"max_q": 2, "max_kv": 20, **kw})

    call()
    bad = [dict(q=q.float()), dict(q=q[:, :3], out=out[:, :3]), dict(q=q.cpu()), dict(out=out.to(torch.bfloat16)),
           dict(out=out[:1]), dict(cu=b["cu"].long()), dict(kv=b["kv"].long()), dict(table=b["table"][0]),
           dict(max_kv=33), dict(q=q.transpose(1, 2)), dict(window=-1), dict(window=2, causal=False),
           dict(lse=torch.empty(2, 4, device="cuda", dtype=torch.float64)), dict(scale=float("nan"))]
    for kw in bad:
        with pytest.raises(mxk.MxkInvalidArgument):
            call(**kw)
    k = torch.zeros(2, 2, 64, device="cuda")
    slots = torch.arange(2, device="cuda")
    for args in ((k, k[:1], slots), (k, k.half(), slots), (k, k, slots.int()), (k[:, :, :32], k, slots),
                 (k, k, slots[:1]), (k.int(), k.int(), slots)):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.cache_write(b["cache"], *args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [8, 4])
def test_serving_example(torch_cuda, mxk, bits):
    """The example's loop; what remains is the output's rounding and that of the weights."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(mxk.__file__), "examples", "serve_cache.py")
    spec = importlib.util.spec_from_file_location("serve_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(bits=bits, steps=9) < 2.0 ** -8 + 2.0 ** -10
