"""Attention over the paged MX cache with shared prefixes against the definition in float64,
with the tolerances of test_cache_attention_gpu (the merge's float32 steps lie within its
2^-20 of the weights and its errors of the scores)."""
import numpy as np
import pytest
from test_cache_attention_gpu import ALL, check

pytestmark = pytest.mark.gpu


def build(torch, mxk, g, groups, heads, kv_heads, dim, page, bits, dtype, scale_k=1.0, scale_v=1.0):
    """groups: (prefix, told, [(new tokens, own tokens)]) each: the first `prefix` tokens (whole
    pages) lie in the same pages for all its sequences, `told` is what the call is told of;
    told = None: the sequences belong to no group.  Slots that nobody owns hold the worst bytes."""
    flat = [(i, p, q, o) for i, (p, _, seqs) in enumerate(groups) for q, o in seqs]
    need = sum(p // page + sum(-(-o // page) for _, o in seqs) for p, _, seqs in groups)
    pages = need + 2
    order = g.permutation(pages)
    width = max(1, max(p // page + -(-o // page) for _, p, _, o in flat))
    table = np.full((len(flat), width), pages - 1, np.int32)
    cache = mxk.PagedCache.empty(pages, page, kv_heads, dim, bits)
    for t in (cache.k_values, cache.k_scales, cache.v_values, cache.v_scales):
        t.fill_(0xff)

    def fill(slots):
        k = (g.standard_normal((len(slots), kv_heads, dim)) * scale_k).astype(np.float32)
        v = (g.standard_normal((len(slots), kv_heads, dim)) * scale_v).astype(np.float32)
        if len(slots):
            k[:, :, :3] *= 6  # a few loud features
            mxk.cache_write(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.from_numpy(slots).cuda())

    at, row, slots, cu_groups, told = 0, 0, [], [], []
    for prefix, tell, seqs in groups:
        assert prefix % page == 0
        shared = order[at:at + prefix // page]
        at += len(shared)
        common = (shared.astype(np.int64)[:, None] * page + np.arange(page)).reshape(-1)
        fill(common)
        if tell is not None:
            if not cu_groups:
                cu_groups = [row]
            assert cu_groups[-1] == row, "sequences without a group come first or last"
            cu_groups.append(row + len(seqs))
            told.append(tell)
        for _, own in seqs:
            mine = order[at:at + -(-own // page)]
            at += len(mine)
            table[row, :len(shared)] = shared
            table[row, len(shared):len(shared) + len(mine)] = mine
            places = (mine.astype(np.int64)[:, None] * page + np.arange(page)).reshape(-1)[:own]
            fill(places)
            slots.append(np.concatenate([common, places]))
            row += 1
    q_lens, kv_lens = [q for _, _, q, _ in flat], [p + o for _, p, _, o in flat]
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    q = torch.from_numpy(g.standard_normal((int(cu[-1]), heads, dim)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(cache=cache, table=torch.from_numpy(table).cuda(), cu=torch.from_numpy(cu).cuda(),
                kv=torch.tensor(kv_lens, **i32), q=q, slots=slots, q_lens=q_lens, kv_lens=kv_lens,
                groups=torch.tensor(cu_groups, **i32), prefixes=torch.tensor(told, **i32), most=max(told + [0]))


def wide_bounds(torch, b):
    """Bounds on prefixes and tokens from which on a call shares whatever there is, and a page
    table for them (the added pages are never looked at)."""
    cache, spare = b["cache"], min(len(b["q_lens"]), sum(b["q_lens"])) - len(b["prefixes"])
    if spare <= 0:
        return b["table"], max(max(b["kv_lens"]), 1), b["most"]
    tokens = max(-(-(400 << 10) * 128 // (cache.head_dim * spare * cache.kv_heads)), b["most"], *b["kv_lens"])
    tokens = -(-tokens // 128) * 128
    more = -(-tokens // cache.page_size) - b["table"].shape[1]
    return torch.nn.functional.pad(b["table"], (0, max(more, 0)), value=1 << 30), tokens, tokens


def attend(torch, mxk, b, lse=True, q=None, out=None, max_q=None, max_kv=None, max_prefix=None, tight=False, **kw):
    """tight, or with bounds that are given: it goes by the sizes whether the call shares."""
    q = b["q"] if q is None else q
    if not tight and max_kv is None and max_prefix is None:
        b = dict(b)
        b["table"], max_kv, max_prefix = wide_bounds(torch, b)
    out = torch.full_like(q, 77.0) if out is None else out
    z = torch.full(q.shape[:2], 55.0, dtype=torch.float32, device="cuda") if lse else None
    mxk.cache_attention_shared(b["cache"], q, b["cu"], b["table"], b["kv"], b["groups"], b["prefixes"], out,
                               max_q=max_q or max(b["q_lens"]), max_kv=max_kv or max(max(b["kv_lens"]), 1),
                               max_prefix=b["most"] if max_prefix is None else max_prefix, lse=z, **kw)
    torch.cuda.synchronize()
    return out, z


@pytest.mark.parametrize("bits,dim,dtype", ALL)
def test_single_tokens(torch_cuda, mxk, bits, dim, dtype):
    """Groups with few rows a key head, with a row tile's and with more than two, their own
    tokens around the tiles' edges."""
    torch, g = torch_cuda, np.random.default_rng(1)
    owns = [1, 2, 127, 128, 129, 300]
    groups = [(640, 640, [(1, owns[i % 6]) for i in range(n)]) for n in (3, 20, 70)]
    b = build(torch, mxk, g, groups, 8, 2, dim, 16, bits, dtype)
    check(torch, b, *attend(torch, mxk, b))


@pytest.mark.parametrize("bits,dim,dtype", ALL)
def test_ragged_chunks(torch_cuda, mxk, bits, dim, dtype):
    """Chunks beside single tokens, sequences without queries, prefixes of all kinds of lengths,
    sequences in no group first and last."""
    torch, g = torch_cuda, np.random.default_rng(2)
    groups = [(96, None, [(1, 40), (5, 300)]),
              (480, 470, [(1, 10), (0, 33), (3, 3), (1, 600)]),
              (48, 48, [(2, 7), (4, 9)]),
              (1200, 1200, [(130, 140), (1, 50), (7, 7), (33, 400), (260, 300)]),
              (144, 144, [(1, 1)]),
              (0, 0, [(2, 5), (1, 1)]),
              (0, None, [(0, 0), (9, 200)])]
    b = build(torch, mxk, g, groups, 6, 2, dim, 48, bits, dtype)
    check(torch, b, *attend(torch, mxk, b))
    check(torch, b, *attend(torch, mxk, b, causal=False), causal=False)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (7, 1), (40, 8), (64, 1)])
def test_head_layouts(torch_cuda, mxk, heads, kv_heads):
    torch, g = torch_cuda, np.random.default_rng(3)
    groups = [(256, 256, [(1, 9), (2, 70), (1, 1)]), (384, 384, [(1, 5)] * 9)]
    b = build(torch, mxk, g, groups, heads, kv_heads, 64, 64, 8, "float16")
    check(torch, b, *attend(torch, mxk, b))


@pytest.mark.parametrize("told", [0, 1, 127, 128, 511, 640, 700, 5000])
def test_what_is_told_of_a_prefix(torch_cuda, mxk, told):
    """Less than what is shared, or more: then what comes before the query tokens is, as far as
    the pages are alike."""
    torch, g = torch_cuda, np.random.default_rng(4)
    # own tokens are query tokens alone, so a prefix that is told too long ends before them
    b = build(torch, mxk, g, [(640, told, [(1, 1), (3, 3), (2, 2)])], 8, 2, 128, 32, 8, "bfloat16")
    check(torch, b, *attend(torch, mxk, b))
    for most in (0, 100, 128, 300):
        check(torch, b, *attend(torch, mxk, b, max_prefix=most))
    check(torch, b, *attend(torch, mxk, b, tight=True))


@pytest.mark.parametrize("most", [127, 128, 300, 384, 1000])
def test_prefix_longer_than_its_bound(torch_cuda, mxk, most):
    """32 key heads of one row a sequence: a prefix of 128 tokens is worth it."""
    torch, g = torch_cuda, np.random.default_rng(18)
    b = build(torch, mxk, g, [(384, 384, [(1, 1 + i) for i in range(30)])], 32, 32, 64, 16, 8, "bfloat16")
    check(torch, b, *attend(torch, mxk, b, max_prefix=most))


@pytest.mark.parametrize("new", [1, 8, 25, 70, 300])
def test_sizes_around_what_is_worth_sharing(torch_cuda, mxk, new):
    """Bounds that are tight, where some calls share and others do not."""
    torch, g = torch_cuda, np.random.default_rng(19)
    for prefix in (512, 2048, 6144):
        b = build(torch, mxk, g, [(prefix, prefix, [(new, new + 7 * i) for i in range(6)])], 8, 2, 128, 64, 8, "bfloat16")
        check(torch, b, *attend(torch, mxk, b, tight=True))
        check(torch, b, *attend(torch, mxk, b))


def test_rows_that_see_nothing(torch_cuda, mxk):
    """More queries than tokens in one sequence of a group: the group shares nothing."""
    torch, g = torch_cuda, np.random.default_rng(5)
    b = build(torch, mxk, g, [(256, 256, [(1, 9), (260, 2)] + [(0, 0)] * 4), (128, 128, [(2, 3), (1, 1)])], 4, 2, 64, 16, 6, "float16")
    check(torch, b, *attend(torch, mxk, b))
    b = build(torch, mxk, g, [(0, 128, [(1, 0), (2, 0)])], 4, 2, 64, 16, 6, "float16")
    out, lse = attend(torch, mxk, b)
    assert (out == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("n", [3, 30, 90, 120])
def test_long_prefix(torch_cuda, mxk, n):
    """A prefix that all CTAs share, joined from many parts; without lse."""
    torch, g = torch_cuda, np.random.default_rng(6)
    b = build(torch, mxk, g, [(20480, 20480, [(1, 1 + 13 * i % 50) for i in range(n)])], 8, 2, 64, 128, 4, "bfloat16")
    out, lse = attend(torch, mxk, b)
    check(torch, b, out, lse)
    again, _ = attend(torch, mxk, b, lse=False)
    assert torch.equal(out, again), "a result depends on timing"


def test_as_the_ordinary_call(torch_cuda, mxk):
    """Nothing to share: the ordinary call's bits."""
    torch, g = torch_cuda, np.random.default_rng(7)
    b = build(torch, mxk, g, [(64, 64, [(1, 300), (5, 40)]), (256, 256, [(3, 7)])], 8, 2, 128, 64, 8, "bfloat16")
    want = torch.empty_like(b["q"])
    mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], want, max_q=5, max_kv=364)
    for most in (256, 127, 0):
        out, _ = attend(torch, mxk, b, max_prefix=most)
        assert (out.float() - want.float()).norm() <= 2.0 ** -8 * want.float().norm()
        if most < 128:
            assert torch.equal(out, want)


def test_strides_and_rows_behind(torch_cuda, mxk):
    """Queries and outputs as slices of wider tensors; rows behind the last sequence stay."""
    torch, g = torch_cuda, np.random.default_rng(8)
    b = build(torch, mxk, g, [(256, 256, [(1, 9), (4, 30), (0, 3), (2, 2)]), (128, None, [(1, 3)])], 6, 3, 64, 32, 8, "bfloat16")
    n = b["q"].shape[0]
    for pad in (1, 8):
        wide = torch.full((n + 3, 9, 64 + pad), 3.0, dtype=torch.bfloat16, device="cuda")
        wide[:n, 1:7, :64] = b["q"]
        out = torch.full((n + 3, 9, 64 + pad), 77.0, dtype=torch.bfloat16, device="cuda")
        _, lse = attend(torch, mxk, b, q=wide[:, 1:7, :64], out=out[:, 2:8, :64])
        check(torch, b, out[:n, 2:8, :64], lse[:n])
        rest = out.clone()
        rest[:n, 2:8, :64] = 77.0
        assert (rest == 77.0).all() and (lse[n:] == 55.0).all()


def test_magnitudes_stay_in_their_rows(torch_cuda, mxk):
    """Huge values in a sequence's own tokens, and NaNs in another group's prefix."""
    torch, g = torch_cuda, np.random.default_rng(9)
    groups = [(256, 256, [(1, 40), (1, 30), (2, 20)]), (256, 256, [(1, 9), (1, 8)])]
    b = build(torch, mxk, g, groups, 4, 2, 64, 32, 8, "bfloat16")
    want, want_lse = attend(torch, mxk, b)
    c = b["cache"]
    loud = torch.from_numpy(b["slots"][1][260:262]).cuda()
    big = torch.full((2, 2, 64), 1e30, device="cuda")
    mxk.cache_write(c, torch.zeros_like(big), big, loud)
    bad = torch.from_numpy(b["slots"][3][5:6]).cuda()
    mxk.cache_write(c, torch.full((1, 2, 64), float("nan"), device="cuda"), torch.zeros(1, 2, 64, device="cuda"), bad)
    out, lse = attend(torch, mxk, b)
    same = [0, 2, 3]
    assert torch.equal(out[same], want[same]) and torch.equal(lse[same], want_lse[same])
    assert (out[1].float() > 1e25).all() and out[4:].isnan().all()


def test_large_scores(torch_cuda, mxk):
    """One token takes all the weight, in the prefix or behind it."""
    torch, g = torch_cuda, np.random.default_rng(10)
    for kind in ("prefix", "own"):
        b = build(torch, mxk, g, [(512, 512, [(1, 40), (1, 30), (1, 600)])], 4, 2, 64, 32, 8, "float16", scale_k=8.0)
        slot = torch.tensor([b["slots"][0][17 if kind == "prefix" else 530]], device="cuda")
        k = b["q"][0].float().view(2, 2, 64).mean(1)[None] * 60
        mxk.cache_write(b["cache"], k.contiguous(), torch.ones(1, 2, 64, device="cuda"), slot)
        check(torch, b, *attend(torch, mxk, b))


def test_captured_and_replayed_as_sequences_grow(torch_cuda, mxk):
    """Lengths, groups and prefixes on the device change between replays; two graphs in turn."""
    torch, g = torch_cuda, np.random.default_rng(11)
    made = [build(torch, mxk, g, groups, 8, 2, 64, 32, 8, "bfloat16") for groups in (
        [(512, 512, [(1, 40), (1, 30), (1, 100)]), (256, 256, [(1, 60), (1, 5)])],
        [(128, 128, [(1, 300), (1, 1)]), (384, 384, [(1, 7), (1, 9), (1, 400)])],
        [(0, 0, [(1, 9), (1, 9), (1, 9), (1, 9)]), (640, 640, [(1, 700)])])]
    base = made[0]
    tables, tokens = zip(*((t, n) for t, n, _ in (wide_bounds(torch, m) for m in made)))
    made = [dict(m, table=t) for m, t in zip(made, tables)]
    width = max(t.shape[1] for t in tables)
    pages = max(m["cache"].pages for m in made)
    cache = mxk.PagedCache.empty(pages, 32, 2, 64, 8)
    held = dict(base, cache=cache, table=torch.zeros(5, width, dtype=torch.int32, device="cuda"),
                cu=base["cu"].clone(), kv=base["kv"].clone(), q=base["q"].clone(), groups=base["groups"].clone(),
                prefixes=base["prefixes"].clone())
    outs = [torch.empty_like(held["q"]) for _ in range(2)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            mxk.cache_attention_shared(cache, held["q"], held["cu"], held["table"], held["kv"], held["groups"],
                                       held["prefixes"], out, max_q=1, max_kv=width * 32, max_prefix=max(tokens))
    for m in made + made[:1]:
        for name in ("k_values", "k_scales", "v_values", "v_scales"):
            getattr(cache, name).fill_(0xff)
            getattr(cache, name)[:m["cache"].pages] = getattr(m["cache"], name)
        held["table"].zero_()
        held["table"][:, :m["table"].shape[1]] = m["table"]
        for name in ("cu", "kv", "q", "groups", "prefixes"):
            held[name].copy_(m[name])
        for graph, out in zip(graphs, outs):
            out.fill_(77.0)
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            check(torch, m, out, None)


def test_bad_tensors_are_refused(torch_cuda, mxk):
    torch, g = torch_cuda, np.random.default_rng(12)
    b = build(torch, mxk, g, [(128, 128, [(1, 9), (1, 8)])], 4, 2, 64, 32, 8, "bfloat16")
    for bad in (dict(groups=b["groups"].long()), dict(groups=b["groups"][:1]), dict(groups=b["groups"].cpu()),
                dict(prefixes=b["prefixes"].float()), dict(prefixes=b["prefixes"].cpu()), dict(kv=b["kv"][:1]),
                dict(table=b["table"][:, :2]), dict(most=-1), dict(q=b["q"].float())):
        with pytest.raises(mxk.MxkInvalidArgument):
            attend(torch, mxk, {**b, **bad}, out=None, tight=True)


# ---- parts of one token, which a warp takes alone where there are many of them

SOLO = [(bits, dim, dtype) for bits in (8, 4) for dim in (64, 128) for dtype in ("bfloat16", "float16")]


@pytest.mark.parametrize("bits,dim,dtype", SOLO)
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (12, 4), (10, 2), (16, 2)])
def test_many_single_tokens(torch_cuda, mxk, bits, dim, dtype, heads, kv_heads):
    """Own tokens around granules, tiles and pages; groups with and without a prefix, sequences
    without queries or tokens, one with several queries, one much longer than the others."""
    torch, g = torch_cuda, np.random.default_rng(13)
    n = 128 // kv_heads + 4
    owns = [1, 2, 15, 16, 17, 31, 33, 47, 48, 49, 95, 96, 127, 128, 129, 300]
    groups = [(0, None, [(1, 700), (0, 5), (0, 0), (1, 0)]),
              (144, 144, [(1, owns[i % 16]) for i in range(n)]),
              (48, 48, [(1, 40), (2, 3), (1, 5)]),
              (384, 384, [(1, 1), (3, 9), (0, 30), (1, 2500)])]
    b = build(torch, mxk, g, groups, heads, kv_heads, dim, 48, bits, dtype)
    check(torch, b, *attend(torch, mxk, b))
    check(torch, b, *attend(torch, mxk, b, causal=False, scale=0.3), causal=False, scale=0.3)


@pytest.mark.parametrize("bits,dim", [(8, 128), (4, 64)])
def test_many_single_tokens_only(torch_cuda, mxk, bits, dim):
    """No sequence has two: prefixes of all sizes go to one kernel.  Unaligned queries, no lse."""
    torch, g = torch_cuda, np.random.default_rng(14)
    groups = [(256, 256, [(1, 1 + 7 * i % 90) for i in range(n)]) for n in (2, 3, 60, 9)] + [(128, None, [(1, 5)] * 3)]
    b = build(torch, mxk, g, groups, 8, 4, dim, 64, bits, "bfloat16")
    want, lse = attend(torch, mxk, b)
    check(torch, b, want, lse)
    n = b["q"].shape[0]
    wide = torch.zeros(n + 2, 8, dim + 1, dtype=torch.bfloat16, device="cuda")
    wide[:n, :, 1:] = b["q"]
    out = torch.full_like(wide, 77.0)
    attend(torch, mxk, b, q=wide[..., 1:], out=out[..., 1:], lse=False)
    assert torch.equal(out[:n, :, 1:], want) and (out[n:] == 77.0).all() and (out[..., 0] == 77.0).all()


@pytest.mark.parametrize("bits,dim", [(8, 128), (8, 64), (4, 128)])
def test_single_tokens_of_many_magnitudes(torch_cuda, mxk, bits, dim):
    """Keys and values that differ by many powers of two from block to block and from token to
    token, blocks of zeros beside tiny values, and single elements that dwarf their block."""
    torch, g = torch_cuda, np.random.default_rng(15)
    b = build(torch, mxk, g, [(128, 128, [(1, 33 + i) for i in range(70)])], 4, 2, dim, 16, bits, "float16", scale_k=0.2)
    for i, kind in enumerate(("blocks", "tokens", "zeros", "tiny", "up", "down")):
        slots = torch.from_numpy(b["slots"][i][128:]).cuda()
        n = len(slots)
        k = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(i)) * 0.2
        v = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(i + 10))
        if kind == "blocks":
            f = torch.exp2(torch.randint(-9, 10, (n, 2, dim // 32, 1), generator=torch.Generator().manual_seed(3)).float())
            v = (v.view(n, 2, -1, 32) * f).view(n, 2, dim)
            k = (k.view(n, 2, -1, 32) / f.clamp(min=1)).view(n, 2, dim)
        elif kind == "tokens":
            v = v * torch.exp2(torch.randint(-10, 11, (n, 1, 1), generator=torch.Generator().manual_seed(4)).float())
        elif kind == "zeros":
            v[::3], k[1::3], v[:, :, :32] = 0, 0, 0
        elif kind == "tiny":
            v = v * 2.0 ** -30
            v[::4] = 0
        elif kind == "up":
            v = v * torch.exp2(torch.arange(n).float() / 3 - 12)[:, None, None]
        else:
            v = v * torch.exp2(12 - torch.arange(n).float() / 3)[:, None, None]
        if kind == "tiny":  # the prefix of its own group is part of what it sees: measured alone below
            continue
        mxk.cache_write(b["cache"], k.cuda(), v.cuda(), slots)
    check(torch, b, *attend(torch, mxk, b))
    # no prefix: what a row sees is tiny values and blocks of zeros
    b = build(torch, mxk, g, [(0, None, [(1, 33 + i) for i in range(70)]), (128, 128, [(1, 1), (1, 2)])], 4, 2, dim, 16, bits,
              "bfloat16", scale_v=2.0 ** -30)
    for i in range(70):
        slots = torch.from_numpy(b["slots"][i][::2]).cuda()
        k = torch.randn(len(slots), 2, dim, device="cuda")
        mxk.cache_write(b["cache"], k, torch.zeros_like(k), slots)
    check(torch, b, *attend(torch, mxk, b))


def test_single_tokens_and_numbers_that_are_none(torch_cuda, mxk):
    """A NaN or an overflowed value stays with its sequence and, where it is a value, its feature."""
    torch, g = torch_cuda, np.random.default_rng(16)
    b = build(torch, mxk, g, [(128, 128, [(1, 20 + i) for i in range(80)])], 4, 2, 64, 32, 8, "bfloat16")
    want, want_lse = attend(torch, mxk, b)
    slot = lambda i, t: torch.tensor([b["slots"][i][128 + t]], device="cuda")  # noqa: E731
    k, v = torch.randn(1, 2, 64, device="cuda"), torch.randn(1, 2, 64, device="cuda")
    v[0, 1, 7] = float("nan")
    mxk.cache_write(b["cache"], k, v, slot(3, 5))
    k[0, 0, 9] = float("nan")
    mxk.cache_write(b["cache"], k, v.nan_to_num(), slot(5, 24))
    out, lse = attend(torch, mxk, b)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[3, 2:, 7] = True
    hit[5, :2] = True
    assert out[hit].isnan().all() and not out[~hit].isnan().any()
    others = [i for i in range(80) if i not in (3, 5)]
    assert torch.equal(out[others], want[others]) and torch.equal(lse[others], want_lse[others])


def test_single_tokens_in_a_padded_batch(torch_cuda, mxk):
    """Most sequences have no tokens; among the others some are long enough for several chunks."""
    torch, g = torch_cuda, np.random.default_rng(17)
    some = [(1, 3 + 211 * i % 1900) for i in range(24)]
    rest = [(0, 0)] * 1500
    b = build(torch, mxk, g, [(0, None, rest), (128, 128, some[:12] + rest), (256, 256, rest[:40] + some[12:])], 8, 2, 64, 16, 8,
              "bfloat16")
    check(torch, b, *attend(torch, mxk, b))
