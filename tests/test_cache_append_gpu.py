"""Rotated appending to the paged MX cache on the GPU, against the rotation and the
quantisation in 64 bits."""
import numpy as np
import pytest

from test_cache_gpu import code_values, decode

pytestmark = pytest.mark.gpu

MOST = {8: 448.0, 6: 7.5, 4: 6.0}


def rotated(x, cos_sin, interleaved):
    """x [tokens, heads, d] float64, cos_sin [tokens, r] float64."""
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[:, None, :half], cos_sin[:, None, half:]
    y = x.copy()
    i = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    j = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def mx_values(x, bits):
    """(values, scale bytes) of float64 rows on their format's grid."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    scale = np.exp2(np.ceil(np.log2(np.where(amax > 0, amax, MOST[bits]) / MOST[bits])))
    scale = np.where(scale * MOST[bits] < amax, scale * 2, scale)
    scale = np.where((amax > 0) & (scale * MOST[bits] / 2 >= amax), scale / 2, scale)
    grid = code_values(bits)[:2 ** (bits - 1)].astype(np.float64)
    grid = grid[np.isfinite(grid)]
    y = np.abs(b / scale)
    up = np.minimum(np.searchsorted(grid, y), len(grid) - 1)
    down = np.maximum(up - 1, 0)
    lo, hi = y - grid[down], grid[up] - y
    pick = np.where((lo < hi) | ((lo == hi) & (down % 2 == 0)), down, up)
    return (np.copysign(grid[pick], b) * scale).reshape(x.shape), (np.log2(scale[..., 0]) + 127).astype(np.int64)


def table(torch, rows, rot):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda()


def make(torch, mxk, n, hq, hk, d, page, bits, dtype, rot, seed, fused=False, rows=5000):
    g = torch.Generator().manual_seed(seed)
    pages = n // page + 3
    cache = mxk.PagedCache.empty(pages, page, hk, d, bits)
    for t in (cache.k_values, cache.k_scales, cache.v_values, cache.v_scales):
        t.fill_(0xa5)
    both = torch.randn(n, hq + 2 * hk, d, generator=g) * torch.exp2(torch.randint(-6, 7, (n, hq + 2 * hk, 1), generator=g))
    both = both.to(getattr(torch, dtype)).cuda()
    q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    if not fused:
        q, k, v = q.clone(), k.clone(), v.clone()
    slots = torch.randperm(pages * page, generator=g)[:n].cuda()
    positions = torch.randint(0, rows, (n,), generator=g).cuda()
    return cache, q, k, v, slots, positions, table(torch, rows, rot)


def at_slots(cache, side, slots):
    """(values, scales) of the slots' rows, numpy."""
    out = []
    for t in (getattr(cache, side + "_values"), getattr(cache, side + "_scales")):
        t = t.cpu().numpy().transpose(0, 2, 1, 3)
        out.append(t.reshape(-1, *t.shape[2:])[slots.cpu().numpy()])
    return out


def check(torch, cache, q, k, v, slots, positions, cos_sin, q_out, interleaved, q_in=None):
    angles = cos_sin[positions].double().cpu().numpy()
    for side, x in (("k", k), ("v", v)):
        x = x.double().cpu().numpy()
        want, scales = mx_values(rotated(x, angles, interleaved) if side == "k" else x, cache.bits)
        got_values, got_scales = at_slots(cache, side, slots)
        assert np.array_equal(got_scales, scales)
        assert np.array_equal(decode(got_values, got_scales, cache.bits), want.astype(np.float32))
    if q_out is not None:
        x = (q if q_in is None else q_in).double().cpu().numpy()
        want = rotated(x, angles, interleaved)
        # Half a step of the type, and three roundings of float32 of the two products.  (Below
        # the normal range a step is 2^-24 in f16: half of it.)
        products = rotated(np.abs(x), np.abs(angles) * np.r_[[1.0] * (angles.shape[1] // 2),
                                                             [-1.0] * (angles.shape[1] // 2)], interleaved)
        products = np.maximum(products, rotated(np.abs(x), np.abs(angles), interleaved))
        step = torch.finfo(q_out.dtype).eps / 2
        limit = (step * np.abs(want) + 3 * 2.0 ** -24 * products) * 1.01 + 2.0 ** -25 * (q_out.dtype == torch.float16)
        assert (np.abs(q_out.double().cpu().numpy() - want) <= limit + 1e-40).all()


SHAPES = [(1, 1, 1, 32, 16, 32), (3, 4, 2, 64, 48, 64), (130, 6, 3, 96, 16, 64), (77, 6, 3, 128, 64, 128),
          (33, 2, 1, 512, 32, 80), (9, 5, 5, 128, 16, 16), (2100, 9, 1, 64, 128, 48), (8, 32, 8, 128, 64, 96)]


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,hq,hk,d,page,rot", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_are_those_of_the_exact_rotation(torch_cuda, mxk, bits, dtype, n, hq, hk, d, page, rot, interleaved):
    torch = torch_cuda
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, page, bits, dtype, rot, n + d + rot,
                                                     fused=n % 2 == 0)
    q_out = torch.empty(n, hq, d, dtype=q.dtype, device="cuda")
    before = q.clone()
    mxk.cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=q_out, interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(q, before)
    check(torch, cache, q, k, v, slots, positions, cos_sin, q_out, interleaved)
    rest = np.setdiff1d(np.arange(cache.pages * page), slots.cpu().numpy())
    for side in "kv":
        for t in at_slots(cache, side, torch.from_numpy(rest)):
            assert (t == 0xa5).all(), "a slot nobody named changed"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,rot,shift", [("bfloat16", 128, 0), ("bfloat16", 48, 0), ("float32", 64, 0),
                                             ("float16", 128, 3), ("float16", 80, 8), ("float32", 16, 1)])
def test_queries_in_place_and_odd_strides(torch_cuda, mxk, dtype, rot, shift, interleaved):
    """Rows that begin `shift` elements after a 128-byte boundary, token strides that are no
    multiple of anything, heads in reverse order."""
    torch = torch_cuda
    n, hq, hk, d = 41, 6, 2, 128
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, 16, 8, dtype, rot, 5)
    wide = torch.zeros(n, (hq + 2 * hk) * d + shift, dtype=q.dtype, device="cuda")
    flat = wide[:, shift:].unflatten(1, (hq + 2 * hk, d))
    flat[:, :hq], flat[:, hq:hq + hk], flat[:, hq + hk:] = q, k, v
    before = wide.clone()
    mxk.cache_append(cache, flat[:, :hq], flat[:, hq:hq + hk], flat[:, hq + hk:], positions, cos_sin, slots,
                     interleaved=interleaved)
    check(torch, cache, None, k, v, slots, positions, cos_sin, flat[:, :hq], interleaved, q_in=q)
    assert torch.equal(wide[:, :shift], before[:, :shift]) and torch.equal(flat[:, hq:], before[:, shift:].unflatten(1, (-1, d))[:, hq:])


def test_padding_and_unknown_positions(torch_cuda, mxk):
    torch = torch_cuda
    n, hq, hk, d, rows = 12, 4, 2, 64, 100
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, 16, 8, "bfloat16", 64, 1, rows=rows)
    slots[[1, 4]] = torch.tensor([-1, cache.pages * 16], device="cuda")
    slots[5] = 1 << 40
    positions[[2, 3]] = torch.tensor([-1, rows], device="cuda")
    positions[6] = -(1 << 45)
    q_out = torch.full_like(q, 7.0)
    mxk.cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=q_out)
    kept = torch.tensor([0, 7, 8, 9, 10, 11], device="cuda")
    check(torch, cache, q[kept], k[kept], v[kept], slots[kept], positions[kept], cos_sin, q_out[kept], False)
    moved = torch.tensor([1, 4, 5], device="cuda")  # not kept, but their queries are there
    angles = cos_sin[positions[moved]].double().cpu().numpy()
    want = rotated(q[moved].double().cpu().numpy(), angles, False)
    assert np.abs(q_out[moved].double().cpu().numpy() - want).max() <= 2.0 ** -8 * np.abs(want).max()
    assert (q_out[[2, 3, 6]] == 0).all()
    rest = np.setdiff1d(np.arange(cache.pages * 16), slots[kept].cpu().numpy())
    assert all((t == 0xa5).all() for t in at_slots(cache, "k", torch.from_numpy(rest)))


@pytest.mark.parametrize("bits", [8, 6, 4])
def test_values_next_to_borders(torch_cuda, mxk, bits):
    """Keys whose exact rotation lies a hair beside the middle between two codes, or beside
    the largest magnitude of a scale: sums that float32 rounds onto the border."""
    torch = torch_cuda
    n, hk, d = 64, 1, 64
    cache, _, k, v, slots, _, _ = make(torch, mxk, n, 1, hk, d, 16, bits, "float32", 64, 2)
    g = np.random.default_rng(3)
    grid = code_values(bits)[:2 ** (bits - 1)].astype(np.float64)
    grid = grid[np.isfinite(grid)]
    middles = (grid[1:] + grid[:-1]) / 2
    x = np.zeros((n, hk, d), np.float32)
    x[..., :32] = g.choice(np.r_[middles, MOST[bits]], (n, hk, 32))
    x[..., 0] = MOST[bits]
    x[..., 32:] = 1.0
    cos_sin = torch.zeros(n, 64)
    cos_sin[:, :32] = 1.0
    # y_i = x_i +- 2^-30 or so: below half a step of float32
    cos_sin[:, 32:] = torch.from_numpy(g.choice([2.0 ** -30, -2.0 ** -30, 2.0 ** -40, 0.0], (n, 32))).float()
    k = torch.from_numpy(x).cuda()
    cos_sin, positions = cos_sin.cuda(), torch.arange(n, device="cuda")
    mxk.cache_append(cache, None, k, v, positions, cos_sin, slots)
    check(torch, cache, None, k, v, slots, positions, cos_sin, None, False)


def test_infinities_and_nans_stay_in_their_block(torch_cuda, mxk):
    torch = torch_cuda
    n, hk, d = 6, 2, 128
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, 2, hk, d, 16, 8, "bfloat16", 64, 4)
    clean = mxk.PagedCache.empty(cache.pages, 16, hk, d, 8)
    mxk.cache_append(clean, None, k, v, positions, cos_sin, slots)
    k[1, 0, 5] = float("nan")
    k[2, 1, 40] = float("inf")
    mxk.cache_append(cache, q, k, v, positions, cos_sin, slots)
    got, got_s = at_slots(cache, "k", slots)
    want, want_s = at_slots(clean, "k", slots)
    got, want = (decode(a, b, 8).reshape(n, hk, 4, 32) for a, b in ((got, got_s), (want, want_s)))
    assert np.isnan(got[1, 0, 0, 5]) and np.isnan(got[1, 0, 1, 5])  # both ends of the pair
    touched = np.zeros((n, hk, 4), bool)
    touched[1, 0, :2] = touched[2, 1, :2] = True
    assert np.array_equal(got[~touched], want[~touched])
    assert np.isfinite(got[0]).all() and np.isfinite(got[3:]).all()


def test_captured_on_another_stream(torch_cuda, mxk):
    torch = torch_cuda
    n, hq, hk, d = 300, 4, 2, 64
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, 32, 6, "float16", 64, 6)
    q_out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mxk.cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=q_out)
    for seed in (1, 2):
        fresh = make(torch, mxk, n, hq, hk, d, 32, 6, "float16", 64, seed)
        for a, b in zip((q, k, v, slots, positions), fresh[1:6]):
            a.copy_(b)
        graph.replay()
        check(torch, cache, q, k, v, slots, positions, cos_sin, q_out, False)


def test_slots_past_2_to_the_31(torch_cuda, mxk):
    """Places whose byte offsets need 64 bits (about 9 GB of values a side)."""
    torch = torch_cuda
    hk, d, page = 1, 32, 16
    pages = (1 << 28) // page + 5
    cache = mxk.PagedCache.empty(pages, page, hk, d, 8)
    k, v = (torch.randn(4, hk, d, device="cuda") for _ in range(2))
    slots = torch.tensor([0, (1 << 27) + 3, (1 << 28) - 1, pages * page - 1], device="cuda")
    positions = torch.arange(4, device="cuda")
    mxk.cache_append(cache, None, k, v, positions, table(torch, 10, 32), slots)
    k_back, v_back = torch.empty_like(k), torch.empty_like(v)
    mxk.cache_read(cache, slots, k_back, v_back)
    angles = table(torch, 10, 32)[positions].double().cpu().numpy()
    want, _ = mx_values(rotated(k.double().cpu().numpy(), angles, False), 8)
    assert np.array_equal(k_back.cpu().numpy(), want.astype(np.float32))


def test_bad_tensors_are_refused(torch_cuda, mxk):
    torch = torch_cuda
    n, hq, hk, d = 5, 4, 2, 64
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, 16, 8, "float16", 64, 7)
    good = dict(q=q, k=k, v=v, positions=positions, cos_sin=cos_sin, slots=slots)
    for bad in (dict(q=q.float()), dict(q=q[:4]), dict(q=q[0]), dict(k=k[:, :1]), dict(v=v.bfloat16()),
                dict(k=k.cpu()), dict(positions=positions.int()), dict(positions=positions[:4]),
                dict(slots=slots.int()), dict(cos_sin=cos_sin.double()), dict(cos_sin=cos_sin[:, :40]),
                dict(cos_sin=cos_sin[0]), dict(cos_sin=cos_sin.cpu()), dict(q_out=q.float()),
                dict(q=None, q_out=q.clone()), dict(q=q.transpose(1, 2)), dict(cos_sin=cos_sin[:, :0])):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.cache_append(cache, **{**good, **bad})
    torch.cuda.synchronize()
    assert all((t == 0xa5).all() for t in (cache.k_values, cache.v_values))


@pytest.mark.parametrize("bits,dtype", [(8, "bfloat16"), (6, "float32"), (4, "float16")])
@pytest.mark.parametrize("n,hq,hk,d,page,rot", [(8200, 7, 3, 96, 16, 64), (6001, 11, 9, 128, 32, 128), (12003, 13, 7, 128, 16, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens_are_those_of_a_few_at_a_time(torch_cuda, mxk, bits, dtype, n, hq, hk, d, page, rot, interleaved):
    """With many a thread goes through several heads of its token, the last ones through fewer."""
    torch = torch_cuda
    cache, q, k, v, slots, positions, cos_sin = make(torch, mxk, n, hq, hk, d, page, bits, dtype, rot, n, fused=True)
    other = mxk.PagedCache.empty(cache.pages, page, hk, d, bits)
    buffers = ("k_values", "k_scales", "v_values", "v_scales")
    for name in buffers:
        getattr(other, name).copy_(getattr(cache, name))
    out, want = (torch.empty(n, hq, d, dtype=q.dtype, device="cuda") for _ in range(2))
    mxk.cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=out, interleaved=interleaved)
    for i in range(0, n, 300):
        part = slice(i, i + 300)
        mxk.cache_append(other, q[part], k[part], v[part], positions[part], cos_sin, slots[part], q_out=want[part],
                         interleaved=interleaved)
    assert torch.equal(out, want)
    for name in buffers:
        assert torch.equal(getattr(cache, name), getattr(other, name))
