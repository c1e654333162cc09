"""Paged MX cache on the GPU: the written bytes are those of quantize_rows, what is
read back is what the bytes stand for."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FORMATS = {8: (3, 7), 6: (3, 1), 4: (1, 1)}


def code_values(bits):
    """float32 value of every element code (8 bits: the two NaN codes too)."""
    mant, bias = FORMATS[bits]
    out = np.empty(2 ** bits, np.float32)
    for c in range(2 ** bits):
        e, m = divmod(c % 2 ** (bits - 1), 2 ** mant)
        v = m * 2.0 ** (1 - bias - mant) if e == 0 else (1 + m / 2 ** mant) * 2.0 ** (e - bias)
        out[c] = -v if c >= 2 ** (bits - 1) else v
    if bits == 8:
        out[[127, 255]] = np.nan
    return out


def unpack(values, bits):
    """Codes of packed rows (numpy uint8, last axis)."""
    v = values.astype(np.int64)
    if bits == 8:
        return v
    if bits == 4:
        return np.stack([v & 15, v >> 4], -1).reshape(*v.shape[:-1], 2 * v.shape[-1])
    t = v.reshape(*v.shape[:-1], v.shape[-1] // 3, 3)
    w = t[..., 0] | (t[..., 1] << 8) | (t[..., 2] << 16)
    return np.stack([(w >> (6 * i)) & 63 for i in range(4)], -1).reshape(*v.shape[:-1], v.shape[-1] // 3 * 4)


def decode(values, scales, bits):
    """float32 rows a packed cache stands for."""
    x = code_values(bits)[unpack(values, bits)]
    with np.errstate(over="ignore"):
        f = np.ldexp(np.float32(1), scales.astype(np.int32) - 127)
        return (x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32) * f[..., None]).astype(np.float32).reshape(x.shape)


def some_rows(g, n, h, d):
    """Ordinary rows with blocks of zeros, tiny, huge and one-sided values among them."""
    x = g.standard_normal((n, h, d)).astype(np.float32)
    x *= np.ldexp(1.0, g.integers(-12, 12, (n, h, 1))).astype(np.float32)
    x[g.random((n, h)) < 0.1] = 0
    x[0, 0, :32] = 0
    x[0, 0, 5] = 448.0  # exactly the largest magnitude of the format
    return x


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,h,d,page", [(1, 1, 32, 16), (3, 2, 64, 48), (130, 5, 96, 16), (77, 3, 128, 64),
                                        (33, 1, 512, 32)])
def test_written_bytes_are_quantize_rows(torch_cuda, mxk, orc, bits, dtype, n, h, d, page):
    torch = torch_cuda
    g = np.random.default_rng(n + d + bits)
    pages = n // page + 4
    cache = mxk.PagedCache.empty(pages, page, h, d, bits)
    for t in (cache.k_values, cache.k_scales, cache.v_values, cache.v_scales):
        t.fill_(0xa5)
    k, v = (torch.from_numpy(some_rows(g, n, h, d)).cuda().to(getattr(torch, dtype)) for _ in range(2))
    slots = torch.from_numpy(g.permutation(pages * page)[:n]).cuda()
    mxk.cache_write(cache, k, v, slots)
    torch.cuda.synchronize()
    s = slots.cpu().numpy()
    for x, values, scales in ((k, cache.k_values, cache.k_scales), (v, cache.v_values, cache.v_scales)):
        ov, os_, _ = orc.quantize_rows(bits, x.float().cpu().numpy().reshape(n * h, d))
        # [pages, h, page, ...] -> [pages * page, h, ...]
        got_v = values.cpu().numpy().transpose(0, 2, 1, 3).reshape(pages * page, h, -1)
        got_s = scales.cpu().numpy().transpose(0, 2, 1, 3).reshape(pages * page, h, -1)
        assert np.array_equal(got_v[s], np.asarray(ov).reshape(n, h, -1))
        assert np.array_equal(got_s[s], np.asarray(os_).reshape(n, h, -1))
        rest = np.setdiff1d(np.arange(pages * page), s)
        assert (got_v[rest] == 0xa5).all() and (got_s[rest] == 0xa5).all(), "a slot nobody named changed"


@pytest.mark.parametrize("bits", [8, 6, 4])
def test_special_values_as_quantize_rows(torch_cuda, mxk, bits):
    torch = torch_cuda
    x = torch.zeros(12, 1, 64)
    x[0, 0, 3] = float("nan")
    x[1, 0, 3], x[1, 0, 4] = float("inf"), 2.0
    x[2, 0, 40], x[2, 0, 41] = -float("inf"), -float("nan")
    x[3] = 3.4e38
    x[4] = 1e-45
    x[5] = -1.2e-38
    x[6, 0, :32] = torch.linspace(-7.5, 7.5, 32)
    x[7] = -0.0
    x[8, 0, 0], x[8, 0, 1] = 448.0 * 2 ** 3 * (1 + 2 ** -23), 1.0
    x[9, 0, 0], x[9, 0, 1] = 6.0, 0.25
    x[10] = torch.tensor([float("nan"), 1.0]).repeat(32)
    x[11] = torch.arange(64) * 2.0 ** -140
    x = x.cuda()
    cache = mxk.PagedCache.empty(1, 16, 1, 64, bits)
    mxk.cache_write(cache, x, x, torch.arange(12, device="cuda"))
    values = torch.empty(12 * 64 * bits // 8, dtype=torch.uint8, device="cuda")
    scales = torch.empty(12 * 2, dtype=torch.uint8, device="cuda")
    mxk.quantize_rows(bits, x.view(12, 64), values, scales)
    torch.cuda.synchronize()
    for t in (cache.k_values, cache.v_values):
        assert torch.equal(t.view(16, -1)[:12].flatten(), values)
    for t in (cache.k_scales, cache.v_scales):
        assert torch.equal(t.view(16, -1)[:12].flatten(), scales)


def test_slots_outside_the_cache(torch_cuda, mxk):
    torch = torch_cuda
    cache = mxk.PagedCache.empty(2, 16, 2, 64, 8)
    x = torch.randn(6, 2, 64, device="cuda")
    slots = torch.tensor([-1, 31, 32, 5, -2 ** 62, 2 ** 62], device="cuda")
    mxk.cache_write(cache, x, x, slots)
    k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    mxk.cache_read(cache, slots, k, v)
    torch.cuda.synchronize()
    assert torch.equal(k, v)
    for i in (0, 2, 4, 5):
        assert (k[i] == 0).all()
    for i in (1, 3):  # 8-bit elements: within half a unit in the fourth bit, of the block's scale at the low end
        assert ((k[i] - x[i]).abs() <= x[i].abs() * 2 ** -4 + x[i].abs().max() * 2 ** -15).all()
    kept = torch.nonzero(cache.k_scales.transpose(1, 2).reshape(32, -1).sum(1)).flatten().tolist()
    assert kept == [5, 31]


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_read_every_code_and_scale(torch_cuda, mxk, bits, dtype):
    """All element codes at all scales (0 .. 254), rounded once to the type."""
    torch = torch_cuda
    d = 96
    rows = 255 * 3
    g = np.random.default_rng(bits)
    page, pages = 16, (rows + 15) // 16
    packed = g.integers(0, 256, (pages, 1, page, d * bits // 8), dtype=np.uint8)
    flat = packed.reshape(-1)
    flat[:256 * 32] = np.tile(np.arange(256, dtype=np.uint8), 32)
    scales = (np.arange(pages * page * 3) % 255).astype(np.uint8).reshape(pages, 1, page, 3)
    vs = scales[::-1].copy()
    cache = mxk.PagedCache(*(torch.from_numpy(a).cuda() for a in (packed, scales, packed, vs)), bits)
    slots = torch.arange(pages * page, device="cuda")
    out = [torch.empty(pages * page, 1, d, dtype=getattr(torch, dtype), device="cuda") for _ in range(2)]
    mxk.cache_read(cache, slots, *out)
    torch.cuda.synchronize()
    for o, s in zip(out, (scales, vs)):
        want = torch.from_numpy(decode(packed, s, bits).reshape(pages * page, 1, d)).to(o.dtype)
        got = o.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (8, 8), (1, 0), (3, 1)])
def test_strides_and_alignment(torch_cuda, mxk, bits, dtype, pad, shift):
    """Slices of wider tensors, element-aligned ones too, give what contiguous rows give."""
    torch = torch_cuda
    n, h, d = 19, 3, 64
    wide = torch.randn(n, h * (d + pad) + shift, device="cuda").to(getattr(torch, dtype))
    k = wide[:, shift:].unflatten(1, (h, d + pad))[:, :, :d]
    v = torch.randn(h, n, d + pad, device="cuda").to(k.dtype)[:, :, pad:].transpose(0, 1)
    slots = torch.randperm(48, device="cuda")[:n]
    a, b = (mxk.PagedCache.empty(3, 16, h, d, bits) for _ in range(2))
    mxk.cache_write(a, k, v, slots)
    mxk.cache_write(b, k.contiguous(), v.contiguous(), slots)
    for x, y in ((a.k_values, b.k_values), (a.v_values, b.v_values), (a.k_scales, b.k_scales), (a.v_scales, b.v_scales)):
        assert torch.equal(x, y)
    plain = [torch.empty(n, h, d, dtype=k.dtype, device="cuda") for _ in range(2)]
    mxk.cache_read(b, slots, *plain)
    wide_out = torch.full((n, h * (d + pad) + shift), 9.0, dtype=k.dtype, device="cuda")
    ko = wide_out[:, shift:].unflatten(1, (h, d + pad))[:, :, :d]
    vo = torch.empty(h, n, d + pad, dtype=k.dtype, device="cuda")[:, :, pad:].transpose(0, 1)
    mxk.cache_read(b, slots, ko, vo)
    torch.cuda.synchronize()
    assert torch.equal(ko, plain[0]) and torch.equal(vo, plain[1])
    untouched = wide_out.clone()
    untouched[:, shift:].unflatten(1, (h, d + pad))[:, :, :d] = 9.0
    assert (untouched == 9.0).all(), "the gaps between the rows were written"


def test_broadcast_rows_and_side_stream(torch_cuda, mxk):
    """A stride of zero (one head's rows for all) on a stream of the caller's."""
    torch = torch_cuda
    one = torch.randn(40, 1, 128, device="cuda")
    k = one.expand(40, 4, 128)
    cache = mxk.PagedCache.empty(4, 16, 4, 128, 8)
    slots = torch.arange(40, device="cuda") + 7
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty(40, 4, 128, device="cuda")
    out2 = torch.empty_like(out)
    mxk.cache_write(cache, k, k, slots, stream=side)
    mxk.cache_read(cache, slots, out, out2, stream=side)
    side.synchronize()
    assert torch.equal(out, out2)
    assert all(torch.equal(out[:, 0], out[:, i]) for i in range(4))


def test_offsets_past_32_bits(torch_cuda, mxk):
    """A cache whose buffers are larger than 2^31 bytes; its last slots."""
    torch = torch_cuda
    pages, page, h, d = 2200, 128, 64, 128
    cache = mxk.PagedCache.empty(pages, page, h, d, 8)
    assert cache.k_values.numel() > 2 ** 31
    slots = torch.tensor([pages * page - 1, pages * page - 130, 3], device="cuda")
    k, v = (torch.randn(3, h, d, device="cuda") for _ in range(2))
    mxk.cache_write(cache, k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    mxk.cache_read(cache, slots, ko, vo)
    small = mxk.PagedCache.empty(1, 16, h, d, 8)
    near = torch.tensor([0, 1, 2], device="cuda")
    mxk.cache_write(small, k, v, near)
    ks, vs = torch.empty_like(k), torch.empty_like(v)
    mxk.cache_read(small, near, ks, vs)
    torch.cuda.synchronize()
    assert torch.equal(ko, ks) and torch.equal(vo, vs)
    assert torch.equal(cache.k_values[-1, :, -1], small.k_values[0, :, 0])
