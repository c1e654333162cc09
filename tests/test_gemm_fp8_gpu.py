"""E4M3 rows with float32 scales and their products on the GPU, against 64 bits."""
import numpy as np
import pytest

from test_cache_gpu import code_values

pytestmark = pytest.mark.gpu


def codes64(torch):
    return torch.from_numpy(code_values(8).astype(np.float64)).cuda()


def scaled(torch, codes, scales, rows):
    """float64 values of codes [n, k] with scales per `rows` rows and 128 columns."""
    n, k = codes.shape
    s = scales.double().repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return codes64(torch)[codes.long()] * s


def nearest(torch, y):
    """Codes of the E4M3 values nearest to y (float64), of two the even one."""
    grid = codes64(torch)[:127]
    a = y.abs().clamp(max=448.0)
    up = torch.bucketize(a, grid).clamp(max=126)
    down = (up - 1).clamp(min=0)
    lo, hi = a - grid[down], grid[up] - a
    return torch.where((lo < hi) | ((lo == hi) & (down % 2 == 0)), down, up) + 128 * torch.signbit(y)


def expected(torch, x, rows):
    """(codes, scales) of x's rows: the definition."""
    n, k = x.shape
    whole = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -n % rows))
    tiles = whole.unflatten(0, (-1, rows)).unflatten(2, (-1, 128))
    scales = (tiles.abs().nan_to_num(nan=0.0, posinf=float("inf")).amax((1, 3)) / 448.0).float().clamp(min=2.0 ** -126)
    codes = nearest(torch, tiles / scales.double()[:, None, :, None])
    return codes.flatten(2, 3).flatten(0, 1)[:n, :k], scales


def some_rows(torch, n, k, dtype, seed):
    """Ordinary values, features far larger than others, zeros, tiny and huge rows."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g)
    x *= torch.where(torch.rand(k, generator=g) < 0.02, 30.0, 1.0)
    x *= torch.exp2(torch.randint(-12, 8, (n, 1), generator=g).float())
    x[torch.rand(n, generator=g) < 0.05] = 0
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("n,k,shift", [(1, 16, 0), (1, 128, 0), (129, 144, 0), (300, 1040, 0), (7, 4096, 0),
                                       (130, 272, 8), (67, 400, 1), (2049, 512, 0)])
def test_codes_are_those_of_the_exact_quotients(torch_cuda, mxk, dtype, block_rows, n, k, shift):
    torch = torch_cuda
    dtype = getattr(torch, dtype)
    wide = torch.zeros(n, k + 24, dtype=dtype, device="cuda")
    x = wide[:, shift:shift + k]
    x.copy_(some_rows(torch, n, k, dtype, n + k))
    blocks = -(-n // block_rows), -(-k // 128)
    values = torch.full((n, k), 0xa5, dtype=torch.uint8, device="cuda")
    scales = torch.full(blocks, 7.0, device="cuda")
    mxk.quantize_fp8(x, values, scales, block_rows=block_rows)
    codes, want = expected(torch, x, block_rows)
    assert torch.equal(scales, want)
    same = values == codes
    # zeros: of either sign
    assert (same | ((values & 127) == 0) & ((codes & 127) == 0)).all()


def test_quotients_next_to_borders(torch_cuda, mxk):
    """Every element of bfloat16's grid below several largest values, whose quotients often
    are the middle between two codes but for the rounding of the scale; float32 elements one
    step beside such middles; tiny blocks."""
    torch = torch_cuda
    mant = torch.arange(128, 256, device="cuda").double() / 128
    rows = []
    for top in (1.0, 1.0546875, 1.3125, 1.5, 1.640625, 1.75, 1.9921875):
        x = torch.cat([mant * 2.0 ** -e for e in range(0, 18)])
        x = torch.where(x > top, x / 2, x)
        x = torch.nn.functional.pad(x, (0, -len(x) % 127)).unflatten(0, (-1, 127))
        rows.append(torch.cat([torch.full_like(x[:, :1], top), x], 1))
    x = torch.cat(rows)
    k = x.shape[1]
    cases = [x.to(torch.bfloat16), (x * 2.0 ** -110).to(torch.bfloat16), (x * 2.0 ** 100).to(torch.bfloat16)]
    s = (x[:, :1] / 448.0).float().double()
    grid = codes64(torch)[:127]
    middle = ((grid[1:] + grid[:-1]) / 2)[torch.arange(k - 1, device="cuda") % 126]
    for step in (-1, 0, 1):  # float32 next to middle * s
        y = torch.cat([x[:, :1], middle * s], 1).float()
        y[:, 1:] = (y[:, 1:].contiguous().view(torch.int32) + step).view(torch.float32)
        cases += [y, y * 2.0 ** -118]
    for y in cases:
        values = torch.empty(y.shape, dtype=torch.uint8, device="cuda")
        scales = torch.empty(len(y), 1, device="cuda")
        mxk.quantize_fp8(y, values, scales)
        codes, want = expected(torch, y, 1)
        assert torch.equal(scales, want)
        assert torch.equal(values.long() & 127, codes & 127)


def test_numbers_that_are_none(torch_cuda, mxk):
    torch = torch_cuda
    x = some_rows(torch, 4, 256, torch.float32, 1)
    x[0] = torch.randn(256, device="cuda")
    x[0, 3], x[1, 130] = float("nan"), float("inf")
    values = torch.empty(4, 256, dtype=torch.uint8, device="cuda")
    scales = torch.empty(4, 2, device="cuda")
    mxk.quantize_fp8(x, values, scales)
    clean = x.clone()
    clean[0, 3] = 0
    codes, want = expected(torch, clean, 1)
    assert torch.equal(scales[[0, 2, 3]], want[[0, 2, 3]]) and scales[1, 1] == float("inf")
    assert (values[0, 3] & 127) == 127 and (values[1, 130] & 127) == 127
    codes[0, 3] = values[0, 3]
    assert torch.equal(values.long()[0] & 127, codes[0] & 127)
    assert ((values[1, 128:] & 127) == 0).sum() == 127


def product_limit(torch, a, b, blocks, dtype, want):
    """How far a sum may be off: a block's 128 products and the blocks' sums, each addition and
    the factor by a step of float32 of the magnitudes' sum, then half a step of the output."""
    mags = a.abs() @ b.abs().T
    half = torch.finfo(dtype).eps / 2
    return (128 + blocks + 2) * 2.0 ** -23 * mags * (1 + half) + half * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)


SIZES = [(1, 1, 16), (1, 128, 128), (3, 130, 144), (64, 256, 1024), (128, 127, 2048), (129, 129, 400), (200, 64, 4096),
         (777, 1003, 1040), (1, 4096, 4096), (17, 1000, 16384), (512, 2304, 640), (2500, 640, 256), (33, 8, 112), (2100, 2561, 400), (4097, 1300, 1040), (300, 16500, 128),
         (2560, 2048, 4096), (2500, 1990, 4112), (2300, 2049, 4096), (600, 6700, 4112), (129, 7100, 144), (200, 7168, 1024), (400, 3600, 656), (128, 9000, 272)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(torch_cuda, mxk, dtype, m, n, k):
    torch = torch_cuda
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, a_scales = expected(torch, torch.randn(m, k, generator=g, device="cuda"), 1)
    b, b_scales = expected(torch, torch.randn(n, k, generator=g, device="cuda") * k ** -0.5, 128)
    a, b = a.to(torch.uint8), b.to(torch.uint8)
    a_scales *= torch.exp2(torch.randint(-3, 4, a_scales.shape, generator=g, device="cuda").float())
    wide = torch.full((m + 2, n + 3), 9.0, dtype=dtype, device="cuda")
    x, w = scaled(torch, a, a_scales, 1), scaled(torch, b, b_scales, 128)
    want = x @ w.T
    limit = product_limit(torch, x, w, -(-k // 128), dtype, want)
    for out in (torch.empty(m, n, dtype=dtype, device="cuda"), wide[1:m + 1, 1:n + 1]):
        mxk.gemm_fp8(a, a_scales, b, b_scales, out)
        assert ((out.double() - want).abs() <= limit).all()
    rest = wide.clone()
    rest[1:m + 1, 1:n + 1] = 9.0
    assert (rest == 9.0).all(), "an element beside the output changed"
    again = torch.empty(m, n, dtype=dtype, device="cuda")
    mxk.gemm_fp8(a.view(torch.float8_e4m3fn), a_scales, b.view(torch.float8_e4m3fn), b_scales, again)
    assert torch.equal(again, wide[1:m + 1, 1:n + 1])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k,shift", [(1, 256, 512, 0), (1, 4096, 4096, 0), (5, 300, 4096, 0), (16, 1000, 4096, 8), (9, 130, 2064, 1),
                                         (16, 20000, 1040, 0), (1, 16, 16, 0), (8, 200, 16384, 0), (17, 128, 512, 0), (64, 1536, 2064, 8), (130, 100, 272, 1),
                                         (1000, 520, 1024, 0), (2500, 2000, 4112, 8)])
def test_layers_are_quantisation_and_product(torch_cuda, mxk, dtype, m, n, k, shift):
    torch = torch_cuda
    dtype = getattr(torch, dtype)
    wide = torch.zeros(m, k + 24, dtype=dtype, device="cuda")
    x = wide[:, shift:shift + k]
    x.copy_(some_rows(torch, m, k, dtype, m))
    b, b_scales = expected(torch, torch.randn(n, k, device="cuda") * k ** -0.5, 128)
    b = b.to(torch.uint8)
    a, a_scales = torch.empty(m, k, dtype=torch.uint8, device="cuda"), torch.empty(m, -(-k // 128), device="cuda")
    mxk.quantize_fp8(x, a, a_scales)
    out, want = (torch.empty(m, n, dtype=dtype, device="cuda") for _ in range(2))
    mxk.gemm_fp8(a, a_scales, b, b_scales, want)
    mxk.linear_fp8(x, b, b_scales, out)
    assert torch.equal(out, want)
    exact = scaled(torch, a, a_scales, 1) @ scaled(torch, b, b_scales, 128).T
    limit = product_limit(torch, scaled(torch, a, a_scales, 1), scaled(torch, b, b_scales, 128), -(-k // 128), dtype, exact)
    assert ((out.double() - exact).abs() <= limit).all()


def test_rows_do_not_touch_each_other(torch_cuda, mxk):
    """NaNs and infinities in a row, and in a weight's row, stay in the outputs that they reach."""
    torch = torch_cuda
    m, n, k = 150, 200, 640
    x = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    b, b_scales = expected(torch, torch.randn(n, k, device="cuda"), 128)
    b = b.to(torch.uint8)
    want, out = (torch.empty(m, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    mxk.linear_fp8(x, b, b_scales, want)
    x[3, 5], x[140, 600] = float("nan"), float("inf")
    b[7, 300] = 127
    mxk.linear_fp8(x, b, b_scales, out)
    hit = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    hit[3], hit[140], hit[:, 7] = True, True, True
    assert torch.equal(out[~hit], want[~hit]) and out[hit].isnan().all()


def test_no_features_give_zeros(torch_cuda, mxk):
    torch = torch_cuda
    wide = torch.full((5, 9), 3.0, device="cuda")
    none = torch.empty(4, 0, dtype=torch.uint8, device="cuda"), torch.empty(4, 0, device="cuda")
    weights = torch.empty(6, 0, dtype=torch.uint8, device="cuda"), torch.empty(1, 0, device="cuda")
    mxk.gemm_fp8(*none, *weights, wide[:4, 1:7])
    assert (wide[:4, 1:7] == 0).all() and (wide[4] == 3).all() and (wide[:, 0] == 3).all() and (wide[:, 7:] == 3).all()


def test_captured_layers_on_another_stream(torch_cuda, mxk):
    """Two graphs of layers, replayed one after the other and again on new rows."""
    torch = torch_cuda
    m, n, k = 40, 384, 1024
    weights = [expected(torch, torch.randn(n, k, device="cuda") * k ** -0.5, 128) for _ in range(2)]
    weights = [(b.to(torch.uint8), s) for b, s in weights]
    x = torch.randn(m, k, device="cuda").half()
    outs = [torch.empty(m, n, dtype=torch.float16, device="cuda") for _ in weights]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for (b, s), out in zip(weights, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            mxk.linear_fp8(x, b, s, out)
            mxk.linear_fp8(x, b, s, out)
    for seed in range(3):
        x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(seed)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (b, s), out in zip(weights, outs):
            want = torch.empty_like(out)
            mxk.linear_fp8(x, b, s, want)
            assert torch.equal(out, want)


def test_large_layers_one_after_the_other(torch_cuda, mxk):
    """Two kernels share a product, beside each other and behind the quantiser: captured, and with
    other rows in every call, whose results go on into the next."""
    torch = torch_cuda
    m, n, k = 2500, 2048, 4112
    first, second = (expected(torch, torch.randn(*size, device="cuda") * size[1] ** -0.5, 128) for size in ((n, k), (k, n)))
    first, second = ((b.to(torch.uint8), s) for b, s in (first, second))
    xs = [torch.randn(m, k, device="cuda").to(torch.bfloat16) for _ in range(4)]
    hidden, out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    want = []
    for x in xs:
        mxk.linear_fp8(x, *first, hidden)
        torch.cuda.synchronize()
        mxk.linear_fp8(hidden, *second, out)
        torch.cuda.synchronize()
        want.append(out.clone())
    got = [torch.empty_like(out) for _ in xs]
    for _ in range(5):
        for x, y in zip(xs, got):
            mxk.linear_fp8(x, *first, hidden)
            mxk.linear_fp8(hidden, *second, y)
    assert all(torch.equal(y, w) for y, w in zip(got, want))
    x = torch.empty_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            mxk.linear_fp8(x, *first, hidden)
            mxk.linear_fp8(hidden, *second, out)
    for i in (0, 1, 2, 3) * 5:
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, want[i])


FIRST = """
import sys
sys.path[:0] = ["mx-kmeans_b200"]
import torch, mxk
m, n, k = {sizes}
x = torch.ones(m, k, device="cuda", dtype=torch.bfloat16)
b, s = torch.full((n, k), 56, dtype=torch.uint8, device="cuda"), torch.full((-(-n // 128), k // 128), 0.5, device="cuda")
out = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    mxk.linear_fp8(x, b, s, out)
graph.replay()
torch.cuda.synchronize()
assert (out == 0.5 * k).all()
"""


@pytest.mark.parametrize("sizes", [(1, 128, 256), (40, 128, 256), (2560, 2048, 128)])
def test_first_call_of_a_process_may_be_captured(torch_cuda, mxk, sizes):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.format(sizes=sizes)], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_offsets_past_32_bits(torch_cuda, mxk):
    """More than 2^32 elements of rows and of quantised rows; the last rows' products."""
    torch = torch_cuda
    m, n, k = (1 << 18) + 300, 48, 16384
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, k, device="cuda")
    b, b_scales = expected(torch, torch.randn(n, k, device="cuda") * k ** -0.5, 128)
    b = b.to(torch.uint8)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    mxk.linear_fp8(x, b, b_scales, out)
    # against 64 bits and not against a call of 300 rows: that splits the 16,384 features over
    # eight CTAs, adds in another order, and may round to the other neighbour
    a, w = (scaled(torch, v.to(torch.uint8), s, rows) for v, s, rows in ((*expected(torch, x[-300:], 1), 1), (b, b_scales, 128)))
    want = a @ w.T
    limit = product_limit(torch, a, w, k // 128, torch.bfloat16, want)
    assert ((out[-300:].double() - want).abs() <= limit).all() and (out[:-300] == 0).all()
    del x, out
    # an output whose rows lie far apart
    wide = torch.zeros(2100, (1 << 21) + 16, dtype=torch.bfloat16, device="cuda")
    a, a_scales = expected(torch, torch.randn(2100, 256, device="cuda"), 1)
    c, c_scales = expected(torch, torch.randn(2400, 256, device="cuda"), 128)
    near = torch.empty(2100, 2400, dtype=torch.bfloat16, device="cuda")
    a, c = a.to(torch.uint8), c.to(torch.uint8)
    mxk.gemm_fp8(a, a_scales, c, c_scales, near)
    mxk.gemm_fp8(a, a_scales, c, c_scales, wide[:, -2400:])
    assert torch.equal(wide[:, -2400:], near) and (wide[:, -2500:-2400] == 0).all()


def test_two_streams_at_once(torch_cuda, mxk):
    """Layers on two streams, each with its own workspace."""
    torch = torch_cuda
    weights = [expected(torch, torch.randn(512, 1024, device="cuda"), 128) for _ in range(2)]
    weights = [(b.to(torch.uint8), s) for b, s in weights]
    xs = [torch.randn(200, 1024, device="cuda").half() for _ in range(2)]
    want = [torch.empty(200, 512, dtype=torch.float16, device="cuda") for _ in range(2)]
    for x, w, out in zip(xs, weights, want):
        mxk.linear_fp8(x, *w, out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(want[0]) for _ in range(20)] for _ in range(2)]
    for i in range(20):
        for j in range(2):
            mxk.linear_fp8(xs[j], *weights[j], got[j][i], stream=streams[j])
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[j]) for j in range(2) for out in got[j])


def test_bad_tensors_are_refused(torch_cuda, mxk):
    torch = torch_cuda
    m, n, k = 4, 200, 256
    x = torch.randn(m, k, device="cuda")
    a, a_scales = torch.empty(m, k, dtype=torch.uint8, device="cuda"), torch.empty(m, 2, device="cuda")
    b, b_scales = torch.empty(n, k, dtype=torch.uint8, device="cuda"), torch.empty(2, 2, device="cuda")
    out = torch.zeros(m, n, device="cuda")
    good = dict(a=a, a_scales=a_scales, b=b, b_scales=b_scales, out=out)
    for bad in (dict(a=a[:3]), dict(a=a[:, :240]), dict(a=a.float()), dict(a=a.cpu()), dict(a_scales=a_scales[:, :1]),
                dict(a_scales=a_scales.double()), dict(b=b[:, :128]), dict(b=b.t()), dict(b_scales=b_scales[:1]),
                dict(out=out.double()), dict(out=out.t()), dict(out=out[0]), dict(out=out[:1].expand(m, n)),
                dict(out=out.cpu())):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.gemm_fp8(**{**good, **bad})
    good = dict(x=x, b=b, b_scales=b_scales, out=out)
    for bad in (dict(x=x[:3]), dict(x=x.half()), dict(x=x.t()), dict(x=x.cpu()), dict(b=b[:100]), dict(out=out.half()),
                dict(out=out[:, ::2])):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.linear_fp8(**{**good, **bad})
    good = dict(x=x, values=a, scales=a_scales)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(values=a[:, :128]), dict(scales=a_scales[:3]),
                dict(block_rows=128), dict(block_rows=2), dict(x=x[:, :250], values=a[:, :250].contiguous())):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.quantize_fp8(**{**good, **bad})
    torch.cuda.synchronize()
    assert (out == 0).all()
