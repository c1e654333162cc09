"""ctypes binding of libmxkmeans.so, the B200 MX-KMeans library (C ABI: include/mxk.h).

The low-level functions take device pointers (ints) exactly as the C ABI does;
the helpers take torch CUDA tensors and pass their data pointers (torch is only
used for device memory and streams here).  Loading fails loudly if the shared
library has not been built -- there is no fallback implementation.
"""
import ctypes
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmxkmeans.so")

OK, ERR_INVALID, ERR_CUDA, ERR_UNSUPPORTED, ERR_NONFINITE, ERR_TIMEOUT, ERR_COMM = range(7)


class MxkError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"mxk status {status}: {message}")
        self.status = status
        self.message = message


class MxkInvalidArgument(MxkError, ValueError):
    pass


class Options(ctypes.Structure):
    """mxk_options; defaults of the reference's KMeansOptions (include/kmeans.cuh:11-16)."""

    _fields_ = [("max_iterations", ctypes.c_int), ("fp32_iterations", ctypes.c_int),
                ("tolerance", ctypes.c_float), ("verbose", ctypes.c_int)]

    def __init__(self, max_iterations=300, fp32_iterations=0, tolerance=1e-4, verbose=False):
        super().__init__(max_iterations, fp32_iterations, tolerance, int(bool(verbose)))


class Trace(ctypes.Structure):
    """mxk_trace: device buffers the next Lloyd call fills per iteration."""

    _fields_ = [("centroids", ctypes.c_void_p), ("labels", ctypes.c_void_p), ("group_sizes", ctypes.c_void_p),
                ("max_iterations", ctypes.c_int)]


class KernelStat(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 48), ("launches", ctypes.c_uint64), ("total_ms", ctypes.c_double)]


F32, F16, BF16 = range(3)  # mxk_dtype


class Cache(ctypes.Structure):
    """mxk_cache: sizes and device pointers of a paged MX cache."""

    _fields_ = [("bits", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("page_size", ctypes.c_int), ("pages", ctypes.c_int64), ("k_values", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_values", ctypes.c_void_p), ("v_scales", ctypes.c_void_p)]


class Rows(ctypes.Structure):
    """mxk_rows: rows of tokens x heads x features with strides in elements."""

    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class Append(ctypes.Structure):
    """mxk_append: the arguments of mxk_cache_append."""

    _fields_ = [("dtype", ctypes.c_int), ("heads", ctypes.c_int), ("tokens", ctypes.c_int64), ("q", Rows),
                ("q_out", Rows), ("k", Rows), ("v", Rows), ("slots", ctypes.c_void_p), ("positions", ctypes.c_void_p),
                ("cos_sin", ctypes.c_void_p), ("table_rows", ctypes.c_int64), ("rot_dim", ctypes.c_int),
                ("interleaved", ctypes.c_int)]


class Attention(ctypes.Structure):
    """mxk_attention: the arguments of mxk_cache_attention."""

    _fields_ = [("dtype", ctypes.c_int), ("heads", ctypes.c_int), ("tokens", ctypes.c_int64),
                ("seqs", ctypes.c_int), ("max_q", ctypes.c_int), ("max_kv", ctypes.c_int64), ("q", Rows),
                ("cu_q", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("page_table_stride", ctypes.c_int64),
                ("kv_lens", ctypes.c_void_p), ("scale", ctypes.c_float), ("causal", ctypes.c_int),
                ("window", ctypes.c_int64), ("out", Rows), ("lse", ctypes.c_void_p)]


class Prefixes(ctypes.Structure):
    """mxk_prefixes: the groups of sequences of mxk_cache_attention_shared."""

    _fields_ = [("groups", ctypes.c_int), ("cu_groups", ctypes.c_void_p), ("prefix_lens", ctypes.c_void_p),
                ("max_prefix", ctypes.c_int64)]


_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I = ctypes.c_int
_F = ctypes.c_float

SIGNATURES = {
    "mxk_version": ([], _I),
    "mxk_last_error": ([], ctypes.c_char_p),
    "mxk_launch_count": ([], ctypes.c_uint64),
    "mxk_compute_l2_norm": ([_I64, _I, _P, _P, _P], _I),
    "mxk_quantize_rows": ([_I, _I64, _I, _P, _P, _P, _P, _P, _P], _I),
    "mxk_precompute_point_bounds": ([_I64, _I, _P, _P, _P, _P], _I),
    "mxk_assign_precisions": ([_I64, _I, _P, _P, _F, _F, _P, _P], _I),
    "mxk_check_mxfp8_scale_codec": ([_P, _P], _I),
    "mxk_check_wait_timeout": ([ctypes.c_longlong, _P, _P], _I),
    "mxk_release_workspace": ([], _I),
    "mxk_gemm_tiles_multiplied": ([ctypes.POINTER(ctypes.c_ulonglong), _I], _I),
    "mxk_gemm_rows_processed": ([ctypes.POINTER(ctypes.c_ulonglong), _I], _I),
    "mxk_init_farthest": ([_I64, _I, _I, _P, _P, _P], _I),
    "mxk_init_kmeanspp": ([_I64, _I, _I, _P, _P, ctypes.c_uint32, _P], _I),
    "mxk_gemm_mx": ([_I, _I64, _I64, _I, _P, _P, _P, _P, _P, _P], _I),
    "mxk_gemm_fp32": ([_I64, _I64, _I, _P, _P, _P, _P], _I),
    "mxk_assign_clusters": ([_I64, _I, _P, _P, _P, _P, _P, _P, _P], _I),
    "mxk_update_centroids": ([_I64, _I, _I, _P, _P, _P, _P, _P, _P], _I),
    "mxk_centroid_shift": ([_I64, _P, _P, _P, _P, _P], _I),
    "mxk_centroid_shift_noalloc": ([_I64, _P, _P, _P, _P, _P], _I),
    "mxk_assign_mx_fused": ([_I, _I64, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P], _I),
    "mxk_assign_f32_fused": ([_I64, _I, _I, _P, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _P], _I),
    "mxk_kmeans_mixed": ([_I64, _I, _I, _P, _P, _P, ctypes.POINTER(Options), ctypes.POINTER(_I), _P], _I),
    "mxk_kmeans_mixed_cached": ([_I64, _I, _I, _P, _P, _P, ctypes.POINTER(Options), ctypes.POINTER(_I), _P], _I),
    "mxk_set_precision_policy": ([_I], _I),
    "mxk_trace_next_call": ([ctypes.POINTER(Trace)], _I),
    "mxk_comm_unique_id": ([ctypes.c_char_p], _I),
    "mxk_comm_init": ([ctypes.POINTER(_P), _I, _I, ctypes.c_char_p], _I),
    "mxk_comm_destroy": ([_P], _I),
    "mxk_inject_rank_failure": ([_I, _I], _I),
    "mxk_kmeans_mixed_sharded": ([_P, _I64, _I, _I, _P, _P, _P, ctypes.POINTER(Options), ctypes.POINTER(_I), _P], _I),
    "mxk_kmeans_mixed_multi": ([_I64, _I, _I, _P, _P, _P, ctypes.POINTER(Options), _I, ctypes.POINTER(_I)], _I),
    "mxk_host_init_kmeanspp": ([_P, _I64, _I, _I, ctypes.c_uint32, _P], _I),
    "mxk_host_init_farthest": ([_P, _I64, _I, _I, _P], _I),
    "mxk_host_read_points": ([ctypes.c_char_p, _I64, _I, _I, _P], _I),
    "mxk_host_read_points_ex": ([ctypes.c_char_p, _I64, _I, _I, _I, _I64, _P], _I),
    "mxk_host_read_points_f32": ([ctypes.c_char_p, _I64, _I, _I, _P], _I),
    "mxk_host_write_labels": ([ctypes.c_char_p, _P, _I64], _I),
    "mxk_cache_write": ([_P, _I, _I64, _P, _P, _P, _P], _I),
    "mxk_cache_read": ([_P, _I, _I64, _P, _P, _P, _P], _I),
    "mxk_cache_append": ([_P, _P, _P], _I),
    "mxk_cache_attention": ([_P, _P, _P], _I),
    "mxk_cache_attention_shared": ([_P, _P, _P, _P], _I),
    "mxk_quantize_fp8": ([_I, _I64, _I64, _P, _I64, _I, _P, _P, _P], _I),
    "mxk_gemm_fp8": ([_I, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64, _P], _I),
    "mxk_linear_fp8": ([_I, _I64, _I64, _I64, _P, _I64, _P, _P, _P, _I64, _P], _I),
    "mxk_profile_enable": ([_I], _I),
    "mxk_profile_read": ([ctypes.POINTER(KernelStat), _I, ctypes.POINTER(_I)], _I),
}

_lib = None


def load(path=None):
    """Load libmxkmeans.so (once) and declare every entry point's signature."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = path or LIB_PATH
    if not os.path.exists(p):
        raise FileNotFoundError(f"{p} is not built; run `make -C mx-kmeans_b200` or __graft_entry__.build()")
    lib = ctypes.CDLL(p)
    for name, (args, res) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    if path is None:
        _lib = lib
    return lib


def check(status):
    if status != OK:
        msg = load().mxk_last_error().decode(errors="replace")
        if status == ERR_INVALID:
            raise MxkInvalidArgument(status, msg)
        raise MxkError(status, msg)


# ----------------------------------------------------------------------------- torch helpers

def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def quantize_rows(bits, points, values, scales, pid=None, max_errors=None, rows=None, stream=None):
    rows = points.shape[0] if rows is None and pid is None else (rows if rows is not None else pid.shape[0])
    check(load().mxk_quantize_rows(bits, rows, points.shape[1], _ptr(points), _ptr(pid), _ptr(values),
                                   _ptr(scales), _ptr(max_errors), _stream(stream)))


def compute_l2_norm(points, norms, stream=None):
    check(load().mxk_compute_l2_norm(points.shape[0], points.shape[1], _ptr(points), _ptr(norms), _stream(stream)))


def precompute_point_bounds(points, norms, upper, stream=None):
    check(load().mxk_precompute_point_bounds(points.shape[0], points.shape[1], _ptr(points), _ptr(norms),
                                             _ptr(upper), _stream(stream)))


def assign_precisions(n, d, upper, gaps, lc, ec, precision, stream=None):
    check(load().mxk_assign_precisions(n, d, _ptr(upper), _ptr(gaps), lc, ec, _ptr(precision), _stream(stream)))


def init_farthest(points, centroids, stream=None):
    """Farthest-first initial centroids (the reference's init_centroids_farthest)
    from device points [n, d] into device centroids [k, d]."""
    n, d = points.shape
    check(load().mxk_init_farthest(n, d, centroids.shape[0], _ptr(points), _ptr(centroids), _stream(stream)))


def init_kmeanspp(points, centroids, seed, stream=None):
    """K-Means++ initial centroids (the reference's init_centroids with
    std::mt19937(seed)) from device points [n, d] into device centroids [k, d]."""
    n, d = points.shape
    check(load().mxk_init_kmeanspp(n, d, centroids.shape[0], _ptr(points), _ptr(centroids), seed & 0xffffffff,
                                   _stream(stream)))


def gemm_tiles_multiplied(reset=False):
    """128 x 192 tiles multiplied by the MX GEMM on the current device since the
    last reset (pruned tiles excluded)."""
    v = ctypes.c_ulonglong(0)
    check(load().mxk_gemm_tiles_multiplied(ctypes.byref(v), 1 if reset else 0))
    return v.value


def gemm_rows_processed(reset=False):
    """Point rows processed by the MX GEMM on the current device since the last
    reset (rows whose labels the loop's bounds proved are not counted)."""
    v = ctypes.c_ulonglong(0)
    check(load().mxk_gemm_rows_processed(ctypes.byref(v), 1 if reset else 0))
    return v.value


def release_workspace():
    """Return the kmeans workspace kept by the library's pool on the current
    device to the driver."""
    check(load().mxk_release_workspace())


def check_mxfp8_scale_codec(result, stream=None):
    """Exhaustive device check of the fused quantizer's MXFP8 scale rule against
    ue8m0(amax / 448); result: 2 int64 device words (count, first pattern)."""
    check(load().mxk_check_mxfp8_scale_codec(_ptr(result), _stream(stream)))


def check_wait_timeout(limit_cycles, outcome, stream=None):
    """Run the bounded-wait self-check (an mbarrier nothing arrives on); returns
    the status the library reports (MXK_ERR_TIMEOUT expected) without raising.
    outcome: 2 int32 device words, 0 = that warp's wait gave up."""
    return load().mxk_check_wait_timeout(int(limit_cycles), _ptr(outcome), _stream(stream))


def gemm_mx(bits, m, n, k, a, a_scales, b, b_scales, out, stream=None):
    check(load().mxk_gemm_mx(bits, m, n, k, _ptr(a), _ptr(a_scales), _ptr(b), _ptr(b_scales), _ptr(out),
                             _stream(stream)))


def gemm_fp32(a, b, out, stream=None):
    check(load().mxk_gemm_fp32(a.shape[0], b.shape[0], a.shape[1], _ptr(a), _ptr(b), _ptr(out), _stream(stream)))


def assign_clusters(rows, k, point_norms, centroid_norms, dots, labels, gaps, pid=None, stream=None):
    check(load().mxk_assign_clusters(rows, k, _ptr(point_norms), _ptr(centroid_norms), _ptr(dots), _ptr(pid),
                                     _ptr(labels), _ptr(gaps), _stream(stream)))


def assign_mx_fused(bits, rows, k, d, a, a_scales, b, b_scales, point_norms, centroid_norms, labels, gaps=None,
                    pid=None, start_hint=None, stream=None):
    check(load().mxk_assign_mx_fused(bits, rows, k, d, _ptr(a), _ptr(a_scales), _ptr(b), _ptr(b_scales),
                                     _ptr(point_norms), _ptr(centroid_norms), _ptr(pid), _ptr(labels), _ptr(gaps),
                                     _ptr(start_hint), _stream(stream)))


def assign_f32_fused(rows, k, d, points, b, b_scales, point_norms, centroid_norms, labels, gaps=None, pid=None,
                     start_hint=None, stream=None):
    check(load().mxk_assign_f32_fused(rows, k, d, _ptr(points), points.shape[0], _ptr(b), _ptr(b_scales),
                                      _ptr(point_norms), _ptr(centroid_norms), _ptr(pid), _ptr(labels), _ptr(gaps),
                                      _ptr(start_hint), _stream(stream)))


def update_centroids(points, labels, old_centroids, centroids, counts, stream=None):
    check(load().mxk_update_centroids(points.shape[0], points.shape[1], centroids.shape[0], _ptr(points),
                                      _ptr(labels), _ptr(old_centroids), _ptr(centroids), _ptr(counts),
                                      _stream(stream)))


def centroid_shift(previous, current, device_sum, stream=None):
    out = ctypes.c_float(0.0)
    check(load().mxk_centroid_shift(previous.numel(), _ptr(previous), _ptr(current), _ptr(device_sum),
                                    ctypes.cast(ctypes.pointer(out), ctypes.c_void_p), _stream(stream)))
    return out.value


def kmeans_mixed(points, centroids, labels, options=None, stream=None, cache_points=False):
    """Run the Lloyd loop in place on device tensors; returns the iteration count.
    cache_points: quantize the points once per call instead of every iteration
    (mxk_kmeans_mixed_cached; same results, reported separately)."""
    opts = options or Options()
    iters = ctypes.c_int(0)
    fn = load().mxk_kmeans_mixed_cached if cache_points else load().mxk_kmeans_mixed
    check(fn(points.shape[0], points.shape[1], centroids.shape[0], _ptr(points), _ptr(centroids), _ptr(labels),
             ctypes.byref(opts), ctypes.byref(iters), _stream(stream)))
    return iters.value


def set_precision_policy(policy):
    """0: the reference's select_precision (always MXFP8, the default); 1: the
    candidate it computes and discards (test hook for the 4/6/8 groups)."""
    check(load().mxk_set_precision_policy(int(policy)))


def trace_next_call(max_iterations, centroids=None, labels=None, group_sizes=None):
    """Arm a trace of the next Lloyd call on the current device: per iteration i <
    max_iterations, centroids[i] <- the centroids it assigns against, labels[i] <-
    its labels, group_sizes[i] <- its (MXFP4, MXFP6, MXFP8) group rows.  The
    tensors are device tensors of shape [max_iterations, ...] (or None)."""
    t = Trace(None if centroids is None else centroids.data_ptr(),
              None if labels is None else labels.data_ptr(),
              None if group_sizes is None else group_sizes.data_ptr(), int(max_iterations))
    check(load().mxk_trace_next_call(ctypes.byref(t)))


def comm_unique_id():
    buf = ctypes.create_string_buffer(128)
    check(load().mxk_comm_unique_id(buf))
    return buf.raw


class Comm:
    """NCCL communicator of one rank (mxk_comm_init / mxk_comm_destroy)."""

    def __init__(self, nranks, rank, unique_id):
        self.handle = ctypes.c_void_p()
        check(load().mxk_comm_init(ctypes.byref(self.handle), nranks, rank, unique_id))

    def close(self):
        if self.handle:
            check(load().mxk_comm_destroy(self.handle))
            self.handle = ctypes.c_void_p()


def inject_rank_failure(rank, iteration):
    """Test hook: the sharded loop of `rank` leaves with an error when it reaches
    `iteration` (rank < 0 disarms)."""
    check(load().mxk_inject_rank_failure(int(rank), int(iteration)))


def shard_rows(n, world, rank):
    """Rows of one rank in the row-sharded path: contiguous shards of n // world
    rows, the first n % world ranks one row more.  -> (first_row, row_count)."""
    if n < 0 or world <= 0 or not 0 <= rank < world:
        raise ValueError(f"shard_rows: bad arguments n={n} world={world} rank={rank}")
    base, extra = divmod(n, world)
    return rank * base + min(rank, extra), base + (1 if rank < extra else 0)


def bootstrap_comm(group=None):
    """This rank's NCCL communicator for kmeans_mixed_sharded.  Rank 0 creates the
    unique id and broadcasts it over an initialized torch.distributed process group
    (any backend, so a gloo group on the host works); a rank that never joins makes
    the broadcast fail with the group's timeout instead of hanging.  -> Comm"""
    import torch.distributed as dist
    rank, world = dist.get_rank(group), dist.get_world_size(group)
    uid = [comm_unique_id() if rank == 0 else None]
    dist.broadcast_object_list(uid, src=dist.get_global_rank(group, 0) if group is not None else 0, group=group)
    return Comm(world, rank, uid[0])


def kmeans_mixed_sharded(comm, points, centroids, labels, options=None, stream=None):
    opts = options or Options()
    iters = ctypes.c_int(0)
    check(load().mxk_kmeans_mixed_sharded(comm.handle, points.shape[0], points.shape[1], centroids.shape[0],
                                          _ptr(points), _ptr(centroids), _ptr(labels), ctypes.byref(opts),
                                          ctypes.byref(iters), _stream(stream)))
    return iters.value


# ----------------------------------------------------------------------------- paged MX cache
# These calls sit on a serving loop's critical path, where a few microseconds of
# checks are a share of the step: each attribute of a tensor is looked at once.

def _bad(message):
    return MxkInvalidArgument(ERR_INVALID, message)


_torch = None
_DTYPES = {}


def _setup():
    global _torch
    import torch
    _torch = torch
    _DTYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})


def _launch_stream(cache, stream):
    """Handle of the stream to launch on: the caller's or the current one of the cache's
    device, which must be the current device."""
    index = cache.index
    if _torch._C._cuda_getDevice() != index:
        raise _bad(f"the cache is on cuda:{index}, which is not the current device")
    return stream.cuda_stream if stream is not None else _torch._C._cuda_getCurrentRawStream(index)


def _vector(t, name, cache, dtype, *shape):
    """Address of t, a contiguous tensor of `dtype` and `shape` on the cache's device."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != cache.index or not t.is_contiguous():
        raise _bad(f"{name}: a contiguous {dtype} tensor of shape {shape} on {cache.device} is needed, got {t.device} "
                   f"{t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _row_fields(t, name, cache, tokens, heads):
    """Fields of the mxk_rows of t [tokens, heads, head_dim], whose features must be contiguous."""
    strides = t.stride()
    if t.shape != (tokens, heads, cache.head_dim) or t.get_device() != cache.index or strides[2] != 1:
        raise _bad(f"{name}: a tensor of shape [{tokens}, {heads}, {cache.head_dim}] on {cache.device} is needed, its "
                   f"features contiguous, got {t.device} {tuple(t.shape)} with strides {strides}")
    return t.data_ptr(), strides[0], strides[1]


def _rows(t, name, cache, tokens, heads):
    return Rows(*_row_fields(t, name, cache, tokens, heads))


# Structs with many fields are packed into bytes, which takes a third of the time of filling
# the ctypes ones.
_APPEND = struct.Struct("@iiq" + "Pqq" * 4 + "PPPqii")
_ATTENTION = struct.Struct("@iiqiiqPqqPPqPfiqPqqP")
_PREFIXES = struct.Struct("@iPPq")
assert [x.size for x in (_APPEND, _ATTENTION, _PREFIXES)] == [ctypes.sizeof(x) for x in (Append, Attention, Prefixes)]


def _packed(layout, *fields):
    try:
        return layout.pack(*fields)
    except struct.error as e:
        raise _bad(f"a number is out of range: {e}") from None


class PagedCache:
    """Paged MX keys and values over the caller's tensors (mxk_cache): values
    [pages, kv_heads, page_size, head_dim * bits / 8] and scales
    [pages, kv_heads, page_size, head_dim / 32], uint8 and contiguous."""

    def __init__(self, k_values, k_scales, v_values, v_scales, bits):
        if _torch is None:
            _setup()
        if bits not in (4, 6, 8):
            raise _bad("bits must be 4, 6 or 8")
        if k_scales.dim() != 4 or not k_scales.is_cuda:
            raise _bad("cache tensors have 4 dimensions and lie on a GPU")
        pages, heads, page, blocks = k_scales.shape
        self.device, self.index = k_scales.device, k_scales.get_device()
        for t, name, last in ((k_values, "k_values", blocks * 4 * bits), (k_scales, "k_scales", blocks),
                              (v_values, "v_values", blocks * 4 * bits), (v_scales, "v_scales", blocks)):
            _vector(t, name, self, _torch.uint8, pages, heads, page, last)
        self.k_values, self.k_scales, self.v_values, self.v_scales = k_values, k_scales, v_values, v_scales
        self.bits, self.pages, self.kv_heads, self.page_size = bits, pages, heads, page
        self.head_dim = blocks * 32
        self.struct = Cache(bits, heads, blocks * 32, page, pages, k_values.data_ptr(), k_scales.data_ptr(),
                            v_values.data_ptr(), v_scales.data_ptr())
        self.handle = ctypes.addressof(self.struct)

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, bits=8, device="cuda"):
        """A cache of zeros."""
        import torch

        def make(last):
            return torch.zeros(pages, kv_heads, page_size, last, dtype=torch.uint8, device=device)
        return cls(make(head_dim * bits // 8), make(head_dim // 32), make(head_dim * bits // 8),
                   make(head_dim // 32), bits)


def _move(fn, cache, k, v, slots, stream):
    dtype, tokens = k.dtype, k.shape[0]
    code = _DTYPES.get(dtype)
    if code is None or v.dtype != dtype:
        raise _bad("k and v: the same one of float32, float16 and bfloat16 is needed")
    kr = _rows(k, "k", cache, tokens, cache.kv_heads)
    vr = _rows(v, "v", cache, tokens, cache.kv_heads)
    at = _vector(slots, "slots", cache, _torch.int64, tokens)
    return fn, code, tokens, kr, vr, at, _launch_stream(cache, stream)


def cache_write(cache, k, v, slots, stream=None):
    """Quantise the rows of k and v [tokens, kv_heads, head_dim] into the cache's
    slots (int64; page * page_size + place; one outside the cache: not kept)."""
    fn, dtype, tokens, kr, vr, at, st = _move(load().mxk_cache_write, cache, k, v, slots, stream)
    check(fn(cache.handle, dtype, tokens, ctypes.byref(kr), ctypes.byref(vr), at, st))


def cache_read(cache, slots, k, v, stream=None):
    """The values that the cache holds at `slots` into k and v [tokens, kv_heads,
    head_dim] (zeros for a slot outside the cache)."""
    fn, dtype, tokens, kr, vr, at, st = _move(load().mxk_cache_read, cache, k, v, slots, stream)
    check(fn(cache.handle, dtype, tokens, at, ctypes.byref(kr), ctypes.byref(vr), st))


_NO_ROWS = 0, 0, 0


def cache_append(cache, q, k, v, positions, cos_sin, slots, q_out=None, interleaved=False, stream=None):
    """Rotate q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] by their
    positions (int64 [tokens]) and quantise the rotated k, and v, into the cache's slots
    (int64 [tokens]; mxk.h, mxk_cache_append).  cos_sin: float32 [positions, rot_dim],
    cosines then sines; pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) if interleaved.  The
    rotated queries go to q_out, or into q itself without one; q may be None."""
    dtype, tokens = k.dtype, k.shape[0]
    code = _DTYPES.get(dtype)
    if code is None or v.dtype != dtype:
        raise _bad("k and v: the same one of float32, float16 and bfloat16 is needed")
    heads, qr, outr = 0, _NO_ROWS, _NO_ROWS
    if q is not None:
        if q.dim() != 3 or q.dtype != dtype or (q_out is not None and q_out.dtype != dtype):
            raise _bad("q and q_out: 3 dimensions and k's type are needed")
        heads = q.shape[1]
        qr = _row_fields(q, "q", cache, tokens, heads)
        outr = qr if q_out is None else _row_fields(q_out, "q_out", cache, tokens, heads)
    elif q_out is not None:
        raise _bad("q_out without q")
    if cos_sin.dim() != 2:
        raise _bad("cos_sin has 2 dimensions")
    rows, rot = cos_sin.shape
    i64 = _torch.int64
    args = _packed(_APPEND, code, heads, tokens, *qr, *outr, *_row_fields(k, "k", cache, tokens, cache.kv_heads),
                   *_row_fields(v, "v", cache, tokens, cache.kv_heads), _vector(slots, "slots", cache, i64, tokens),
                   _vector(positions, "positions", cache, i64, tokens),
                   _vector(cos_sin, "cos_sin", cache, _torch.float32, rows, rot), rows, rot, 1 if interleaved else 0)
    check(load().mxk_cache_append(cache.handle, args, _launch_stream(cache, stream)))


def _attention(cache, q, cu_q, page_table, kv_lens, out, max_q, max_kv, scale, causal, window, lse):
    """mxk_attention of a call's tensors."""
    if q.dim() != 3 or page_table.dim() != 2:
        raise _bad("q has 3 dimensions, page_table 2")
    tokens, heads, _ = q.shape
    dtype, i32 = q.dtype, _torch.int32
    if out.dtype != dtype:
        raise _bad("out must have q's type")
    qr = _row_fields(q, "q", cache, tokens, heads)
    outr = _row_fields(out, "out", cache, tokens, heads)
    seqs, pages = page_table.shape
    stride, step = page_table.stride()
    if page_table.dtype != i32 or page_table.get_device() != cache.index or step != 1 < pages:
        raise _bad(f"page_table: int32 rows on {cache.device} are needed")
    if pages * cache.page_size < max_kv:
        raise _bad("page_table has fewer pages than max_kv tokens need")
    return _packed(_ATTENTION, _DTYPES.get(dtype, -1), heads, tokens, seqs, max_q, max_kv, *qr,
                   _vector(cu_q, "cu_q", cache, i32, seqs + 1), page_table.data_ptr(), stride,
                   _vector(kv_lens, "kv_lens", cache, i32, seqs),
                   cache.head_dim ** -0.5 if scale is None else scale, 1 if causal else 0, window, *outr,
                   0 if lse is None else _vector(lse, "lse", cache, _torch.float32, tokens, heads))


def cache_attention(cache, q, cu_q, page_table, kv_lens, out, max_q, max_kv, scale=None, causal=True, window=0,
                    lse=None, stream=None):
    """Attention of each sequence's newest tokens over its cached ones (mxk.h,
    mxk_cache_attention): q, out [tokens, heads, head_dim] float16 or bfloat16;
    cu_q [seqs + 1], page_table [seqs, pages], kv_lens [seqs] int32; max_q, max_kv:
    bounds on a sequence's new and cached tokens; scale: 1 / sqrt(head_dim) unless
    given; lse: float32 [tokens, heads] or None."""
    args = _attention(cache, q, cu_q, page_table, kv_lens, out, max_q, max_kv, scale, causal, window, lse)
    check(load().mxk_cache_attention(cache.handle, args, _launch_stream(cache, stream)))


def cache_attention_shared(cache, q, cu_q, page_table, kv_lens, cu_groups, prefix_lens, out, max_q, max_kv, max_prefix,
                           scale=None, causal=True, lse=None, stream=None):
    """cache_attention of a batch in which sequences cu_groups[g] .. cu_groups[g + 1] - 1 (int32
    [groups + 1]) have their first prefix_lens[g] (int32 [groups], at most max_prefix) tokens in
    the same slots, which are read once for them all (mxk.h, mxk_cache_attention_shared)."""
    args = _attention(cache, q, cu_q, page_table, kv_lens, out, max_q, max_kv, scale, causal, 0, lse)
    groups = prefix_lens.shape[0] if prefix_lens.dim() else 0
    prefixes = _packed(_PREFIXES, groups, _vector(cu_groups, "cu_groups", cache, _torch.int32, groups + 1),
                       _vector(prefix_lens, "prefix_lens", cache, _torch.int32, groups), max_prefix)
    check(load().mxk_cache_attention_shared(cache.handle, args, prefixes, _launch_stream(cache, stream)))


# ----------------------------------------------------------------------------- E4M3 products

def _matrix(t, name, dtype, index):
    """(address, row stride) of a matrix on cuda:index whose rows are contiguous."""
    if t.dim() != 2 or t.dtype != dtype or t.get_device() != index or (t.stride(1) != 1 and t.shape[1] > 1):
        raise _bad(f"{name}: {dtype} rows on cuda:{index} are needed, got {t.device} {t.dtype} {tuple(t.shape)} with "
                   f"strides {t.stride()}")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1]  # (one row may have any stride)


def _whole(t, name, dtype, index, *shape):
    """Address of a contiguous tensor of `shape` on cuda:index.  Its elements may be bytes or
    torch.float8_e4m3fn where dtype is uint8."""
    if t.shape != shape or t.get_device() != index or not t.is_contiguous() or \
            (t.dtype != dtype and (dtype != _torch.uint8 or t.dtype != _torch.float8_e4m3fn)):
        raise _bad(f"{name}: a contiguous {dtype} tensor of shape {shape} on cuda:{index} is needed, got {t.device} "
                   f"{t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _device_of(t, name):
    """Index of t's device, which must be the current one."""
    if _torch is None:
        _setup()
    index = t.get_device()
    if index < 0 or _torch._C._cuda_getDevice() != index:
        raise _bad(f"{name} must lie on the current GPU, is on {t.device}")
    return index


def _stream_on(index, stream):
    return stream.cuda_stream if stream is not None else _torch._C._cuda_getCurrentRawStream(index)


def quantize_fp8(x, values, scales, block_rows=1, stream=None):
    """E4M3 values (uint8 or float8_e4m3fn [rows, k]) and float32 scales [rows / block_rows,
    k / 128] (rounded up) of the rows of x (mxk.h, mxk_quantize_fp8); block_rows 1 or 128."""
    index = _device_of(x, "x")
    code = _DTYPES.get(x.dtype)
    if code is None or block_rows not in (1, 128):
        raise _bad("x: float32, float16 or bfloat16 is needed; block_rows is 1 or 128")
    at, stride = _matrix(x, "x", x.dtype, index)
    rows, k = x.shape
    check(load().mxk_quantize_fp8(code, rows, k, at, stride, block_rows, _whole(values, "values", _torch.uint8, index, rows, k),
                                  _whole(scales, "scales", _torch.float32, index, -(-rows // block_rows), -(-k // 128)),
                                  _stream_on(index, stream)))


def gemm_fp8(a, a_scales, b, b_scales, out, stream=None):
    """out [m, n] (float32, float16 or bfloat16 rows) = a [m, k] times b [n, k] transposed, E4M3
    with scales per row (a) or 128 rows (b) and 128 features (mxk.h, mxk_gemm_fp8)."""
    index = _device_of(out, "out")
    code = _DTYPES.get(out.dtype)
    if code is None or out.dim() != 2 or a.dim() != 2:
        raise _bad("out: a matrix of float32, float16 or bfloat16 is needed; a has 2 dimensions")
    at, stride = _matrix(out, "out", out.dtype, index)
    (m, n), k = out.shape, a.shape[1]
    blocks = -(-k // 128)
    check(load().mxk_gemm_fp8(code, m, n, k, _whole(a, "a", _torch.uint8, index, m, k),
                              _whole(a_scales, "a_scales", _torch.float32, index, m, blocks),
                              _whole(b, "b", _torch.uint8, index, n, k),
                              _whole(b_scales, "b_scales", _torch.float32, index, -(-n // 128), blocks), at,
                              stride, _stream_on(index, stream)))


def linear_fp8(x, b, b_scales, out, stream=None):
    """out [m, n] = x [m, k] times b [n, k] transposed: quantize_fp8 of x's rows and gemm_fp8 in
    one call (mxk.h, mxk_linear_fp8); x and out have the same type."""
    index = _device_of(out, "out")
    code = _DTYPES.get(out.dtype)
    if code is None or out.dim() != 2 or x.dim() != 2 or x.shape[0] != out.shape[0]:
        raise _bad("x and out: matrices of as many rows, of one of float32, float16 and bfloat16, are needed")
    xa, x_stride = _matrix(x, "x", out.dtype, index)
    at, stride = _matrix(out, "out", out.dtype, index)
    (m, n), k = out.shape, x.shape[1]
    check(load().mxk_linear_fp8(code, m, n, k, xa, x_stride, _whole(b, "b", _torch.uint8, index, n, k),
                                _whole(b_scales, "b_scales", _torch.float32, index, -(-n // 128), -(-k // 128)), at,
                                stride, _stream_on(index, stream)))


def profile_enable(on=True):
    check(load().mxk_profile_enable(1 if on else 0))


def profile_read():
    """{kernel name: (launches, total_ms)} for the current device since profile_enable()."""
    count = ctypes.c_int(0)
    check(load().mxk_profile_read(None, 0, ctypes.byref(count)))
    arr = (KernelStat * max(count.value, 1))()
    check(load().mxk_profile_read(arr, count.value, ctypes.byref(count)))
    return {arr[i].name.decode(): (arr[i].launches, arr[i].total_ms) for i in range(count.value)}


def _np(a):
    return ctypes.c_void_p(a.ctypes.data)


def kmeans_mixed_multi(points, centroids, labels, options, num_gpus):
    """kmeans_mixed over num_gpus GPUs of this node from HOST numpy arrays
    (points n x d float32, centroids k x d float32 in/out, labels n int32 out)."""
    import numpy as np
    for a, t in ((points, np.float32), (centroids, np.float32), (labels, np.int32)):
        if a.dtype != t or not a.flags.c_contiguous:
            raise TypeError("kmeans_mixed_multi: contiguous float32 points/centroids and int32 labels required")
    it = ctypes.c_int(0)
    check(load().mxk_kmeans_mixed_multi(points.shape[0], points.shape[1], centroids.shape[0], _np(points),
                                        _np(centroids), _np(labels), ctypes.byref(options), num_gpus,
                                        ctypes.byref(it)))
    return it.value


def host_init_kmeanspp(points, k, seed):
    """K-Means++ on a host float32 array [n, d] (same selections as the reference)."""
    import numpy as np
    p = np.ascontiguousarray(points, np.float32)
    out = np.empty((k, p.shape[1]), np.float32)
    check(load().mxk_host_init_kmeanspp(_np(p), p.shape[0], p.shape[1], k, seed, _np(out)))
    return out


def host_init_farthest(points, k):
    import numpy as np
    p = np.ascontiguousarray(points, np.float32)
    out = np.empty((k, p.shape[1]), np.float32)
    check(load().mxk_host_init_farthest(_np(p), p.shape[0], p.shape[1], k, _np(out)))
    return out


def host_read_points(path, n, d, padded_d, threads=None, chunk_bytes=0):
    """The reference's CSV reader (parallel); threads/chunk_bytes only change
    how the file is split, never the result."""
    import numpy as np
    out = np.empty((n, padded_d), np.float32)
    if threads is None and not chunk_bytes:
        check(load().mxk_host_read_points(str(path).encode(), n, d, padded_d, _np(out)))
    else:
        check(load().mxk_host_read_points_ex(str(path).encode(), n, d, padded_d, threads or 0, chunk_bytes,
                                             _np(out)))
    return out


def host_read_points_f32(path, n, d, padded_d):
    """Raw little-endian float32 rows (n x d, no header), zero padded."""
    import numpy as np
    out = np.empty((n, padded_d), np.float32)
    check(load().mxk_host_read_points_f32(str(path).encode(), n, d, padded_d, _np(out)))
    return out


def launch_count():
    return load().mxk_launch_count()
