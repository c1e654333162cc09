"""Measured cases of the quantised layer around the paged MX cache: the products
that make queries, keys and values, their rotation and storing, and the attention
of a batch whose sequences begin alike.

  append   rotate the queries and keys of some tokens by their positions (pairs of
           features i and i + r / 2, or 2 i and 2 i + 1, by the angles of a table of
           cosines and sines), the queries rounded to their type, the keys and the
           values quantised into the tokens' slots of the cache; the slots' new
           contents are returned as the values they stand for, read back through
           the cache's reading operator
  shared   softmax(scale * q k^T) v of each sequence's new tokens over its cached
           ones, causal; the sequences of a group have their first tokens in the
           same slots, a prefix that is read once for all of them
  product  out[i, j] = sum over blocks b of 128 of sa[i, b] * sb[j / 128, b] *
           sum over k in b of a[i, k] * c[j, k], a and c in E4M3
  linear   the same from rows in 16 bits, which are quantised on the way: per row and
           block of 128 the scale max |x| / 448, the quotients to the nearest E4M3

The cache is that of perf/operators.py: MX elements of 8, 6 or 4 bits (E4M3, E2M3,
E2M1), one power-of-two scale (a UE8M0 byte) per 32 features, values [pages, heads,
page, dim * bits / 8] and scales [pages, heads, page, dim / 32].

`own` is set by the caller: False computes everything with elementary torch
operations, True calls the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# bits: (mantissa bits, exponent bias, largest magnitude)
FORMATS = {8: (3, 7, 448.0), 6: (3, 1, 7.5), 4: (1, 1, 6.0)}


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # The new tokens of one decode step of a small batch: a few rows, all latency.
        dict(name="append decode step 8 bit", op="append", bits=8, tokens=8, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, page=64, dtype="bf16", fused=True, far=131072, pool=4096),
        # A long prompt: streaming.
        dict(name="append prompt 8 bit", op="append", bits=8, tokens=16384, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, page=64, dtype="bf16", fused=True, far=32768, pool=32768),
        # An odd number of float32 rows of narrow heads, half of each rotated in pairs, 6 bits.
        dict(name="append odd rows 6 bit f32", op="append", bits=6, tokens=4099, heads=15, kv_heads=5, dim=64, rot=32,
             interleaved=True, page=16, dtype="f32", fused=False, far=8192, pool=8192),
        # A few conversations under a short common instruction: latency.
        dict(name="shared few short 8 bit", op="shared", bits=8, groups=1, seqs=4, prefix_lo=1000, prefix_hi=1000, q_lo=1,
             q_hi=1, own_lo=20, own_hi=100, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", lse=False, fused=True),
        # One decode step of a busy server whose requests all carry the same instructions.
        dict(name="shared decode batch 8 bit", op="shared", bits=8, groups=1, seqs=64, prefix_lo=8192, prefix_hi=8192,
             q_lo=1, q_hi=1, own_lo=1, own_hi=512, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", lse=False,
             fused=True),
        # Drafted tokens of several tenants, each with its own odd prefix; narrow heads, 4 bits.
        dict(name="shared drafts of 3 groups 4 bit", op="shared", bits=4, groups=3, seqs=17, prefix_lo=777,
             prefix_hi=3001, q_lo=2, q_hi=5, own_lo=5, own_hi=700, heads=24, kv_heads=4, dim=64, page=16, dtype="f16",
             lse=True, fused=False),
        # Many questions about one long document.
        dict(name="shared long document 8 bit", op="shared", bits=8, groups=1, seqs=256, prefix_lo=32768,
             prefix_hi=32768, q_lo=1, q_hi=1, own_lo=10, own_hi=300, heads=32, kv_heads=8, dim=128, page=128,
             dtype="bf16", lse=False, fused=True),
        # A single token through a projection: the weights' bytes.
        dict(name="linear single token", op="linear", m=1, n=4096, k=4096, dtype="bf16"),
        # A decode batch through a fused projection.
        dict(name="linear decode batch", op="linear", m=64, n=6144, k=4096, dtype="bf16"),
        # A prompt chunk through a wide layer.
        dict(name="linear prompt chunk", op="linear", m=2048, n=14336, k=4096, dtype="bf16"),
        # Odd everything, float32 out.
        dict(name="product odd sizes f32", op="product", m=777, n=1003, k=1040, dtype="f32"),
        # The largest product: compute.
        dict(name="product large", op="product", m=8192, n=8192, k=8192, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "shared", "shared", "linear", "product"])
    if op in ("linear", "product"):
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 16384), 16 * _log_int(rng, 4, 1024)
        while m * n * k > 8192 ** 3:
            m = max(1, m // 2)
        return dict(op=op, m=m, n=n, k=k, dtype=rng.choice(["bf16", "f16"] + (["f32"] if op == "product" else [])))
    bits = rng.choice([8, 8, 6, 4])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 48, 64, 128])
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "append":
        tokens = min(_log_int(rng, 1, 16384), 16384 * 40 // (heads + 8))
        return dict(op=op, bits=bits, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 16 * rng.randint(1, dim // 16)]),
                    interleaved=rng.random() < 0.4, page=page, dtype=rng.choice(["bf16", "f16", "f32"]),
                    fused=rng.random() < 0.5, far=_log_int(rng, 4096, 262144), pool=tokens + rng.randint(0, 8192))
    seqs = _log_int(rng, 1, 256)
    groups = rng.choice([1, 1, rng.randint(1, min(seqs, 8))])
    prefix_hi = _log_int(rng, 16, 32768)
    prefix_lo = rng.choice([prefix_hi, rng.randint(1, prefix_hi)])
    q_hi = rng.choice([1, 1, rng.randint(1, 8), _log_int(rng, 8, 512)])
    q_lo = rng.choice([1, q_hi, rng.randint(1, q_hi)])
    own_hi = q_hi + _log_int(rng, 1, 4096)
    # no more scores than the largest listed case has, nor cached tokens
    while seqs > groups and (seqs * q_hi * (prefix_hi + own_hi) * heads > 256 * 33000 * 32 or seqs * own_hi > 131072):
        seqs -= 1
    while seqs * q_hi * (prefix_hi + own_hi) * heads > 256 * 33000 * 32:
        q_hi = max(1, q_hi // 2)
        q_lo = min(q_lo, q_hi)
        own_hi = max(q_hi, own_hi // 2)
        prefix_hi = max(1, prefix_hi // 2)
        prefix_lo = min(prefix_lo, prefix_hi)
    own_lo = rng.choice([q_hi, own_hi, rng.randint(q_hi, own_hi)])
    return dict(op=op, bits=bits, groups=groups, seqs=seqs, prefix_lo=prefix_lo, prefix_hi=prefix_hi, q_lo=q_lo,
                q_hi=q_hi, own_lo=own_lo, own_hi=own_hi, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=rng.choice(["bf16", "f16"]), lse=rng.random() < 0.5, fused=rng.random() < 0.5)


def _spread(i, n, step, lo, hi):
    """The i-th of n numbers that are spread between two bounds in no order."""
    return lo + int(round((i * step % n) / (n - 1) * (hi - lo))) if n > 1 else hi


def _lengths(case):
    """Of each group its prefix and the (new tokens, own tokens) of its sequences."""
    groups, n = case["groups"], case["seqs"]
    out = []
    for g in range(groups):
        first, last = g * n // groups, (g + 1) * n // groups
        seqs = []
        for i in range(first, last):
            q = _spread(i, n, 37, case["q_lo"], case["q_hi"])
            seqs.append((q, max(q, _spread(i, n, 23, case["own_lo"], case["own_hi"]))))
        out.append((_spread(g, groups, 1, case["prefix_lo"], case["prefix_hi"]), seqs))
    return out


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // 128)
        a = m * k * size if case["op"] == "linear" else m * k + 4 * m * blocks
        return {"bytes": a + n * k + 4 * -(-n // 128) * blocks + m * n * size, "flops": 2 * m * n * k}
    row = case["dim"] * case["bits"] // 8 + case["dim"] // 32  # a cached row of one head
    if case["op"] == "append":
        q, kv = case["tokens"] * case["heads"], 2 * case["tokens"] * case["kv_heads"]
        # queries in and out; keys and values in, kept, kept again by the reading, out; the table's rows
        data = 2 * (q + kv) * case["dim"] * size + 2 * kv * row + case["tokens"] * (16 + 4 * case["rot"])
        return {"bytes": data, "flops": 3 * (q + kv // 2) * case["rot"] + 6 * kv * case["dim"]}
    cached = new = seen = 0
    for prefix, seqs in _lengths(case):
        rest = prefix % case["page"]  # in a page of its own for every sequence
        cached += prefix - rest
        for q, kv in seqs:
            cached += rest + kv
            new += q
            seen += sum(prefix + p + 1 for p in range(kv - q, kv))
    data = 2 * new * case["heads"] * case["dim"] * size + 2 * cached * case["kv_heads"] * row
    if case["lse"]:
        data += 4 * new * case["heads"]
    return {"bytes": data, "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ the inputs

def _keys(gen, *shape):
    """Keys as models have them: a few features of each head far larger than the rest."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-2:], generator=gen, device="cuda") < 0.03
    return x * torch.where(loud, 8.0, 1.0) + torch.where(loud, 6.0, 0.0)


def _values(gen, *shape):
    x = torch.randn(*shape, generator=gen, device="cuda")
    return x * torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))


def _packed(x, bits):
    """Rows of float values as (packed MX elements, scales), uint8: how a cache that
    is at hand before the call came to hold them."""
    mant, bias, most = FORMATS[bits]
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    frac, expo = torch.frexp(amax / most)
    expo = torch.where(frac == 0.5, expo - 1, expo).clamp(-127, 127)
    expo = torch.where(amax > 0, expo, 0)
    y = torch.ldexp(blocks, -expo)
    mag = y.abs().clamp(max=most)
    step = torch.frexp(mag)[1].sub(1).clamp(min=1 - bias) - mant
    mag = torch.ldexp(torch.round(torch.ldexp(mag, -step)), step).clamp(max=most)
    e = torch.frexp(mag)[1] - 1
    low = (e < 1 - bias) | (mag == 0)
    code = torch.where(low, torch.ldexp(mag, torch.full_like(e, bias - 1 + mant)),
                       (e + bias) * 2 ** mant + torch.ldexp(mag, mant - e) - 2 ** mant).int()
    code = (code + ((y < 0).int() << (bits - 1))).flatten(-2)
    if bits == 6:
        four = code.unflatten(-1, (-1, 4)) << torch.tensor([0, 6, 12, 18], device=x.device, dtype=torch.int32)
        word = four.sum(-1, keepdim=True) >> torch.tensor([0, 8, 16], device=x.device, dtype=torch.int32)
        code = (word & 255).flatten(-2)
    elif bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code.to(torch.uint8).contiguous(), (expo.squeeze(-1) + 127).to(torch.uint8).contiguous()


def _blocked(x, rows):
    """x [n, k] as E4M3 values (their bytes) and a float32 scale per `rows` rows and 128
    columns: max |x| / 448 rounded once, the quotients to the nearest value."""
    n, k = x.shape
    whole = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -n % rows))
    tiles = whole.unflatten(0, (-1, rows)).unflatten(2, (-1, 128))
    scale = (tiles.abs().amax((1, 3), keepdim=True) / 448.0).float().clamp(min=2.0 ** -126)
    codes = (_round8(tiles / scale.double())).flatten(2, 3).flatten(0, 1)[:n, :k].float()
    return codes.to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), scale[:, 0, :, 0].contiguous()


def _round8(y):
    """y (64 bits) to the nearest value of E4M3, of two to the even one."""
    step = torch.frexp(y)[1].sub(1).clamp(min=-6) - 3
    return torch.ldexp(torch.round(torch.ldexp(y, -step)), step).clamp(-448.0, 448.0)


def _table(rows, rot):
    """Cosines and sines of the first positions, as a program keeps them: float32, from
    angles in 64 bits."""
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * \
        10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _cache_of(state, pages, gen, filled):
    case = state["case"]
    hk, dim, page, bits = case["kv_heads"], case["dim"], case["page"], case["bits"]
    for side, make in (("k", _keys), ("v", _values)):
        if filled:
            values, scales = _packed(make(gen, pages * page, hk, dim).to(DTYPES[case["dtype"]]), bits)
            values, scales = (t.unflatten(0, (pages, page)).transpose(1, 2).contiguous() for t in (values, scales))
        else:
            values = torch.zeros(pages, hk, page, dim * bits // 8, dtype=torch.uint8, device="cuda")
            scales = torch.zeros(pages, hk, page, dim // 32, dtype=torch.uint8, device="cuda")
        state[side + "_values"], state[side + "_scales"] = values, scales


def _prepare_product(case, state, gen):
    m, n, k = case["m"], case["n"], case["k"]
    # activations with a few loud features, weights of a layer
    x = torch.randn(m, k, generator=gen, device="cuda")
    x *= torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    w = torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5
    state["w"], state["w_scales"] = _blocked(w, 128)
    if case["op"] == "linear":
        state["x"] = x.to(DTYPES[case["dtype"]])
    else:
        state["a"], state["a_scales"] = _blocked(x, 1)
    state["out"] = torch.empty(m, n, dtype=DTYPES[case["dtype"]], device="cuda")
    return state


def _prepare_append(case, state, gen):
    page, tokens, hq, hk, dim = case["page"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    pages = -(-case["pool"] // page)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens]
    positions = torch.randint(0, case["far"], (tokens,), generator=gen, device="cuda")
    if tokens > 64:  # a prompt fills whole pages, in any order of pages, one position after the other
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(tokens, device="cuda")
        slots = order[at // page] * page + at % page
        positions = (at + int(torch.randint(0, case["far"], (1,), generator=gen, device="cuda"))) % case["far"]
    state["slots"], state["positions"] = slots, positions
    state["cos_sin"] = _table(case["far"], case["rot"])
    _cache_of(state, pages, gen, False)
    q, k, v = torch.randn(tokens, hq, dim, generator=gen, device="cuda"), _keys(gen, tokens, hk, dim), \
        _values(gen, tokens, hk, dim)
    if case["fused"]:  # slices of one projection's output
        both = torch.cat([q, k, v], 1).to(dtype)
        q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    state["q"], state["k"], state["v"] = (t.to(dtype) for t in (q, k, v))
    state["q_out"] = torch.empty(tokens, hq, dim, dtype=dtype, device="cuda")
    state["k_out"] = torch.empty(tokens, hk, dim, dtype=dtype, device="cuda")
    state["v_out"] = torch.empty(tokens, hk, dim, dtype=dtype, device="cuda")
    return state


def _prepare_shared(case, state, gen):
    page, hq, hk, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    lens = _lengths(case)
    flat = [(g, prefix, q, kv) for g, (prefix, seqs) in enumerate(lens) for q, kv in seqs]
    # The whole pages of a prefix are shared; where it ends inside a page, every sequence has
    # that page for itself.
    width = max(-(-(prefix + kv) // page) for _, prefix, _, kv in flat)
    pages, rows, seen = 0, [], {}
    for g, prefix, _, kv in flat:
        common = prefix // page
        if g not in seen:
            seen[g] = pages
            pages += common
        need = -(-(prefix + kv) // page)
        row = list(range(seen[g], seen[g] + common)) + list(range(pages, pages + need - common))
        rows.append(row + [0] * (width - need))
        pages += need - common
    pages += 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    _cache_of(state, pages, gen, True)
    state["table"] = order[torch.tensor(rows, device="cuda")].to(torch.int32)
    shared = [prefix // page * page for prefix, _ in lens]
    state["prefix_lens"] = torch.tensor(shared, dtype=torch.int32, device="cuda")
    state["max_prefix"] = max(shared)
    state["kv_lens"] = torch.tensor([prefix + kv for _, prefix, _, kv in flat], dtype=torch.int32, device="cuda")
    state["max_kv"] = max(prefix + kv for _, prefix, _, kv in flat)
    state["max_q"] = max(q for _, _, q, _ in flat)
    n = torch.tensor([q for _, _, q, _ in flat], device="cuda")
    state["cu_q"] = torch.nn.functional.pad(n.cumsum(0), (1, 0)).to(torch.int32)
    sizes = torch.tensor([len(seqs) for _, seqs in lens], device="cuda")
    state["cu_groups"] = torch.nn.functional.pad(sizes.cumsum(0), (1, 0)).to(torch.int32)
    # what the plain form goes by
    state["seq"] = torch.repeat_interleave(torch.arange(len(flat), device="cuda"), n)
    state["group"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), sizes)
    state["most_own"] = max(prefix + kv - shared[g] for g, prefix, _, kv in flat)
    state["most_rows"] = max(sum(q for q, _ in seqs) for _, seqs in lens)
    new = int(n.sum())
    q = torch.randn(new, hq, dim, generator=gen, device="cuda")
    if case["fused"]:  # slices of one projection's output
        q = torch.cat([q, torch.zeros(new, 2 * hk, dim, device="cuda")], 1).to(dtype)[:, :hq]
    state["q"] = q.to(dtype)
    state["out"] = torch.empty(new, hq, dim, dtype=dtype, device="cuda")
    state["lse"] = torch.empty(new, hq, dtype=torch.float32, device="cuda") if case["lse"] else None
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"append": _prepare_append, "shared": _prepare_shared}.get(case["op"], _prepare_product)
    return make(case, {"case": case}, gen)


# -------------------------------------------------------------- the plain form

def _round_trip(x, bits):
    """The values that rows of x (64 bits, or exact in 32) stand for once they are held
    as MX elements."""
    mant, bias, most = FORMATS[bits]
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    frac, expo = torch.frexp(amax / most)
    expo = torch.where(frac == 0.5, expo - 1, expo)
    expo = torch.where(amax > 0, expo, 0)
    y = torch.ldexp(blocks, -expo)
    step = torch.frexp(y)[1].sub(1).clamp(min=1 - bias) - mant
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step).clamp(-most, most)
    return torch.ldexp(y, expo).flatten(-2)


def _unpacked(values, scales, bits):
    """float32 values of packed rows."""
    mant, bias, _ = FORMATS[bits]
    code = values.int()
    if bits == 6:
        b = code.unflatten(-1, (-1, 3))
        word = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
        code = torch.stack([word & 63, (word >> 6) & 63, (word >> 12) & 63, word >> 18], -1).flatten(-2)
    elif bits == 4:
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    mag = code & ((1 << (bits - 1)) - 1)
    e, m = mag >> mant, mag & ((1 << mant) - 1)
    x = torch.ldexp((torch.where(e > 0, m + (1 << mant), m)).float(), e.clamp(min=1) - bias - mant)
    x = torch.where(code >> (bits - 1) > 0, -x, x)
    return torch.ldexp(x.unflatten(-1, (-1, 32)), (scales.int() - 127)[..., None]).flatten(-2)


def _at_slots(state, side, slots):
    case = state["case"]
    page, place = slots // case["page"], slots % case["page"]
    return _unpacked(state[side + "_values"][page, :, place], state[side + "_scales"][page, :, place], case["bits"])


def _rotated(x, cos, sin, interleaved):
    """x [tokens, heads, dim] with the pairs of its first features turned; cos, sin
    [tokens, 1, r / 2]."""
    half = cos.shape[-1]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1)


def _plain_append(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    cos, sin = state["cos_sin"][state["positions"]].double()[:, None].chunk(2, -1)
    # keys in 64 bits: many lie next to a border between two elements
    k = _round_trip(_rotated(state["k"].double(), cos, sin, case["interleaved"]), case["bits"])
    q = _rotated(state["q"].float(), cos.float(), sin.float(), case["interleaved"])
    return [q.to(dtype), k.float().to(dtype), _round_trip(state["v"].float(), case["bits"]).to(dtype)]


def _plain_shared(state):
    case = state["case"]
    dtype, page = DTYPES[case["dtype"]], case["page"]
    hq, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    seq, group, cu_q, table = state["seq"], state["group"], state["cu_q"].long(), state["table"].long()
    groups, seqs, share = case["groups"], case["seqs"], hq // hk
    prefix, first = state["prefix_lens"].long(), state["cu_groups"].long()
    row = torch.arange(seq.shape[0], device="cuda")
    q = state["q"].float()
    # the prefixes: all rows of a group at once
    in_group = row - cu_q[first[group[seq]]]
    most_rows, max_prefix = state["most_rows"], state["max_prefix"]
    t = torch.arange(max_prefix, device="cuda")
    slots = table[first[:-1]][:, t // page] * page + t % page
    k1, v1 = (_at_slots(state, s, slots) for s in "kv")  # [groups, max_prefix, hk, dim]
    q1 = torch.zeros(groups, most_rows, hq, dim, device="cuda")
    q1[group[seq], in_group] = q
    q1 = q1.view(groups, most_rows, hk, share, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s1 = torch.matmul(q1, k1.permute(0, 2, 3, 1)).mul_(dim ** -0.5)  # [groups, hk, share * rows, max_prefix]
    s1.masked_fill_((t >= prefix[:, None])[:, None, None], -math.inf)
    # each sequence's own tokens
    n = cu_q[1:] - cu_q[:-1]
    in_seq = row - cu_q[seq]
    max_q, most_own, start = state["max_q"], state["most_own"], prefix[group]
    t = start[:, None] + torch.arange(most_own, device="cuda")
    at = (t // page).clamp(max=table.shape[1] - 1)
    slots = torch.gather(table, 1, at) * page + t % page
    k2, v2 = (_at_slots(state, s, slots) for s in "kv")
    q2 = torch.zeros(seqs, max_q, hq, dim, device="cuda")
    q2[seq, in_seq] = q
    q2 = q2.view(seqs, max_q, hk, share, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s2 = torch.matmul(q2, k2.permute(0, 2, 3, 1)).mul_(dim ** -0.5).unflatten(2, (share, max_q))
    pos = (state["kv_lens"] - n)[:, None] + torch.arange(max_q, device="cuda")
    s2.masked_fill_((t[:, None, :] > pos[..., None])[:, None, None], -math.inf)
    s2 = s2.flatten(2, 3)

    def part(s, v, heads_first):
        """Maxima, sums of weights and weighted values, by token and head."""
        top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full_like(s[..., :0].sum(-1, keepdim=True), -math.inf)
        top = torch.where(top == -math.inf, -3e38, top)
        s.sub_(top).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s, v.permute(0, 2, 1, 3))
        return [x.unflatten(2, (share, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)[heads_first] for x in (top, total, o)]
    top1, total1, o1 = part(s1, v1, (group[seq], in_group))
    top2, total2, o2 = part(s2, v2, (seq, in_seq))
    top = torch.maximum(top1, top2)
    f1, f2 = torch.exp(top1 - top), torch.exp(top2 - top)
    total = total1 * f1 + total2 * f2
    out = ((o1 * f1 + o2 * f2) / total).to(dtype)
    return [out, (top + torch.log(total)).squeeze(-1)] if case["lse"] else [out]


def _whole(codes, scales, rows):
    """float32 values of E4M3 bytes and their scales per `rows` rows and 128 columns."""
    n, k = codes.shape
    scales = scales.repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return codes.view(torch.float8_e4m3fn).float() * scales


def _plain(state):
    case = state["case"]
    if case["op"] == "append":
        return _plain_append(state)
    if case["op"] == "shared":
        return _plain_shared(state)
    w = _whole(state["w"], state["w_scales"], 128)
    # (quotients in 64 bits: some lie next to a border between two elements)
    a, a_scales = _blocked(state["x"], 1) if case["op"] == "linear" else (state["a"], state["a_scales"])
    return [torch.matmul(_whole(a, a_scales, 1), w.T).to(DTYPES[case["dtype"]])]


# ---------------------------------------------------------------------- a pass

def _library():
    import sys
    if "mx-kmeans_b200" not in sys.path:
        sys.path.insert(0, "mx-kmeans_b200")
    import mxk
    return mxk


def run(state):
    if not own:
        return _plain(state)
    mxk = _library()
    case = state["case"]
    if case["op"] == "linear":
        mxk.linear_fp8(state["x"], state["w"], state["w_scales"], state["out"])
        return [state["out"]]
    if case["op"] == "product":
        mxk.gemm_fp8(state["a"], state["a_scales"], state["w"], state["w_scales"], state["out"])
        return [state["out"]]
    cache = state.get("cache")
    if cache is None:  # a handle on the cache's tensors, which a program keeps as long as they
        cache = state["cache"] = mxk.PagedCache(state["k_values"], state["k_scales"], state["v_values"],
                                                state["v_scales"], case["bits"])
    if case["op"] == "append":
        mxk.cache_append(cache, state["q"], state["k"], state["v"], state["positions"], state["cos_sin"],
                         state["slots"], q_out=state["q_out"], interleaved=case["interleaved"])
        mxk.cache_read(cache, state["slots"], state["k_out"], state["v_out"])
        return [state["q_out"], state["k_out"], state["v_out"]]
    mxk.cache_attention_shared(cache, state["q"], state["cu_q"], state["table"], state["kv_lens"], state["cu_groups"],
                               state["prefix_lens"], state["out"], max_q=state["max_q"], max_kv=state["max_kv"],
                               max_prefix=state["max_prefix"], lse=state["lse"])
    return [state["out"], state["lse"]] if case["lse"] else [state["out"]]


# ------------------------------------------------------- the definition in 64 bits

def _elements(bits):
    """float64 value of every element code."""
    mant, bias, _ = FORMATS[bits]
    out = []
    for c in range(2 ** bits):
        mag = c % 2 ** (bits - 1)
        e, m = divmod(mag, 2 ** mant)
        x = m * 2.0 ** (1 - bias - mant) if e == 0 else (1 + m / 2 ** mant) * 2.0 ** (e - bias)
        out.append(-x if c >= 2 ** (bits - 1) else x)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _on_grid(y, bits):
    """|y| on the format's grid: of the two nearest values the nearer, of equally near
    ones that with the even code."""
    most = FORMATS[bits][2]
    grid = _elements(bits)[:2 ** (bits - 1)]
    grid = grid[grid <= most]  # 8 bits: the last code is no number
    y = y.abs().clamp(max=most)
    up = torch.bucketize(y, grid).clamp(max=len(grid) - 1)  # grid[up - 1] < y <= grid[up]
    down = (up - 1).clamp(min=0)
    a, c = y - grid[down], grid[up] - y
    return grid[torch.where((a < c) | ((a == c) & (down % 2 == 0)), down, up)]


def _nearest(x, bits):
    """x (float64 rows) with every block of 32 on its format's grid, the scale the
    smallest power of two that keeps the block in range."""
    most = FORMATS[bits][2]
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(amax > 0, amax, most) / most)))
    scale = torch.where(scale * most < amax, scale * 2, torch.where(scale * most / 2 >= amax, scale / 2, scale))
    scale = torch.where(amax > 0, scale, 1.0)
    return (torch.copysign(_on_grid(b / scale, bits), b) * scale).flatten(-2)


def _cached64(state, side, slots):
    case = state["case"]
    page, place, bits = slots // case["page"], slots % case["page"], case["bits"]
    raw = state[side + "_values"][page, :, place].long()
    scale = torch.exp2(state[side + "_scales"][page, :, place].double() - 127)
    if bits == 8:
        code = raw
    else:
        flat = (raw[..., None] >> torch.arange(8, device="cuda")) & 1  # the row as a string of bits, lowest first
        code = (flat.flatten(-2).unflatten(-1, (-1, bits)) << torch.arange(bits, device="cuda")).sum(-1)
    return (_elements(bits)[code].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _exact_append(case, state):
    half = case["rot"] // 2
    angles = state["cos_sin"][state["positions"]].double()
    out = []
    for name in ("q", "k"):
        x = state[name].double()
        y = x.clone()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
            c, s = angles[:, i, None], angles[:, half + i, None]
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., b] * c + x[..., a] * s
        out.append(y if name == "q" else _nearest(y, case["bits"]))
    return out + [_nearest(state["v"].double(), case["bits"])]


def _exact_shared(case, state):
    hq, hk, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = hq // hk
    out = torch.zeros(state["q"].shape[0], hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    row = i = 0
    kept = None  # the first sequence's keys and values hold the prefix of its group
    for g, (prefix, seqs) in enumerate(_lengths(case)):
        shared = prefix // page * page
        for j, (n, own_len) in enumerate(seqs):
            kv = prefix + own_len
            t = torch.arange(shared if j else 0, kv, device="cuda")
            slots = state["table"][i, t // page].long() * page + t % page
            mine = [_cached64(state, s, slots) for s in "kv"]
            if j == 0:
                kept = [x[:shared] for x in mine]
            else:
                mine = [torch.cat([a, b]) for a, b in zip(kept, mine)]
            k, v = (x.permute(1, 0, 2) for x in mine)  # [hk, kv, dim]
            q = state["q"][row:row + n].double().unflatten(1, (hk, group)).permute(1, 2, 0, 3).flatten(1, 2)
            s = (q @ k.transpose(1, 2)) / math.sqrt(dim)  # [hk, group * n, kv]
            see = torch.arange(kv, device="cuda")[None, :] <= kv - n + torch.arange(n, device="cuda")[:, None]
            s = s.unflatten(1, (group, n)).masked_fill(~see, -math.inf).flatten(1, 2)
            z = torch.logsumexp(s, -1)
            o = torch.exp(s - z[..., None]) @ v
            out[row:row + n] = o.unflatten(1, (group, n)).permute(2, 0, 1, 3).flatten(1, 2)
            lse[row:row + n] = z.unflatten(1, (group, n)).permute(2, 0, 1).flatten(1, 2)
            row += n
            i += 1
    return [out, lse] if case["lse"] else [out]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, state)
    if case["op"] == "shared":
        return _exact_shared(case, state)
    values = _elements(8)
    values[127], values[255] = math.nan, math.nan
    k = case["k"]
    out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for b in range(-(-k // 128)):
        at = slice(128 * b, min(k, 128 * b + 128))
        w = values[state["w"][:, at].long()]
        w = w * torch.repeat_interleave(state["w_scales"][:, b].double(), 128)[:case["n"], None]
        if case["op"] == "linear":
            x = state["x"][:, at].double()
            s = torch.clamp((x.abs().amax(1) / 448.0).float(), min=2.0 ** -126).double()[:, None]
            a = torch.copysign(_on_grid(x / s, 8), x) * s
        else:
            a = values[state["a"][:, at].long()] * state["a_scales"][:, b, None].double()
        out += a @ w.T
    return [out]
