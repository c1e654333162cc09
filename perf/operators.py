"""Measured cases of the paged MX cache: storing keys and values, reading them
back, and the attention of new tokens over them.

A cache holds the keys and values of many sequences in pages of `page` tokens.
Each row of `dim` features (one token, one head) is kept as MX elements of 8, 6
or 4 bits (E4M3, E2M3, E2M1) with one power-of-two scale (a UE8M0 byte) per 32
features: values [pages, heads, page, dim * bits / 8] and scales
[pages, heads, page, dim / 32], both uint8.  A token's place is its slot,
page number * page + place in the page.

  store   quantise the keys and values of some tokens into their slots; the
          slots' new contents are returned as the values they stand for, read
          back through the cache's reading operator
  read    the values that some slots stand for
  attend  softmax(scale * q k^T) v of each sequence's new tokens over its cached
          tokens, the new ones included; several query heads share a key head;
          token j of n new ones in a sequence of length L sits at position
          L - n + j and sees the positions up to its own (`causal`), the last
          `window` of them if that is not 0; a row that sees nothing is zero
          with a log-sum-exp of -inf

`own` is set by the caller: False computes everything with elementary torch
operations in float32, True calls the library.
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
        # The new tokens of one decode step of a small batch, stored: a few rows,
        # all latency.
        dict(name="store decode step 8 bit", op="store", bits=8, tokens=8, kv_heads=8, dim=128, page=64, dtype="bf16",
             fused=True, pool=4096),
        # A long prompt's keys and values, stored and handed back: streaming.
        dict(name="store prompt 8 bit", op="store", bits=8, tokens=16384, kv_heads=8, dim=128, page=64, dtype="bf16",
             fused=True, pool=32768),
        # An odd number of float32 rows of narrow heads in 6 bits.
        dict(name="store odd rows 6 bit f32", op="store", bits=6, tokens=4099, kv_heads=5, dim=64, page=16,
             dtype="f32", fused=False, pool=8192),
        # A shared prefix in 4 bits, read back for a consumer in bf16.
        dict(name="read prefix 4 bit", op="read", bits=4, tokens=65536, kv_heads=8, dim=128, page=64, dtype="bf16",
             pool=98304),
        # A short odd prefix, read back in float32.
        dict(name="read short prefix 8 bit f32", op="read", bits=8, tokens=777, kv_heads=4, dim=64, page=32,
             dtype="f32", pool=4096),
        # One decode step of a few short conversations: launch latency.
        dict(name="attend few short 8 bit", op="attend", bits=8, seqs=4, q_lo=1, q_hi=1, kv_lo=17, kv_hi=900, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False, fused=True),
        # One decode step of a busy server, lengths spread from one token to 8192.
        dict(name="attend decode batch 8 bit", op="attend", bits=8, seqs=64, q_lo=1, q_hi=1, kv_lo=1, kv_hi=8192,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False, fused=True),
        # Two long documents in 4 bits, one token each: the long axis is split.
        dict(name="attend decode long 4 bit", op="attend", bits=4, seqs=2, q_lo=1, q_hi=1, kv_lo=131000,
             kv_hi=131072, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=True,
             fused=False),
        # Drafted tokens checked in one pass, sliding window, narrow heads, 6 bits.
        dict(name="attend drafts window 6 bit", op="attend", bits=6, seqs=24, q_lo=2, q_hi=5, kv_lo=100, kv_hi=6000,
             heads=24, kv_heads=4, dim=64, page=16, dtype="f16", causal=True, window=1024, lse=True, fused=True),
        # Prompt chunks beside decoding sequences in one call, ragged and odd.
        dict(name="attend mixed chunks 4 bit", op="attend", bits=4, seqs=9, q_lo=1, q_hi=701, kv_lo=333, kv_hi=5003,
             heads=16, kv_heads=4, dim=64, page=32, dtype="f16", causal=True, window=0, lse=False, fused=True),
        # A chunk of a long prompt over what is cached already.
        dict(name="attend chunk 8 bit", op="attend", bits=8, seqs=1, q_lo=512, q_hi=512, kv_lo=16384, kv_hi=16384,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=True, fused=True),
        # The largest chunk: compute.
        dict(name="attend large chunk 8 bit", op="attend", bits=8, seqs=1, q_lo=4096, q_hi=4096, kv_lo=16384,
             kv_hi=16384, heads=32, kv_heads=8, dim=128, page=128, dtype="bf16", causal=True, window=0, lse=False,
             fused=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend"])
    bits = rng.choice([8, 8, 6, 4])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 48, 64, 128])
    kv_heads = rng.randint(1, 8)
    if op in ("store", "read"):
        tokens = _log_int(rng, 1, 16384)
        case = dict(op=op, bits=bits, tokens=tokens, kv_heads=kv_heads, dim=dim, page=page,
                    dtype=rng.choice(["bf16", "f16", "f32"]), pool=tokens + rng.randint(0, 8192))
        if op == "store":
            case["fused"] = rng.random() < 0.5
        return case
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    seqs = _log_int(rng, 1, 64)
    q_hi = rng.choice([1, rng.randint(1, 8), _log_int(rng, 8, 4096)])
    q_lo = rng.choice([1, q_hi, rng.randint(1, q_hi)])
    kv_hi = max(q_hi, _log_int(rng, 1, 131072))
    # no more than the largest listed case works on: scores, and cached tokens
    while seqs > 1 and (seqs * q_hi * kv_hi * group * kv_heads > 32 * 4096 * 4096 or seqs * kv_hi > 262144):
        seqs -= 1
    while q_hi * kv_hi * group * kv_heads > 32 * 4096 * 4096:
        q_hi = max(1, q_hi // 2)
        q_lo = min(q_lo, q_hi)
        kv_hi = max(q_hi, kv_hi // 2)
    kv_lo = rng.choice([q_hi, kv_hi, rng.randint(q_hi, kv_hi)])
    causal = rng.random() < 0.85
    window = _log_int(rng, 1, 4096) if causal and rng.random() < 0.25 else 0
    return dict(op=op, bits=bits, seqs=seqs, q_lo=q_lo, q_hi=q_hi, kv_lo=kv_lo, kv_hi=kv_hi,
                heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=rng.choice(["bf16", "f16"]),
                causal=causal, window=window, lse=rng.random() < 0.5, fused=rng.random() < 0.5)


def _lengths(case):
    """(new tokens, length) of each sequence: spread between the bounds."""
    n = case["seqs"]
    out = []
    for i in range(n):
        a = (i * 37 % n) / (n - 1) if n > 1 else 1.0
        b = (i * 23 % n) / (n - 1) if n > 1 else 1.0
        q = case["q_lo"] + int(round(min(1.0, a) * (case["q_hi"] - case["q_lo"])))
        kv = case["kv_lo"] + int(round(min(1.0, b) * (case["kv_hi"] - case["kv_lo"])))
        out.append((q, max(q, kv)))
    return out


def _seen(case):
    """Sum over the sequences of the (new token, cached token) pairs that take part."""
    total = 0
    for q, kv in _lengths(case):
        if not case["causal"]:
            total += q * kv
            continue
        for p in range(kv - q, kv):
            total += min(p + 1, case["window"]) if case["window"] else p + 1
    return total


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    row = case["dim"] * case["bits"] // 8 + case["dim"] // 32  # a cached row of one head
    if case["op"] in ("store", "read"):
        rows = 2 * case["tokens"] * case["kv_heads"]
        full = rows * case["dim"] * size
        if case["op"] == "read":
            return {"bytes": rows * row + full + 8 * case["tokens"], "flops": rows * case["dim"]}
        # in, kept, kept again by the reading, out
        return {"bytes": 2 * (rows * row + full) + 8 * case["tokens"], "flops": 6 * rows * case["dim"]}
    lens = _lengths(case)
    new = sum(q for q, _ in lens)
    cached = 0
    for q, kv in lens:  # the tokens that any new token of the sequence sees
        first = max(0, kv - q + 1 - case["window"]) if case["window"] else 0
        cached += kv - first
    data = 2 * new * case["heads"] * case["dim"] * size + 2 * cached * case["kv_heads"] * row
    if case["lse"]:
        data += 4 * new * case["heads"]
    return {"bytes": data, "flops": 4 * _seen(case) * case["heads"] * case["dim"]}


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


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim, page, hk = DTYPES[case["dtype"]], case["dim"], case["page"], case["kv_heads"]
    state = {"case": case}
    if case["op"] in ("store", "read"):
        pages = -(-case["pool"] // page)
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:case["tokens"]]
        if case["tokens"] > 64:  # a prompt fills whole pages, in any order of pages
            order = torch.randperm(pages, generator=gen, device="cuda")
            at = torch.arange(case["tokens"], device="cuda")
            slots = order[at // page] * page + at % page
        state["slots"] = slots
        new = case["tokens"]
    else:
        lens = _lengths(case)
        new = sum(q for q, _ in lens)
        need = [-(-kv // page) for _, kv in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda")
        # one row of page numbers per sequence; what lies past a sequence's pages is never used
        width = max(need)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        table = first[:, None] + torch.arange(width, device="cuda")[None, :]
        state["table"] = order[table.clamp(max=pages - 1)].to(torch.int32)
        state["kv_lens"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        starts = [0]
        for q, _ in lens:
            starts.append(starts[-1] + q)
        state["cu_q"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        state["max_q"] = max(q for q, _ in lens)
        state["max_kv"] = max(kv for _, kv in lens)
        state["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"),
                                               torch.tensor([q for q, _ in lens], device="cuda"))
    if case["op"] != "store":
        # what the cache holds already
        state["k_values"], state["k_scales"] = _packed(_keys(gen, pages * page, hk, dim).to(dtype), case["bits"])
        state["v_values"], state["v_scales"] = _packed(_values(gen, pages * page, hk, dim).to(dtype), case["bits"])
        for name in ("k_values", "v_values", "k_scales", "v_scales"):
            state[name] = state[name].unflatten(0, (pages, page)).transpose(1, 2).contiguous()
    else:
        shape = (pages, hk, page)
        for side in "kv":
            state[side + "_values"] = torch.zeros(*shape, dim * case["bits"] // 8, dtype=torch.uint8, device="cuda")
            state[side + "_scales"] = torch.zeros(*shape, dim // 32, dtype=torch.uint8, device="cuda")
    if case["op"] == "read":
        state["k_out"] = torch.empty(new, hk, dim, dtype=dtype, device="cuda")
        state["v_out"] = torch.empty(new, hk, dim, dtype=dtype, device="cuda")
        return state
    hq = case.get("heads", 0)
    q = torch.randn(new, hq, dim, generator=gen, device="cuda")
    k, v = _keys(gen, new, hk, dim), _values(gen, new, hk, dim)
    if case["fused"]:  # slices of one projection's output
        both = torch.cat([q, k, v], 1).to(dtype)
        q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    state["q"], state["k"], state["v"] = (t.to(dtype) for t in (q, k, v))
    if case["op"] == "store":
        state["k_out"] = torch.empty(new, hk, dim, dtype=dtype, device="cuda")
        state["v_out"] = torch.empty(new, hk, dim, dtype=dtype, device="cuda")
    else:
        state["out"] = torch.empty(new, hq, dim, dtype=dtype, device="cuda")
        state["lse"] = torch.empty(new, hq, dtype=torch.float32, device="cuda") if case["lse"] else None
    return state


# -------------------------------------------------------------- the plain form

def _round_trip(x, bits):
    """The values that rows of x stand for once they are held as MX elements."""
    mant, bias, most = FORMATS[bits]
    blocks = x.float().unflatten(-1, (-1, 32))
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


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "store":
        return [_round_trip(state[s], case["bits"]).to(dtype) for s in "kv"]
    if case["op"] == "read":
        return [_at_slots(state, s, state["slots"]).to(dtype) for s in "kv"]
    seqs, max_q, max_kv, page = case["seqs"], state["max_q"], state["max_kv"], case["page"]
    hq, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    at = torch.arange(max_kv, device="cuda")
    slots = state["table"][:, at // page].long() * page + at % page
    k, v = (_at_slots(state, s, slots) for s in "kv")  # [seqs, max_kv, hk, dim]
    n = state["cu_q"][1:] - state["cu_q"][:-1]
    local = torch.arange(state["q"].shape[0], device="cuda") - state["cu_q"][state["seq"]]
    q = torch.zeros(seqs, max_q, hq, dim, device="cuda")
    q[state["seq"], local] = state["q"].float()
    q = q.view(seqs, max_q, hk, hq // hk, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seqs, hk, group * max_q, dim]
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(dim ** -0.5).unflatten(2, (hq // hk, max_q))
    pos = (state["kv_lens"] - n)[:, None] + torch.arange(max_q, device="cuda")[None, :]
    hidden = (at >= state["kv_lens"][:, None])[:, None, :].expand(seqs, max_q, max_kv)
    if case["causal"]:
        hidden = hidden | (at > pos[..., None])
    if case["window"]:
        hidden = hidden | (at <= pos[..., None] - case["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (hq // hk, max_q))
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[state["seq"], local].to(dtype)
    if not case["lse"]:
        return [out]
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).flatten(2, 3)[state["seq"], local]
    return [out, lse]


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
    cache = state.get("cache")
    if cache is None:  # a handle on the cache's tensors, which a program keeps as long as they
        cache = state["cache"] = mxk.PagedCache(state["k_values"], state["k_scales"], state["v_values"],
                                                state["v_scales"], case["bits"])
    if case["op"] == "store":
        mxk.cache_write(cache, state["k"], state["v"], state["slots"])
    if case["op"] in ("store", "read"):
        mxk.cache_read(cache, state["slots"], state["k_out"], state["v_out"])
        return [state["k_out"], state["v_out"]]
    mxk.cache_attention(cache, state["q"], state["cu_q"], state["table"], state["kv_lens"], state["out"],
                        max_q=state["max_q"], max_kv=state["max_kv"], causal=case["causal"], window=case["window"],
                        lse=state["lse"])
    return [state["out"], state["lse"]] if case["lse"] else [state["out"]]


# ------------------------------------------------------- the definition in 64 bits

def _table(bits):
    """float64 value of every element code."""
    mant, bias, _ = FORMATS[bits]
    out = []
    for c in range(2 ** bits):
        mag = c % 2 ** (bits - 1)
        e, m = divmod(mag, 2 ** mant)
        x = m * 2.0 ** (1 - bias - mant) if e == 0 else (1 + m / 2 ** mant) * 2.0 ** (e - bias)
        out.append(-x if c >= 2 ** (bits - 1) else x)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _nearest(x, bits):
    """x (float64 rows) with every block of 32 on its format's grid: the scale is the
    smallest power of two that keeps the block in range, each element goes to the
    nearest value of the format, of two to the one with an even code."""
    most = FORMATS[bits][2]
    grid = _table(bits)[:2 ** (bits - 1)]
    grid = grid[grid <= most]  # 8 bits: the last code is no number
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(amax > 0, amax, most) / most)))
    scale = torch.where(scale * most < amax, scale * 2, torch.where(scale * most / 2 >= amax, scale / 2, scale))
    scale = torch.where(amax > 0, scale, 1.0)
    y = (b / scale).abs()
    up = torch.bucketize(y, grid).clamp(max=len(grid) - 1)  # grid[up - 1] < y <= grid[up]
    down = (up - 1).clamp(min=0)
    a, c = y - grid[down], grid[up] - y
    pick = torch.where((a < c) | ((a == c) & (down % 2 == 0)), down, up)
    return (torch.copysign(grid[pick], b) * scale).flatten(-2)


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
    return (_table(bits)[code].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "store":
        return [_nearest(state[s].double(), case["bits"]) for s in "kv"]
    if case["op"] == "read":
        return [_cached64(state, s, state["slots"]) for s in "kv"]
    hq, hk, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = hq // hk
    out = torch.zeros(state["q"].shape[0], hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for i, (n, kv) in enumerate(_lengths(case)):
        t = torch.arange(kv, device="cuda")
        slots = state["table"][i, t // page].long() * page + t % page
        k, v = (_cached64(state, s, slots) for s in "kv")
        span = max(1, 2 ** 26 // kv)
        for j in range(0, n, span):
            m = min(span, n - j)
            p = kv - n + j + torch.arange(m, device="cuda")
            see = torch.ones(m, kv, dtype=torch.bool, device="cuda")
            if case["causal"]:
                see &= t[None, :] <= p[:, None]
            if case["window"]:
                see &= t[None, :] > p[:, None] - case["window"]
            for h in range(hq):
                s = (state["q"][row + j:row + j + m, h].double() @ k[:, h // group].T) / math.sqrt(dim)
                s = torch.where(see, s, -math.inf)
                z = torch.logsumexp(s, -1)
                lse[row + j:row + j + m, h] = z
                w = torch.where(see, torch.exp(s - torch.where(see.any(-1), z, 0.0)[:, None]), 0.0)
                out[row + j:row + j + m, h] = w @ v[:, h // group]
        row += n
    return [out, lse] if case["lse"] else [out]
