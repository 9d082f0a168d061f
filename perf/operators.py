"""Timed cases of the paged 4-bit key/value cache: its page plan, writes, reads and attention.

The cache is a uint8 tensor [pages, kv_heads, 72 * D] (D = head dim, 64 or 128).
A page holds 64 tokens of one kv head as four blocks of 16 tokens, 18 * D bytes
each: K codes (8 D), K scales (D), V codes (8 D), V scales (D). A code is an
e2m1 number (sign, two exponent bits, one mantissa bit), a scale an e4m3 number
shared by 16 neighbouring channels of one token; a value is
code * scale * (one 32-bit factor per kv head). ``_layout`` has the byte
positions inside a page.
"""

import math
import random

import torch

own = False

PAGE = 64
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases

def listed():
    return [
        # a decoding step of 64 running requests: one token each, a new page now and then
        {"name": "plan-tokens", "op": "plan", "requests": 64, "tokens": 1, "context": 8192, "ended": 0},
        # a refill step: prompts and running requests together, some requests ended
        {"name": "plan-mixed", "op": "plan", "requests": 1000, "tokens": 129, "context": 32768, "ended": 7},
        # the keys and values of one decoding step
        {"name": "write-tokens", "op": "write", "tokens": 64, "kv_heads": 8, "dim": 128, "dtype": "fp16"},
        # the keys and values of a batch of prompts
        {"name": "write-prompt", "op": "write", "tokens": 16411, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # a short prefix taken out of the cache
        {"name": "read-short", "op": "read", "tokens": 257, "kv_heads": 4, "dim": 64, "dtype": "fp16"},
        # a long prefix taken out of the cache, to be moved or attended to in 16 bits
        {"name": "read-prefix", "op": "read", "tokens": 32768, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # the smallest attention call: one request, a short context, no shared heads
        {"name": "attn-one-short", "op": "attn", "requests": 1, "tokens": 1, "context": 1000, "kv_heads": 8,
         "group": 1, "dim": 64, "dtype": "fp16", "causal": True, "ragged": False},
        # one request with a very long context: the key axis has to be split
        {"name": "attn-one-long", "op": "attn", "requests": 1, "tokens": 1, "context": 131072, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "fp16", "causal": True, "ragged": False},
        # a decoding step of a ragged batch
        {"name": "attn-batch", "op": "attn", "requests": 32, "tokens": 1, "context": 16384, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "bf16", "causal": True, "ragged": True},
        # a few drafted tokens for each of several requests
        {"name": "attn-drafts", "op": "attn", "requests": 16, "tokens": 5, "context": 4096, "kv_heads": 24,
         "group": 1, "dim": 128, "dtype": "fp16", "causal": True, "ragged": True},
        # prompts behind cached prefixes
        {"name": "attn-prompts", "op": "attn", "requests": 4, "tokens": 1021, "context": 8192, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "bf16", "causal": True, "ragged": True},
        # one block of new positions that sees itself and a long past without a causal mask
        {"name": "attn-block-long", "op": "attn", "requests": 1, "tokens": 4096, "context": 16384, "kv_heads": 24,
         "group": 1, "dim": 128, "dtype": "fp16", "causal": False, "ragged": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "write", "read", "attn", "attn", "attn", "attn"])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1000), "tokens": _log(rng, 1, 129),
                "context": _log(rng, 64, 32768), "ended": rng.choice([0, 0, 3, 7])}
    if op in ("write", "read"):
        kv_heads, dim = rng.choice([1, 2, 4, 8, 24]), rng.choice([64, 128])
        most = 16411 * 8 * 128 // (kv_heads * dim)
        return {"op": op, "tokens": _log(rng, 1, min(most, 65536)), "kv_heads": kv_heads, "dim": dim,
                "dtype": rng.choice(["fp16", "bf16"])}
    kv_heads, group, dim = rng.choice([1, 2, 4, 8, 24]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128])
    requests = _log(rng, 1, 32)
    # no more cached values than the largest listed batch, no more products than the longest listed block
    context = _log(rng, 1, max(2, min(131072, 32 * 16384 * 8 * 128 // (2 * requests * kv_heads * dim))))
    most = min(4096, context, 4096 * 24 * 16384 // (2 * requests * kv_heads * group * context))
    few = rng.random() < 0.5
    return {"op": op, "requests": requests, "tokens": rng.choice([1, 1, 2, 5]) if few or most < 2 else _log(rng, 1, most),
            "context": context, "kv_heads": kv_heads, "group": group, "dim": dim, "dtype": rng.choice(["fp16", "bf16"]),
            "causal": rng.random() < 0.7, "ragged": rng.random() < 0.6}


def _sizes(case):
    """(tokens to add, tokens in the cache after that) of each request: the case alone decides."""
    rng = random.Random("%d %d %d" % (case["requests"], case["tokens"], case["context"]))
    got = []
    for _ in range(case["requests"]):
        n, length = case["tokens"], case["context"]
        if case.get("ragged"):
            n, length = rng.randint((n + 1) // 2, n), rng.randint((length + 3) // 4, length)
        got.append((n, length))
    return got


def _plan_sizes(case):
    """(tokens held before, tokens to add or -1 for a request that ended) of each request."""
    rng = random.Random("%d %d %d" % (case["requests"], case["tokens"], case["context"]))
    got = []
    for r in range(case["requests"]):
        n = 1 if case["tokens"] == 1 or rng.random() < 0.5 else rng.randint(0, case["tokens"])
        got.append((rng.randint(0, case["context"] - 1), -1 if case["ended"] and r % 16 < case["ended"] else n))
    return got


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


# ------------------------------------------------------------------ inputs

def _layout(dim, device):
    """Byte positions in a page of each token's K codes, K scales, V codes and V scales."""
    t = torch.arange(PAGE, device=device)[:, None]
    d = torch.arange(0, dim, 2, device=device)[None]
    g = torch.arange(dim // 16, device=device)[None]
    block, u = t // 16 * 18 * dim, t % 16
    half, pair, odd = u // 8, u % 8 // 2, u % 2
    lanes, wide = dim // 64, dim // 8
    kc = block + u * (dim // 2) + d // 2
    ks = block + 8 * dim + (u % 8 * 4 + g // lanes) * 2 * lanes + half * lanes + g % lanes
    vc = block + 9 * dim + half * 4 * dim + (d // wide * 4 + pair) * wide + odd * (wide // 2) + d % wide // 2
    vs = block + 17 * dim + (g * 4 + pair) * 4 + half * 2 + odd
    return kc, ks, vc, vs


def _quantise(x, factor):
    """x [..., heads, D] as bytes of two codes [..., heads, D / 2] and scales [..., heads, D / 16] in e4m3."""
    x = x.float().unflatten(-1, (-1, 16))
    f = factor[:, None, None]
    scale = (x.abs().amax(-1, keepdim=True) / (6.0 * f)).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
    y = x / (scale.float() * f)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int() + (torch.signbit(y).int() << 3)).flatten(-2)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), scale.squeeze(-1).view(torch.uint8)


def _store(cache, slots, k, v, k_factor, v_factor):
    """Writes the tokens k and v [T, heads, D] to their slots."""
    dim = k.shape[-1]
    heads = torch.arange(k.shape[1], device=k.device)[None, :, None]
    page, at = (slots // PAGE).long()[:, None, None], (slots % PAGE).long()
    kc, ks, vc, vs = _layout(dim, k.device)
    codes, scales = _quantise(k, k_factor)
    cache[page, heads, kc[at][:, None]] = codes
    cache[page, heads, ks[at][:, None]] = scales
    codes, scales = _quantise(v, v_factor)
    cache[page, heads, vc[at][:, None]] = codes
    cache[page, heads, vs[at][:, None]] = scales


def _values(codes, scales, factor):
    """32-bit values [..., heads, n, D] of bytes of two codes and of scales [..., heads, n, ...]."""
    one = torch.tensor(E2M1 + tuple(-e for e in E2M1), device=codes.device)
    both = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)
    x = both[codes.int()].flatten(-2).unflatten(-1, (-1, 16))
    return (x * (scales.view(torch.float8_e4m3fn).float() * factor[:, None, None])[..., None]).flatten(-2)


def _unpack(pages, dim, k_factor, v_factor):
    """K and V [..., heads, 64, D] in 32 bits of pages [..., heads, 72 * D]."""
    kc, ks, vc, vs = _layout(dim, pages.device)
    return (_values(pages[..., kc], pages[..., ks], k_factor), _values(pages[..., vc], pages[..., vs], v_factor))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _fill(cache, g, dim, k_factor, v_factor):
    """Keys with a few large channels and values, over the whole cache, 4096 pages at a time."""
    heads = cache.shape[1]
    wide = 1.0 + 3.0 * (torch.rand(heads, dim, generator=g, device="cuda") > 0.95).float()
    for p in range(0, cache.shape[0], 4096):
        slots = torch.arange(p * PAGE, min(p + 4096, cache.shape[0]) * PAGE, device="cuda")
        n = slots.numel()
        _store(cache, slots, _normal(g, n, heads, dim) * wide, _normal(g, n, heads, dim), k_factor, v_factor)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "plan":
        sizes = _plan_sizes(case)
        held, counts = [s[0] for s in sizes], [s[1] for s in sizes]
        width = _pages(case["context"] + case["tokens"])
        used = sum(_pages(n) for n in held)
        spare = sum(_pages(n + max(c, 0)) - _pages(n) for n, c in sizes) + 5
        order = torch.randperm(used + spare, generator=g, device="cuda", dtype=torch.int32)
        have = torch.tensor([_pages(n) for n in held], device="cuda")
        tables = torch.zeros(len(sizes), width, dtype=torch.int32, device="cuda")
        tables[torch.arange(width, device="cuda")[None] < have[:, None]] = order[:used]
        free_pages = torch.full((used + spare,), -1, dtype=torch.int32, device="cuda")
        free_pages[:spare] = order[used:]
        total = sum(max(c, 0) for c in counts)
        # the token buffer of a program is a little larger than most steps need
        return {"op": op, "tables": tables, "free_pages": free_pages, "tokens": (total + 127) // 64 * 64,
                "lengths": torch.tensor(held, dtype=torch.int32, device="cuda"),
                "counts": torch.tensor(counts, dtype=torch.int32, device="cuda"),
                "free_count": torch.tensor([spare], dtype=torch.int32, device="cuda")}
    heads, dim = case["kv_heads"], case["dim"]
    k_factor = 0.5 + torch.rand(heads, generator=g, device="cuda") * 0.1
    v_factor = 0.25 + torch.rand(heads, generator=g, device="cuda") * 0.1
    state = {"op": op, "dim": dim, "dtype": _dtype(case), "k_factor": k_factor, "v_factor": v_factor}
    if op in ("write", "read"):
        tokens = case["tokens"]
        pages = _pages(tokens) + 3
        state["cache"] = torch.zeros(pages, heads, 72 * dim, dtype=torch.uint8, device="cuda")
        table = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        at = torch.arange(tokens, device="cuda") + 7  # the first page is partly filled already
        state["slots"] = (table[at // PAGE] * PAGE + at % PAGE).int()
        if op == "write":
            # K and V as the two last thirds of a fused projection's output
            qkv = _normal(g, tokens, 3, heads, dim, dtype=state["dtype"])
            state["k"], state["v"] = qkv[:, 1], qkv[:, 2]
        else:
            _fill(state["cache"], g, dim, k_factor, v_factor)
        return state
    sizes = _sizes(case)
    starts = [0]
    for n, _ in sizes:
        starts.append(starts[-1] + n)
    need = [_pages(length) for _, length in sizes]
    state["cache"] = torch.zeros(sum(need) + 2, heads, 72 * dim, dtype=torch.uint8, device="cuda")
    _fill(state["cache"], g, dim, k_factor, v_factor)
    order = torch.randperm(sum(need) + 2, generator=g, device="cuda", dtype=torch.int32)
    state["tables"] = torch.zeros(len(sizes), max(need), dtype=torch.int32, device="cuda")
    have = torch.tensor(need, device="cuda")
    state["tables"][torch.arange(max(need), device="cuda")[None] < have[:, None]] = order[:sum(need)]
    state["lengths"] = torch.tensor([s[1] for s in sizes], dtype=torch.int32, device="cuda")
    state["query_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["q"] = _normal(g, starts[-1], heads * case["group"], dim, dtype=state["dtype"])
    state["scale"], state["causal"], state["most"] = dim ** -0.5, case["causal"], case["tokens"]
    return state


# --------------------------------------------------------------- operators

def run(s):
    if own:
        import gfx906_b200

        if s["op"] == "plan":
            plan = gfx906_b200.cache4_plan(s["tables"], s["lengths"], s["counts"], s["free_pages"], s["free_count"],
                                           s["tokens"])
            return {"tables": s["tables"], "free_pages": s["free_pages"], "query_start": plan.query_start,
                    "lengths": plan.lengths, "added": plan.added, "slots": plan.slots, "positions": plan.positions,
                    "free_count": plan.free_count}
        if s["op"] == "write":
            gfx906_b200.cache4_write(s["k"], s["v"], s["cache"], s["slots"], s["k_factor"], s["v_factor"])
        if s["op"] in ("write", "read"):
            k, v = gfx906_b200.cache4_read(s["cache"], s["slots"], s["k_factor"], s["v_factor"], dtype=s["dtype"])
            return {"k": k, "v": v}
        return {"o": gfx906_b200.attn_cache4(s["q"], s["cache"], s["tables"], s["lengths"], s["query_start"],
                                             s["scale"], causal=s["causal"], k_scale=s["k_factor"],
                                             v_scale=s["v_factor"], max_tokens=s["most"])}
    if s["op"] == "plan":
        return _plan(s)
    if s["op"] == "write":
        _store(s["cache"], s["slots"], s["k"], s["v"], s["k_factor"], s["v_factor"])
    if s["op"] in ("write", "read"):
        return _read(s)
    return {"o": _attention(s)}


def _plan(s):
    tables, lengths, counts, stack = s["tables"], s["lengths"], s["counts"], s["free_pages"]
    requests, width = tables.shape
    device = tables.device
    ended = counts < 0
    n = counts.clamp(min=0)
    held = (lengths + PAGE - 1) // PAGE
    start = torch.cumsum(n, 0)
    first = start - n
    columns = torch.arange(width, device=device)
    # pages of ended requests go on top of the stack, in the order of the requests and of their tables
    back = torch.where(ended, held, 0)
    back_end = torch.cumsum(back, 0)
    row, column = torch.nonzero(columns[None] < back[:, None], as_tuple=True)
    stack[s["free_count"].long() + (back_end - back)[row] + column] = tables[row, column]
    free = s["free_count"] + back_end[-1]
    # pages for the new tokens come off the top, as long as there are any
    fits = ~ended & (lengths + n <= width * PAGE) & (start <= s["tokens"])
    need = torch.where(fits, (lengths + n + PAGE - 1) // PAGE - held, 0)
    need_end = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (need_end <= free))
    take = torch.where(granted, need, 0)
    row, column = torch.nonzero(columns[None] < take[:, None], as_tuple=True)
    tables[row, held[row] + column] = stack[(free - 1 - (need_end - need)[row] - column).long()]
    # each token's request, position and slot
    token = torch.arange(s["tokens"], device=device)
    r = torch.searchsorted(start, token, right=True).clamp(max=requests - 1)
    position = lengths[r] + token - first[r]
    there = granted[r] & (token < start[-1])
    page = tables[r, (position // PAGE).clamp(0, width - 1)]
    added = torch.where(granted, n, 0)
    return {"tables": tables, "free_pages": stack,
            "query_start": torch.cat([torch.zeros(1, device=device), start]).int(),
            "lengths": torch.where(ended, 0, lengths + added).int(), "added": added.int(),
            "slots": torch.where(there, page * PAGE + position % PAGE, -1).int(),
            "positions": torch.where(there, position, -1).int(), "free_count": (free - take.sum()).int()}


def _read(s):
    kc, ks, vc, vs = _layout(s["dim"], s["cache"].device)
    at = (s["slots"] % PAGE).long()
    pages = (s["slots"] // PAGE).long()[:, None, None]
    heads = torch.arange(s["cache"].shape[1], device=at.device)[None, :, None]
    got = [s["cache"][pages, heads, c[at][:, None]] for c in (kc, ks, vc, vs)]
    # _values has heads before tokens
    got = [x.transpose(0, 1)[None].contiguous() for x in got]
    k = _values(got[0], got[1], s["k_factor"])
    v = _values(got[2], got[3], s["v_factor"])
    return {"k": k[0].transpose(0, 1).to(s["dtype"]).contiguous(), "v": v[0].transpose(0, 1).to(s["dtype"]).contiguous()}


def _attention(s):
    q, start, lengths = s["q"], s["query_start"].long(), s["lengths"].long()
    heads, dim = s["cache"].shape[1], s["dim"]
    k, v = _unpack(s["cache"][s["tables"].long()], dim, s["k_factor"], s["v_factor"])
    k, v = k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)  # [requests, heads, keys, D]
    n = start[1:] - start[:-1]
    i = torch.arange(s["most"], device=q.device)
    there = i[None] < n[:, None]
    at = (start[:-1, None] + i[None]).clamp(max=q.shape[0] - 1)
    # queries by kv head, the heads of its group one after the other: [requests, heads, group * tokens, D]
    x = q[at].float().unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4)
    group = x.shape[2]
    score = x.flatten(2, 3) @ k.transpose(-1, -2)
    score *= s["scale"]
    key = torch.arange(k.shape[2], device=q.device)
    last = lengths[:, None] - 1
    if s["causal"]:
        last = last - n[:, None] + 1 + i[None]
    gone = key[None, None] > last.expand(-1, s["most"])[:, :, None]
    score.unflatten(2, (group, -1)).masked_fill_(gone[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    o = (score @ v) / total.clamp(min=1e-30)
    o = o.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = torch.empty_like(q)
    out[at[there]] = o[there].to(q.dtype)
    return out


# ------------------------------------------------------------------- exact

def _exact_numbers(cache, head, page, token, dim, which):
    """64-bit code * scale of `which` (0: K, 1: V) of one head's tokens, read byte by byte."""
    base = token // 16 * 18 * dim + which * 9 * dim
    t = token % 16
    rows = cache[page, head]
    channel = torch.arange(dim, device=cache.device)[None]
    group = channel // 16
    if which == 0:
        code_at = base[:, None] + t[:, None] * dim // 2 + channel // 2
        per = dim // 64
        scale_at = base[:, None] + 8 * dim + (t[:, None] % 8) * 8 * per + group // per * 2 * per + t[:, None] // 8 * per + group % per
    else:
        eighth = channel // (dim // 8)
        code_at = (base[:, None] + t[:, None] // 8 * 4 * dim + eighth * (dim // 2) + t[:, None] % 8 // 2 * (dim // 8)
                   + t[:, None] % 2 * (dim // 16) + channel % (dim // 8) // 2)
        scale_at = base[:, None] + 8 * dim + group * 16 + t[:, None] % 8 // 2 * 4 + t[:, None] // 8 * 2 + t[:, None] % 2
    byte = rows.gather(1, code_at).long()
    code = torch.where(channel % 2 == 1, byte >> 4, byte & 15)
    e, m = (code >> 1) & 3, (code & 1).double()
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.pow(2.0, (e - 1).double()))
    b = rows.gather(1, scale_at).long()
    se, sm = (b >> 3) & 15, (b & 7).double()
    scale = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.pow(2.0, (se - 7).double()))
    return torch.where(code >= 8, -size, size) * scale


def _exact_held(x, factor):
    """What is read back of x [T, D] of one head after it has been held in 4 bits."""
    x = x.double().unflatten(-1, (-1, 16))
    s = (x.abs().amax(-1, keepdim=True) / (6 * factor)).clamp(2.0 ** -9, 448.0)
    step = torch.pow(2.0, torch.floor(torch.log2(s)).clamp(min=-6) - 3)
    s = torch.round(s / step) * step  # to nearest, ties to even
    table = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    far = (x.abs()[..., None] / (s[..., None] * factor) - table).abs()
    # of two codes that are equally near, the even one
    far = far * 16 + torch.tensor([0.0, 1.0] * 4, dtype=torch.float64, device=x.device) * 1e-9
    return (torch.sign(x) * table[far.argmin(-1)] * s * factor).flatten(-2)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    kf, vf = s["k_factor"].double(), s["v_factor"].double()
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "write":
        return {"k": torch.stack([_exact_held(s["k"][:, h], kf[h]) for h in range(heads)], 1),
                "v": torch.stack([_exact_held(s["v"][:, h], vf[h]) for h in range(heads)], 1)}
    if case["op"] == "read":
        page, token = s["slots"].long() // PAGE, s["slots"].long() % PAGE
        k, v = ([_exact_numbers(s["cache"], h, page, token, dim, w) * f[h] for h in range(heads)]
                for w, f in ((0, kf), (1, vf)))
        return {"k": torch.stack(k, 1), "v": torch.stack(v, 1)}
    q = s["q"].double()
    out = torch.zeros_like(q)
    group, begin = case["group"], 0
    for r, (n, length) in enumerate(_sizes(case)):
        position = torch.arange(length, device=q.device)
        page, token = s["tables"][r].long()[position // PAGE], position % PAGE
        last = torch.arange(n, device=q.device) + length - n if case["causal"] else torch.full((n,), length - 1, device=q.device)
        for h in range(heads):
            k = _exact_numbers(s["cache"], h, page, token, dim, 0) * kf[h]
            v = _exact_numbers(s["cache"], h, page, token, dim, 1) * vf[h]
            for a in range(h * group, h * group + group):
                score = q[begin:begin + n, a] @ k.T * case["dim"] ** -0.5
                score = torch.where(position[None] <= last[:, None], score, -math.inf)
                p = torch.where(last[:, None] >= 0, torch.softmax(score, -1), 0.0)
                out[begin:begin + n, a] = p @ v
        begin += n
    return {"o": out}


# -------------------------------------------------------------------- work

def work(case):
    if case["op"] == "plan":
        sizes = _plan_sizes(case)
        tokens = (sum(max(c, 0) for _, c in sizes) + 127) // 64 * 64
        moved = sum(_pages(h) if c < 0 else _pages(h + c) - _pages(h) for h, c in sizes)
        # lengths and counts in; starts, lengths and added out; slots and positions; a page id read and written
        return {"bytes": 4 * (5 * len(sizes) + 2 * tokens + 2 * moved + 3), "flops": 0}
    dim, heads = case["dim"], case["kv_heads"]
    held = heads * (dim // 2 + dim // 16) * 2  # a token in the cache, K and V
    if case["op"] in ("write", "read"):
        wide = heads * dim * 2 * 2
        # a write is measured together with the read that shows what it wrote
        return {"bytes": case["tokens"] * ((2 if case["op"] == "write" else 1) * (wide + held) + 4), "flops": 0}
    heads_q = heads * case["group"]
    flops = bytes_ = 0
    for n, length in _sizes(case):
        seen = sum(max(0, length - n + 1 + i) for i in range(n)) if case["causal"] else n * length
        flops += 4 * heads_q * dim * seen
        bytes_ += 2 * 2 * n * heads_q * dim + length * held + 4 * _pages(length) + 8
    return {"bytes": bytes_, "flops": flops}
