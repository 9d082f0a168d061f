"""Plain restatement of the paged 4-bit cache: plan, quantisation, bytes, attention.

Python loops and numpy in 64 bits (32 where the definition rounds to 32), on
the CPU, one number at a time where that is the clearest.
"""

import numpy as np
import torch

PAGE = 64
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """The 256 numbers of e4m3 by byte (bytes 0x7f and 0xff are NaN)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e.astype(float) - 7))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


def to_e4m3(x):
    """Bytes of the nearest non-negative e4m3 numbers (ties to even); 0 <= x <= 448."""
    values = e4m3_values()[:127]
    x = np.asarray(x, dtype=np.float64)
    hi = np.clip(np.searchsorted(values, x), 1, 126)
    lo = hi - 1
    dl, dh = x - values[lo], values[hi] - x
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)


def to_e2m1(x):
    """Codes (sign in bit 3) of the nearest e2m1 numbers, ties to even, saturating at 6."""
    a = np.minimum(np.abs(np.asarray(x, dtype=np.float64)), 8.0)[..., None]  # beyond 6 all the same
    far = np.abs(a - E2M1)
    near = far.min(-1, keepdims=True)
    even = np.where(far == near, np.arange(8) % 2, 2).argmin(-1)  # of equals, the even code
    return (even | np.where(np.signbit(x), 8, 0)).astype(np.uint8)


def quantise(x, factor):
    """x [T, H, D] (any float tensor), factor [H] float32 -> codes [T, H, D], scale bytes [T, H, D/16]."""
    x = x.float().numpy()
    x = np.where(np.isnan(x), np.float32(0), x)
    T, H, D = x.shape
    g = x.reshape(T, H, D // 16, 16)
    f = np.asarray(factor, dtype=np.float32)[None, :, None]
    most = np.abs(g).max(-1)
    with np.errstate(over="ignore"):
        q = (most / (np.float32(6) * f)).astype(np.float32)
    scale = to_e4m3(np.clip(q, np.float32(2.0 ** -9), np.float32(448)))
    step = (e4m3_values()[scale].astype(np.float32) * f).astype(np.float32)
    with np.errstate(over="ignore"):
        y = (g / step[..., None]).astype(np.float32)
    return to_e2m1(y).reshape(T, H, D), scale


def numbers(codes, scale, factor):
    """The 64-bit numbers of codes [T, H, D] and scale bytes [T, H, D/16]; the
    product with the factor is that of the definition (scale * factor in 32 bits)."""
    size = np.where(codes >= 8, -1.0, 1.0) * E2M1[codes & 7]
    f = np.asarray(factor, dtype=np.float32)[None, :, None]
    step = (e4m3_values()[scale].astype(np.float32) * f).astype(np.float32)
    return size * np.repeat(step.astype(np.float64), 16, axis=-1)


def byte_of(which, token, channel, D):
    """(byte, is the high half) of one code in a page: which 0 = K, 1 = V."""
    base, t = token // 16 * 18 * D + which * 9 * D, token % 16
    if which == 0:
        return base + t * D // 2 + channel // 2, channel % 2 == 1
    n, d = channel // (D // 8), channel % (D // 8)
    return base + t // 8 * 4 * D + (n * 4 + t % 8 // 2) * (D // 8) + t % 2 * (D // 16) + d // 2, channel % 2 == 1


def scale_byte_of(which, token, group, D):
    base, t = token // 16 * 18 * D + which * 9 * D + 8 * D, token % 16
    if which == 0:
        per = D // 64
        return base + (t % 8 * 4 + group // per) * 2 * per + t // 8 * per + group % per
    return base + (group * 4 + t % 8 // 2) * 4 + t // 8 * 2 + t % 2


def put(cache, slot, head, which, codes, scales):
    """Writes one token's codes [D] and scale bytes [D/16] into cache [pages, H, 72 D] (numpy)."""
    D = len(codes)
    page, t = slot // PAGE, slot % PAGE
    for d in range(0, D, 2):
        at, _ = byte_of(which, t, d, D)
        cache[page, head, at] = codes[d] | codes[d + 1] << 4
    for g in range(D // 16):
        cache[page, head, scale_byte_of(which, t, g, D)] = scales[g]


def get(cache, slot, head, which, D):
    page, t = slot // PAGE, slot % PAGE
    codes = np.zeros(D, dtype=np.uint8)
    for d in range(0, D, 2):
        at, _ = byte_of(which, t, d, D)
        b = cache[page, head, at]
        codes[d], codes[d + 1] = b & 15, b >> 4
    return codes, np.array([cache[page, head, scale_byte_of(which, t, g, D)] for g in range(D // 16)], dtype=np.uint8)


def plan(tables, lengths, counts, free_pages, free_count, tokens):
    """One step of page bookkeeping, request by request, on lists; returns everything anew."""
    tables = [list(row) for row in tables]
    free_pages = list(free_pages)
    width = len(tables[0]) if tables else 0
    lengths = [min(max(n, 0), width * PAGE) for n in lengths]
    pages = lambda n: -(-n // PAGE)  # noqa: E731
    free = min(max(free_count, 0), len(free_pages))
    for r, c in enumerate(counts):
        if c < 0:
            for page in tables[r][:pages(lengths[r])]:
                if free < len(free_pages):
                    free_pages[free] = page
                    free += 1
    query_start, slots, positions, added, new = [0], [-1] * tokens, [-1] * tokens, [], []
    wanted = taken = 0
    for r, c in enumerate(counts):
        n, start = max(c, 0), query_start[-1]
        query_start.append(start + n)
        fits = c >= 0 and lengths[r] + n <= width * PAGE and start + n <= tokens
        need = pages(lengths[r] + n) - pages(lengths[r]) if fits else 0
        wanted += need
        ok = fits and (need == 0 or wanted <= free)
        if ok:
            for i in range(need):
                tables[r][pages(lengths[r]) + i] = free_pages[free - 1 - (wanted - need) - i]
            taken += need
            for i in range(n):
                at = lengths[r] + i
                positions[start + i] = at
                page = tables[r][at // PAGE]
                if 0 <= page <= (2 ** 31 - 1) // PAGE:  # else no slot has its number
                    slots[start + i] = page * PAGE + at % PAGE
        added.append(n if ok else 0)
        new.append(0 if c < 0 else lengths[r] + added[-1])
    query_start = [min(n, 2 ** 31 - 1) for n in query_start]
    return {"tables": tables, "free_pages": free_pages, "query_start": query_start, "lengths": new, "added": added,
            "slots": slots, "positions": positions, "free_count": free - taken}


def attention(q, k, v, scale, causal):
    """Rows q [n, D] against keys k, v [len, D] in float64 -> (output, sum of p |v| / sum of p)."""
    n, length = q.shape[0], k.shape[0]
    out, size = torch.zeros(n, v.shape[1], dtype=torch.float64), torch.zeros(n, v.shape[1], dtype=torch.float64)
    for i in range(n):
        last = length - n + i + 1 if causal else length
        if last <= 0:
            continue
        p = torch.softmax(scale * (k[:last].double() @ q[i].double()), 0)
        out[i], size[i] = p @ v[:last].double(), p @ v[:last].double().abs()
    return out, size
