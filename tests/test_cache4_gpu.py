"""The paged 4-bit cache on the GPU against its oracle (needs a B200)."""

import random

import numpy as np
import pytest
import torch

import gfx906_b200 as g
from oracle import cache4 as oracle

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def operator():
    assert g.load_attention() is not None, g.last_error()
    yield
    assert g.device_status(reset=True) == 0


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# -------------------------------------------------------------------- plan

def check_plan(tables, lengths, counts, free_pages, free_count, tokens):
    want = oracle.plan(tables, lengths, counts, free_pages, free_count, tokens)
    width = len(tables[0]) if tables else 3
    t, f = ints(tables).reshape(len(tables), width), ints(free_pages)
    for _ in range(2):  # a step may be planned again
        plan = g.cache4_plan(t, ints(lengths), ints(counts), f, ints([free_count]), tokens)
        assert t.tolist() == want["tables"]
        assert f.tolist() == want["free_pages"]
        for name in ("query_start", "lengths", "added", "slots", "positions"):
            assert getattr(plan, name).tolist() == want[name], name
        assert plan.free_count.tolist() == [want["free_count"]]


def random_state(rng, requests, width, longest, extra, ended=0.2):
    lengths = [rng.randint(0, min(longest, width * 64)) for _ in range(requests)]
    held = [-(-n // 64) for n in lengths]
    order = list(range(sum(held) + extra))
    rng.shuffle(order)
    tables, at = [], 0
    for h in held:
        tables.append(order[at:at + h] + [-7] * (width - h))
        at += h
    free = order[at:]
    return tables, lengths, free + [-1] * at, len(free)


@pytest.mark.parametrize("requests,width,extra,seed", [(1, 4, 3, 0), (3, 2, 0, 1), (33, 5, 20, 2), (257, 9, 100, 3),
                                                       (1000, 17, 900, 4), (1500, 3, 5, 5)])
def test_plan_random(requests, width, extra, seed):
    rng = random.Random(seed)
    tables, lengths, free, count = random_state(rng, requests, width, 64 * width, extra)
    counts = [rng.choice([-1, 0, 1, 1, 2, 64, rng.randint(0, 200)]) for _ in range(requests)]
    total = sum(max(c, 0) for c in counts)
    for tokens in (total, total + 100, total // 2):
        check_plan(tables, lengths, counts, free, count, tokens)


def test_plan_edges():
    check_plan([], [], [], [3, 4], 2, 5)                                  # no requests
    check_plan([[0, 1]], [128], [0], [], 0, 0)                            # nothing to add, no tokens
    check_plan([[0, 1]], [128], [1], [2], 1, 4)                           # the row is full
    check_plan([[0, -1], [1, -1]], [64, 63], [1, 1], [2, 3], 0, 4)        # no free page: only one fits
    check_plan([[5, 6], [-1, -1]], [70, 0], [-1, 128], [0, 0], 0, 128)    # pages returned and granted at once
    check_plan([[-1] * 3, [-1] * 3], [0, 0], [192, 1], [9, 8, 7, 6], 3, 193)   # the first takes all
    check_plan([[-1] * 3, [-1] * 3], [0, 0], [192, 1], [9, 8, 7, 6], 2, 193)   # nobody overtakes
    check_plan([[4, 5], [6, -1]], [-3, 999], [1, -5], [0, 0, 0], 1, 8)    # lengths out of range
    check_plan([[-1] * 2], [0], [2 ** 31 - 1], [1, 2], 2, 16)             # far too many tokens
    check_plan([[-1] * 2] * 3, [0] * 3, [2 ** 31 - 1] * 3, [1, 2], 2, 0)  # sums past 32 bits: query_start saturates


def test_plan_refusals():
    ok = dict(tables=ints([[0, 1]]), lengths=ints([0]), counts=ints([1]), free_pages=ints([1, 2]), free_count=ints([2]),
              tokens=1)
    g.cache4_plan(**ok)
    for bad in ({"tables": ok["tables"].long()}, {"tables": ok["tables"].cpu()}, {"tables": ok["tables"][0]},
                {"tables": ints([[0, 1], [2, 3]])}, {"tables": ints([[0, 1, 2, 3]])[:, ::2]}, {"lengths": ints([0, 1])},
                {"counts": ints([[1]])}, {"free_pages": ok["free_pages"].float()}, {"free_count": ints([1, 2])},
                {"tokens": -1}, {"tokens": 2 ** 31},
                {"tables": ints([[0]] * 8193), "lengths": ints([0] * 8193), "counts": ints([0] * 8193)}):
        with pytest.raises(RuntimeError):
            g.cache4_plan(**{**ok, **bad})


# ---------------------------------------------------------- write and read

def expect_bytes(cache, slots, k, v, kf, vf):
    """The cache's bytes (numpy) after a write."""
    cache = cache.copy()
    T, H, D = k.shape
    for which, x, f in ((0, k, kf), (1, v, vf)):
        codes, scales = oracle.quantise(x, f)
        for t, slot in enumerate(slots):
            if 0 <= slot < cache.shape[0] * 64:
                for h in range(H):
                    oracle.put(cache, slot, h, which, codes[t, h], scales[t, h])
    return cache


def awkward(T, H, D, dtype, seed):
    """Numbers of many sizes, with ties, zeros, subnormals, infinities and NaN."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=gen) * torch.exp2(torch.randint(-12, 6, (T, H, D // 16), generator=gen).float()
                                                         ).repeat_interleave(16, -1)
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(D // 8)
    x[0] = grid * torch.exp2(torch.arange(H).float())[:, None]  # ties of scale 2^h
    x[0, :, 1::2] *= -1
    x[1 % T] = 0
    if T > 3:
        x[2, 0, 3], x[2, 0, 20], x[3, 0, 5] = float("inf"), -float("inf"), float("nan")
        x[3, 0, 16:32] = float("nan")
    x = x.to(dtype)
    if T > 4 and dtype == torch.float16:
        x[4, 0, :16] = torch.arange(16).to(torch.int16).view(torch.float16)  # subnormal fp16
    return x


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H", [(1, 1), (7, 3), (70, 2), (131, 5)])
def test_write_every_byte(D, dtype, T, H):
    k, v = awkward(T, H, D, dtype, 1), awkward(T, H, D, dtype, 2)
    rng = random.Random(T)
    pages = T // 64 + 3
    slots = rng.sample(range(pages * 64), T)
    if T > 6:
        slots[5], slots[6] = -1, pages * 64  # skipped
    gen = torch.Generator().manual_seed(3)
    before = torch.randint(0, 256, (pages, H, 72 * D), generator=gen, dtype=torch.uint8)
    kf = torch.tensor([2.0 ** (h - 1) for h in range(H)])
    vf = torch.rand(H, generator=gen) + 0.1
    want = expect_bytes(before.numpy(), slots, k, v, kf.numpy(), vf.numpy())
    cache = before.cuda()
    g.cache4_write(k.cuda(), v.cuda(), cache, ints(slots), kf.cuda(), vf.cuda())
    assert np.array_equal(cache.cpu().numpy(), want)
    for out in (torch.float32, torch.float16, torch.bfloat16):
        rk, rv = g.cache4_read(cache, ints(slots), kf.cuda(), vf.cuda(), dtype=out)
        assert rk.shape == (T, H, D) and rk.dtype == out and rk.is_contiguous()
        for which, got, f in ((0, rk, kf), (1, rv, vf)):
            exact = np.zeros((T, H, D))
            for t, slot in enumerate(slots):
                if 0 <= slot < pages * 64:
                    for h in range(H):
                        c, s = oracle.get(want, slot, h, which, D)
                        exact[t, h] = oracle.numbers(c[None, None], s[None, None], f[h:h + 1].numpy())[0, 0]
            # one rounding to 32 bits, one to the type asked for
            assert torch.equal(got.cpu(), torch.from_numpy(exact).float().to(out))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_write_rounds_every_quotient_as_a_division(dtype):
    """Every finite 16-bit number beside each of several largest ones, under factors of any size:
    the codes are those of the 32-bit quotient."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    numbers = bits[torch.isfinite(bits)]
    numbers = numbers[numbers.abs() <= 3.0]  # the 16th of a group is its largest
    numbers = numbers[:numbers.numel() // 15 * 15].view(-1, 15)
    for factor in (1.0, 0.3, 7.1e-3, 1.7e5, 3e-30, 2e30):
        for most in (3.0, 3.7, 5.99):
            x = torch.cat([numbers, torch.full((len(numbers), 1), most, dtype=dtype)], 1)
            x = x[:x.shape[0] // 4 * 4].reshape(-1, 1, 64)
            T = x.shape[0]
            cache = g.cache4_alloc(-(-T // 64), 1, 64)
            f = torch.tensor([factor], device="cuda")
            g.cache4_write(x.cuda(), -x.cuda(), cache, ints(range(T)), f, f)
            k, v = g.cache4_read(cache, ints(range(T)), f, f, dtype=torch.float32)
            codes, scales = oracle.quantise(x, f.cpu().numpy())
            want = torch.from_numpy(oracle.numbers(codes, scales, f.cpu().numpy())).float()
            assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want), (factor, most)


def test_write_without_factors_and_from_strided_rows():
    T, H, D = 40, 4, 128
    qkv = torch.randn(T, 3 * H * D + 64, generator=torch.Generator().manual_seed(5)).half()
    k, v = qkv[:, H * D:2 * H * D].reshape(T, H, D), qkv[:, 2 * H * D:3 * H * D].reshape(T, H, D)
    want = expect_bytes(np.zeros((2, H, 72 * D), dtype=np.uint8), list(range(9, 9 + T)), k, v, np.ones(H), np.ones(H))
    dev = qkv.cuda()
    views = {
        "rows": dev[:, H * D:3 * H * D].unflatten(1, (2, H, D)),
        "heads first": torch.stack([k, v], 1).cuda().transpose(0, 2).contiguous().transpose(0, 2),
        "odd start": torch.cat([torch.zeros(1, device="cuda").half(), dev[:, H * D:3 * H * D].flatten()])[1:].view(T, 2, H, D),
        "strided channels": torch.stack([k, v], 1).cuda().repeat_interleave(2, -1)[..., ::2],
    }
    for name, kv in views.items():
        cache = g.cache4_alloc(2, H, D)
        g.cache4_write(kv[:, 0], kv[:, 1], cache, ints(range(9, 9 + T)))
        assert np.array_equal(cache.cpu().numpy(), want), name


def test_write_and_read_of_nothing():
    cache = g.cache4_alloc(1, 2, 64)
    none = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    g.cache4_write(none, none, cache, ints([]))
    k, v = g.cache4_read(cache, ints([]))
    assert k.shape == v.shape == (0, 2, 64)
    k, v = g.cache4_read(g.cache4_alloc(0, 2, 64), ints([0, 3]))
    assert not k.any() and not v.any()
    g.cache4_write(k, v, g.cache4_alloc(0, 2, 64), ints([0, 3]))


def test_write_and_read_refusals():
    cache = g.cache4_alloc(2, 2, 64)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    s, f = ints([0, 1, 2]), torch.ones(2, device="cuda")
    g.cache4_write(k, k, cache, s, f, f)
    for args in ((k.float(), k.float(), cache, s), (k, k.bfloat16(), cache, s), (k.cpu(), k, cache, s),
                 (k[:, :1], k[:, :1], cache, s), (k, k[:2], cache, s), (k, k, cache, s[:2]), (k, k, cache, s.long()),
                 (k, k, cache[:, :, ::2], s), (k, k, cache.float(), s), (k, k, cache.cpu(), s), (k, k, cache, s.cpu()),
                 (k, k, cache, s, f[:1], f), (k, k, cache, s, f.half(), f), (k, k, cache, s, f, f.cpu()),
                 (k, k, torch.zeros(2, 2, 100, dtype=torch.uint8, device="cuda"), s)):
        with pytest.raises(RuntimeError):
            g.cache4_write(*args)
    for args in ((cache, s.long()), (cache, s[None]), (cache.cpu(), s), (cache, s, f[:1])):
        with pytest.raises(RuntimeError):
            g.cache4_read(*args)
    with pytest.raises(RuntimeError, match="dtype"):
        g.cache4_read(cache, s, dtype=torch.float64)


# --------------------------------------------------------------- attention

class Problem:
    """A cache with scattered pages whose unused places hold 0xff (NaN scales), and its numbers."""

    def __init__(self, counts, lengths, kv_heads, group, D, dtype, seed=0, factors=True, std=1.0, spare=2):
        gen = torch.Generator().manual_seed(seed)
        self.D, self.dtype, self.group, self.kv_heads = D, dtype, group, kv_heads
        self.counts, self.lengths = list(counts), list(lengths)
        need = [-(-n // 64) for n in lengths]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=gen).tolist()
        width = max(need + [1]) + 1
        self.tables, at = [], 0
        for h in need:
            self.tables.append(order[at:at + h] + [10 ** 6] * (width - h))
            at += h
        self.kf = torch.rand(kv_heads, generator=gen) + 0.5 if factors else None
        self.vf = torch.rand(kv_heads, generator=gen) + 0.5 if factors else None
        one = torch.ones(kv_heads)
        self.cache = torch.full((pages, kv_heads, 72 * D), 255, dtype=torch.uint8)
        self.k, self.v = [], []
        cache = self.cache.cuda()
        for r, n in enumerate(lengths):
            k, v = (torch.randn(n, kv_heads, D, generator=gen).half() for _ in range(2))
            k *= std
            slots = [self.tables[r][i // 64] * 64 + i % 64 for i in range(n)]
            g.cache4_write(k.cuda(), v.cuda(), cache, ints(slots), *self.factors())
            k, v = g.cache4_read(cache, ints(slots), *self.factors(), dtype=torch.float32)
            self.k.append(k.cpu())  # the writes and reads have their own tests
            self.v.append(v.cpu())
        self.cache = cache
        self.q = torch.randn(sum(counts), kv_heads * group, D, generator=gen).to(dtype)
        self.query_start = [0]
        for n in counts:
            self.query_start.append(self.query_start[-1] + n)
        self.scale = D ** -0.5

    def factors(self):
        return (None, None) if self.kf is None else (self.kf.cuda(), self.vf.cuda())

    def run(self, q=None, **kw):
        kf, vf = self.factors()
        width = len(self.tables[0]) if self.tables else 1
        return g.attn_cache4((self.q if q is None else q).cuda(), self.cache, ints(self.tables).reshape(-1, width),
                             ints(self.lengths), ints(self.query_start), kw.pop("scale", self.scale), k_scale=kf,
                             v_scale=vf, **kw)

    def check(self, out, causal=True, scale=None, rows=None):
        """Elementwise bound. Each p is rounded to fp16 (2^-11 of itself, or 2^-25 below fp16's normal
        range, per key); scores and exponentials in 32 bits are off by less than 2^-12 of p for the
        scores of these tests; the output is rounded once."""
        out = out.cpu()
        for r, n in enumerate(self.counts):
            first = self.query_start[r]
            pick = range(n) if rows is None else [i for i in rows if i < n]
            for h in range(self.q.shape[1]):
                kv = h // self.group
                k, v = self.k[r][:, kv], self.v[r][:, kv]
                most = float(v.abs().max()) if len(v) else 0.0
                for i in pick:
                    last = self.lengths[r] - n + i + 1 if causal else self.lengths[r]
                    ref, size = oracle.attention(self.q[first + i, h][None], k[:max(last, 0)], v[:max(last, 0)],
                                                 self.scale if scale is None else scale, False)
                    tol = size * (2.0 ** -11 + 2.0 ** -12) + HALF_STEP[self.dtype] * ref.abs() * 1.01 \
                        + max(last, 0) * 2.0 ** -25 * most + 2.0 ** -25
                    off = (out[first + i, h].double() - ref[0]).abs()
                    assert (off <= tol[0]).all(), (r, i, h, float((off / tol[0]).max()))


SHAPES = [  # counts, lengths, kv heads, group
    ([1], [1], 1, 1), ([1], [33], 2, 3), ([1], [1000], 8, 1), ([1, 1, 1], [64, 65, 63], 2, 4),
    ([1] * 9, [5, 700, 31, 32, 128, 1, 300, 96, 511], 1, 8), ([2, 5, 1, 3], [2, 300, 64, 130], 2, 2),
    ([7], [129], 1, 5), ([17], [200], 3, 1), ([1] * 40, [(37 * i) % 190 + 1 for i in range(40)], 2, 1),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_attention_few_tokens(shape, D, dtype):
    p = Problem(*shape, D, dtype, seed=len(shape[0]))
    most = max(shape[0])
    p.check(p.run(max_tokens=most))
    p.check(p.run(max_tokens=most, causal=False), causal=False)


MANY = [  # counts, lengths, kv heads, group, rows checked
    ([65], [65], 1, 1, range(65)), ([130], [130], 1, 1, range(130)), ([100], [77], 1, 2, range(100)),
    ([257], [300], 2, 1, [0, 1, 43, 84, 85, 127, 128, 129, 213, 255, 256]),
    ([33], [1000], 1, 4, range(33)), ([129, 40], [129, 2000], 2, 3, [0, 1, 39, 40, 63, 64, 85, 86, 127, 128]),
    ([1, 90, 0, 3, 64, 300, 2], [700, 90, 5, 1, 64, 513, 130], 1, 2, [0, 1, 2, 63, 64, 89, 127, 128, 255, 256, 299]),
    ([600], [4500], 1, 1, [0, 127, 128, 255, 256, 511, 512, 599]),
    ([70] * 30, [(61 * i) % 300 + 70 for i in range(30)], 5, 1, [0, 63, 69]),  # enough units for every SM
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", MANY, ids=range(len(MANY)))
def test_attention_many_tokens(shape, D, dtype):
    p = Problem(*shape[:4], D, dtype, seed=len(shape[0]))
    p.check(p.run(), rows=shape[4])
    p.check(p.run(causal=False), causal=False, rows=shape[4])
    assert torch.equal(p.run(), p.run())


def test_attention_many_tokens_of_many_requests():
    """More requests than are sorted by length, short and long ones mixed."""
    rng = random.Random(7)
    counts = [rng.choice([1, 2, 65, 70]) for _ in range(150)]
    p = Problem(counts, [n + rng.randint(0, 100) for n in counts], 1, 1, 64, torch.float16)
    p.check(p.run(), rows=[0, 1, 64, 69])


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_attention_many_tokens_scales(scale):
    p = Problem([150], [400], 1, 1, 64, torch.float16)
    p.check(p.run(scale=scale), scale=scale, rows=[0, 77, 149])


def test_attention_many_tokens_bad_pages_nan_queries_and_strides():
    p = Problem([140, 200], [300, 500], 2, 1, 128, torch.float16)
    p.tables[0][0] = -1
    p.tables[0][3] = 10 ** 9
    p.tables[1][2] = 10 ** 9
    p.q[7, 1] = float("nan")
    q = torch.zeros(340, 5, 128, dtype=torch.float16, device="cuda")
    q[:, 2:4] = p.q.cuda()
    out = p.run(q=q[:, 2:4], causal=False)
    assert out[7, 1].isnan().all()
    p.q[7, 1] = 0
    out[7, 1] = p.run(causal=False)[7, 1]
    for r, gone in ((0, [0, 3]), (1, [2])):
        keep = [i for i in range(p.lengths[r]) if i // 64 not in gone]
        p.k[r], p.v[r], p.lengths[r] = p.k[r][keep], p.v[r][keep], len(keep)
    p.check(out, causal=False, rows=[0, 7, 8, 127, 128, 139, 199])


def test_attention_many_tokens_enormous_scores():
    """bf16 rows of any size: beyond 32 bits of score the largest one takes all."""
    p = Problem([130], [300], 1, 1, 128, torch.bfloat16)
    p.q[::2] *= 2.0 ** 60
    p.q[1] *= 2.0 ** -100
    out = p.run(causal=False)
    k, v = p.k[0][:, 0].double(), p.v[0][:, 0].double()
    for i in range(0, 130, 2):
        best = (k @ p.q[i, 0].double()).argmax()
        assert (out[i, 0].cpu().double() - v[best]).abs().max() <= 2.0 ** -8 * v[best].abs().max(), i
    p.q[::2] = 0
    p.check(p.run(causal=False), causal=False, rows=[0, 1, 2, 3, 129])


def test_attention_many_tokens_growing_scores():
    """Scores that grow along the keys move every row's maximum again and again."""
    p = Problem([130], [700], 1, 1, 64, torch.float16)
    p.q *= torch.linspace(0.0, 6.0, 130)[:, None, None].half()
    p.q += 0.5
    p.k[0] += 0.02 * torch.arange(700)[:, None, None]
    slots = ints([p.tables[0][i // 64] * 64 + i % 64 for i in range(700)])
    g.cache4_write(p.k[0].half().cuda(), p.v[0].half().cuda(), p.cache, slots, *p.factors())
    k, v = g.cache4_read(p.cache, slots, *p.factors(), dtype=torch.float32)
    p.k[0], p.v[0] = k.cpu(), v.cpu()
    out = p.run(causal=False).cpu()
    for i in (0, 1, 60, 129):
        ref, size = oracle.attention(p.q[i], p.k[0][:, 0], p.v[0][:, 0], p.scale, False)
        # scores up to 600: 32 bits hold them to 600 * 2^-24 * 64 products, far less than 2^-8 of p
        assert ((out[i, 0].double() - ref[0]).abs() <= size[0] * 2.0 ** -8 + 2.0 ** -11 * ref[0].abs() + 1e-4).all(), i


@pytest.mark.parametrize("D", [64, 128])
def test_attention_long_context_is_split(D):
    p = Problem([1, 1], [20011, 37], 2, 4, D, torch.float16, factors=False)
    p.check(p.run(max_tokens=1))


@pytest.mark.parametrize("requests", [130, 700])
def test_attention_many_requests(requests):
    rng = random.Random(requests)
    lengths = [rng.randint(1, 90) for _ in range(requests)]
    p = Problem([1] * requests, lengths, 1, 2, 64, torch.float16)
    p.check(p.run(max_tokens=1))


def test_attention_empty_rows_and_requests():
    # lengths shorter than the rows (a refused request keeps its length), of zero, requests without rows
    p = Problem([3, 2, 0, 1, 4], [1, 0, 70, 64, 2], 2, 2, 64, torch.float16)
    out = p.run(max_tokens=4)
    p.check(out)
    assert not out[0].any() and not out[1].any() and out[2].any()  # [1 - 3 + i + 1] tokens seen
    assert not out[3:5].any()
    p.check(p.run(max_tokens=4, causal=False), causal=False)


def test_attention_rows_behind_the_last_request():
    p = Problem([2, 1], [40, 100], 2, 1, 128, torch.float16)
    q = torch.cat([p.q, torch.full((5, 2, 128), float("nan")).half()])
    out = p.run(q=q, max_tokens=2)
    p.check(out[:3])
    assert out.shape[0] == 8 and not out[3:].any()
    given = torch.full((8, 2, 128), 7.0, dtype=torch.float16, device="cuda")
    p.run(q=q, max_tokens=2, out=given)
    assert torch.equal(given[:3], out[:3]) and (given[3:] == 7).all()


def test_attention_of_nothing():
    p = Problem([], [], 2, 2, 64, torch.float16)
    assert p.run().shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, dtype=torch.float16)
    assert not p.run(q=q).any()


def test_attention_strided_rows_and_out():
    p = Problem([1, 4], [77, 130], 2, 2, 128, torch.bfloat16)
    want = p.run(max_tokens=4)
    wide = torch.zeros(5, 3, 4, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = p.q.cuda()
    out = torch.zeros(4, 5, 256, dtype=torch.bfloat16, device="cuda").transpose(0, 1)[..., :128]
    p.run(q=wide[:, 1], max_tokens=4, out=out)
    assert torch.equal(out, want)
    heads_first = p.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(p.run(q=heads_first, max_tokens=4), want)
    odd = torch.cat([torch.zeros(1, dtype=torch.bfloat16), p.q.flatten()]).cuda()[1:].view_as(p.q)
    assert torch.equal(p.run(q=odd, max_tokens=4), want)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_attention_scales(scale):
    p = Problem([1, 3], [90, 200], 1, 3, 64, torch.float16)
    p.check(p.run(max_tokens=3, scale=scale), scale=scale)


def test_attention_bf16_rows_of_any_size():
    p = Problem([4], [150], 1, 2, 64, torch.bfloat16)
    p.q[0] *= 2.0 ** 60
    p.q[1] *= 2.0 ** -100
    p.q[2] = 0
    p.q[3, :, ::2] *= 2.0 ** -30
    out = p.run(max_tokens=4, causal=False)
    # the first row's scores pick a single key
    k, v = p.k[0][:, 0].double(), p.v[0][:, 0].double()
    for h in range(2):
        best = (k @ p.q[0, h].double()).argmax()
        assert (out[0, h].cpu().double() - v[best]).abs().max() <= 2.0 ** -8 * v[best].abs().max()
    p.counts, p.query_start = [0, 3], [0, 1, 4]
    p.lengths, p.k, p.v = [0, 150], [p.k[0][:0], p.k[0]], [p.v[0][:0], p.v[0]]
    p.check(out, causal=False)


def test_attention_nan_and_infinite_queries_stay_in_their_rows():
    p = Problem([4], [100], 1, 2, 128, torch.float16)
    p.q[1, 0] = float("nan")
    p.q[2, 1, 5] = float("inf")
    out = p.run(max_tokens=4)
    assert out[1, 0].isnan().all() and out[2, 1].isnan().any()
    clean = torch.ones(4, 2, dtype=torch.bool)
    clean[1, 0] = clean[2, 1] = False
    p.q[~clean] = 0
    want = p.run(max_tokens=4)
    assert torch.equal(out.cpu()[clean], want.cpu()[clean])


def test_attention_bad_pages_take_no_part():
    p = Problem([1, 2], [200, 190], 2, 1, 64, torch.float16)
    p.tables[0][1] = -1          # tokens 64..127
    p.tables[1][0] = 10 ** 9     # tokens 0..63
    out = p.run(max_tokens=2)
    for r, gone in ((0, range(64, 128)), (1, range(0, 64))):
        keep = [i for i in range(p.lengths[r]) if i not in gone]
        p.k[r], p.v[r] = p.k[r][keep], p.v[r][keep]
        p.lengths[r] = len(keep)
    p.check(out)


def test_attention_survives_wild_index_tensors():
    p = Problem([1, 2], [100, 90], 1, 2, 64, torch.float16)
    kf, vf = p.factors()
    width = len(p.tables[0])
    for lengths, starts in (([2 ** 31 - 1, -5], [0, 1, 3]), ([100, 90], [-3, 2 ** 31 - 1, 3]), ([100, 90], [3, 2, 1])):
        out = g.attn_cache4(p.q.cuda(), p.cache, ints(p.tables), ints(lengths), ints(starts), p.scale, k_scale=kf, v_scale=vf)
        assert out.shape == p.q.shape and width
    p = Problem([100, 200], [100, 290], 1, 2, 128, torch.float16)
    for lengths, starts in (([2 ** 31 - 1, -5], [0, 100, 300]), ([100, 90], [-3, 2 ** 31 - 1, 3]),
                            ([100, 90], [300, 200, 100]), ([100, 290], [0, 300, 300]), ([100, 290], [250, 300, 2 ** 31 - 1])):
        out = g.attn_cache4(p.q.cuda(), p.cache, ints(p.tables), ints(lengths), ints(starts), p.scale)
        assert out.shape == p.q.shape
    # decreasing starts may make the requests' rows more than there are
    starts = [0, 300] * 50 + [0]
    out = g.attn_cache4(p.q.cuda(), p.cache, ints(p.tables[:1] * 100), ints([100] * 100), ints(starts), p.scale)
    torch.cuda.synchronize()


def test_attention_in_place():
    for counts in ([1, 2], [100, 2]):
        p = Problem(counts, [3000, 90], 2, 2, 64, torch.float16)
        want = p.run(max_tokens=max(counts))
        q = p.q.cuda()
        p.run(q=q, max_tokens=max(counts), out=q)
        assert torch.equal(q, want)


def test_attention_of_many_heads_on_one():
    p = Problem([1, 2], [700, 90], 1, 96, 64, torch.bfloat16)  # more rows of one token than the small kernel takes
    p.check(p.run(max_tokens=2))


def test_attention_is_deterministic_and_ignores_the_hint():
    p = Problem([1, 1, 2], [3000, 77, 1500], 2, 3, 128, torch.float16)
    a, b = p.run(max_tokens=2), p.run(max_tokens=2)
    assert torch.equal(a, b)
    for hint in (0, 1, 50, None):
        p.check(p.run(max_tokens=hint))


def test_attention_refusals():
    p = Problem([1, 2], [10, 20], 2, 2, 64, torch.float16)
    ok = dict(q=p.q.cuda(), cache=p.cache, tables=ints(p.tables), lengths=ints(p.lengths),
              query_start=ints(p.query_start), scale=0.125)
    g.attn_cache4(**ok)
    q = ok["q"]
    for bad in ({"q": q.float()}, {"q": q.cpu()}, {"q": q[0]}, {"q": q[:, :3]}, {"q": q[..., :32]},
                {"tables": ok["tables"].long()}, {"tables": ok["tables"][:1]}, {"lengths": ints([1])},
                {"query_start": ints([0, 1])}, {"query_start": ok["query_start"].cpu()}, {"scale": float("nan")},
                {"scale": 1e300}, {"max_tokens": -1}, {"out": q.float()}, {"out": q[:2]}, {"out": q.cpu()},
                {"out": torch.empty(3, 4, 128, dtype=torch.float16, device="cuda")[..., ::2]},
                {"out": torch.empty(1, 4, 64, dtype=torch.float16, device="cuda").expand(3, 4, 64)},
                {"k_scale": torch.ones(4, device="cuda")}, {"v_scale": torch.ones(2)},
                {"cache": p.cache.transpose(0, 1)}, {"cache": p.cache[..., :100].contiguous()}):
        with pytest.raises(RuntimeError):
            g.attn_cache4(**{**ok, **bad})


@pytest.mark.parametrize("counts", [[1, 1], [70, 1], [3, 300]])  # one kernel, both, both
def test_attention_on_other_streams_and_in_graphs(counts):
    p = Problem(counts, [5000, 300], 2, 4, 128, torch.float16)
    q2 = torch.randn(p.q.shape, generator=torch.Generator().manual_seed(9)).half()
    want, want2 = p.run(max_tokens=max(counts)), p.run(q=q2, max_tokens=max(counts))
    kf, vf = p.factors()
    fixed = (p.cache, ints(p.tables), ints(p.lengths), ints(p.query_start), p.scale)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    qs = [p.q.cuda(), q2.cuda()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):  # two calls at once, each on its own stream
        for i in range(2):
            with torch.cuda.stream(side[i]):
                outs[i].append(g.attn_cache4(qs[i], *fixed, k_scale=kf, v_scale=vf, max_tokens=max(counts)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs[0]) and all(torch.equal(o, want2) for o in outs[1])
    graphs, results = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(g.attn_cache4(qs[i], *fixed, k_scale=kf, v_scale=vf, max_tokens=max(counts)))
        graphs.append(graph)
    for _ in range(3):
        results[0].zero_()
        results[1].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(results[0], want) and torch.equal(results[1], want2)


def test_offsets_past_32_bits():
    H, D, pages = 16, 128, 18000  # 2.65 GB
    cache = torch.zeros(pages, H, 72 * D, dtype=torch.uint8, device="cuda")
    table = [pages - 1, 17000, 3]
    slots = ints([table[i // 64] * 64 + i % 64 for i in range(150)])
    k = torch.randn(150, H, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    g.cache4_write(k, -k, cache, slots)
    small = g.cache4_alloc(3, H, D)
    g.cache4_write(k, -k, small, ints(range(150)))
    for a, b in zip(g.cache4_read(cache, slots), g.cache4_read(small, ints(range(150)))):
        assert torch.equal(a, b)
    q = k[:1].contiguous()
    args = (ints([150]), ints([0, 1]), 0.1)
    assert torch.equal(g.attn_cache4(q, cache, ints([table]), *args), g.attn_cache4(q, small, ints([[0, 1, 2]]), *args))


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("graph", [False, True])
def test_generation_of_a_batch(graph):
    """Prompts, then token after token, with requests that end and others that take their pages: every
    step's attention against the keys and values that were written."""
    H, group, D, R, width, tokens = 2, 2, 64, 4, 6, 64
    rng, gen = random.Random(0), torch.Generator().manual_seed(0)
    tables, lengths = torch.zeros(R, width, dtype=torch.int32, device="cuda"), ints([0] * R)
    free_pages, free_count, counts = ints(list(range(12)) + [0] * 4), ints([12]), ints([0] * R)
    cache = torch.full((12, H, 72 * D), 255, dtype=torch.uint8, device="cuda")
    q, k, v = (torch.zeros(tokens, h, D, dtype=torch.float16, device="cuda") for h in (H * group, H, H))
    kf, vf = torch.tensor([0.5, 2.0], device="cuda"), torch.tensor([1.0, 0.25], device="cuda")

    def step():
        plan = g.cache4_plan(tables, lengths, counts, free_pages, free_count, tokens)
        g.cache4_write(k, v, cache, plan.slots, kf, vf)
        out = g.attn_cache4(q, cache, tables, plan.lengths, plan.query_start, 0.2, k_scale=kf, v_scale=vf)
        lengths.copy_(plan.lengths)
        free_count.copy_(plan.free_count)
        return plan, out

    captured = None
    past = [([], []) for _ in range(R)]
    for turn in range(14):
        n = [rng.choice([1, 1, 1, 17, -1]) if past[r][0] else rng.randint(1, 20) for r in range(R)]
        counts.copy_(ints(n))
        q.copy_(torch.randn(q.shape, generator=gen))
        k.copy_(torch.randn(k.shape, generator=gen))
        v.copy_(torch.randn(v.shape, generator=gen))
        if graph:
            if captured is None:
                captured = torch.cuda.CUDAGraph()
                saved = lengths.clone(), free_count.clone(), tables.clone(), free_pages.clone(), cache.clone()
                with torch.cuda.graph(captured):
                    plan, out = step()
                for t, s in zip((lengths, free_count, tables, free_pages, cache), saved):
                    t.copy_(s)
            captured.replay()
        else:
            plan, out = step()
        kq, vq = (torch.from_numpy(oracle.numbers(*oracle.quantise(x.cpu(), f.cpu().numpy()), f.cpu().numpy()))
                  for x, f in ((k, kf), (v, vf)))
        starts, added = plan.query_start.tolist(), plan.added.tolist()
        for r in range(R):
            if n[r] < 0:
                past[r] = ([], [])
                continue
            assert added[r] in (0, n[r])
            a = starts[r]
            past[r][0].extend(kq[a:a + added[r]])
            past[r][1].extend(vq[a:a + added[r]])
            if not added[r]:
                continue
            keys, values = torch.stack(past[r][0]), torch.stack(past[r][1])
            for h in range(H * group):
                ref, size = oracle.attention(q[a:a + n[r], h].cpu(), keys[:, h // group], values[:, h // group], 0.2, True)
                off = (out[a:a + n[r], h].cpu().double() - ref).abs()
                assert (off <= size * (2.0 ** -11 + 2.0 ** -12) + 2.0 ** -11 * ref.abs() * 1.01 + 1e-5).all(), (turn, r, h)
        held = sum(-(-len(x[0]) // 64) for x in past)
        assert int(free_count) == 12 - held and [len(x[0]) for x in past] == lengths.tolist()


def test_read_prefix_feeds_dense_attention():
    """Keys and values taken out of the cache give `attn` what attn_cache4 computes from it."""
    p = Problem([130], [300], 4, 1, 64, torch.float16)
    slots = ints([p.tables[0][i // 64] * 64 + i % 64 for i in range(300)])
    k, v = g.cache4_read(p.cache, slots, *p.factors())
    dense = g.attn(*(x.cuda().transpose(0, 1)[None] for x in (p.q, k, v)), p.scale)
    out = p.run(causal=False)
    # both round p and the output; the values read back are rounded to fp16 once more
    assert (dense[0].transpose(0, 1).float() - out.float()).abs().max() <= 4 * 2.0 ** -11 * float(p.v[0].abs().max())
