"""The paged 4-bit cache at the edges of its numbers, sizes and memory (needs a B200)."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

import gfx906_b200 as g
from gfx906_b200 import build
from gfx906_b200.cabi import CABI, STATUS, Cache4AttnArgs
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


def held(k, v, pages=None):
    """k and v [n, heads, D] in a cache of their own, in order: (cache, table, what it holds of k and v in 32 bits)."""
    n, heads, D = k.shape
    need = -(-n // 64)
    cache = g.cache4_alloc(pages or need, heads, D)
    slots = ints(range(n))
    g.cache4_write(k.cuda(), v.cuda(), cache, slots)
    k, v = g.cache4_read(cache, slots, dtype=torch.float32)
    return cache, ints([list(range(need))]), k.cpu(), v.cpu()


# rows of one request: the small kernel in both its instances, the large one (two tiles of rows)
@pytest.mark.parametrize("rows", [1, 12, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nats", [9.0, 14.0, 18.0])
def test_small_weights_beside_large_ones(nats, dtype, D, rows):
    """One key in 32 outweighs the others by far and has values of zero: all of the output comes from small weights."""
    n, gen = 1600, torch.Generator().manual_seed(1)
    k = torch.zeros(n, 1, D)
    k[5::32, 0, 0] = 6.0
    v = 1.0 + 0.25 * torch.randn(n, 1, D, generator=gen)
    v[5::32] = 0
    cache, table, k, v = held(k.half(), v.half())
    q = torch.zeros(rows, 1, D)
    q[:, 0, 0] = 2.0
    scale = nats / 12
    # a factor that brings the output to fp16's normal range
    out = g.attn_cache4(q.to(dtype).cuda(), cache, table, ints([n]), ints([0, rows]), scale, causal=False,
                        v_scale=torch.tensor([2.0 ** 14], device="cuda"), max_tokens=rows).cpu()
    v = v[:, 0] * 2.0 ** 14
    ref, size = oracle.attention(q[:1, 0], k[:, 0], v, scale, False)
    # Of each weight p (the largest 1): 2^-11 of itself for its rounding to fp16, and 2^-12 for 32-bit scores and
    # exponentials; where it is below 2^-21, 2^-32. Then one rounding of the output.
    total = float(torch.softmax(scale * (k[:, 0].double() @ q[0, 0].double()), 0).max()) ** -1
    tol = size * (2.0 ** -11 + 2.0 ** -12) + n * 2.0 ** -32 * float(v.abs().max()) / total \
        + HALF_STEP[dtype] * ref.abs() * 1.01 + 2.0 ** -25
    off = (out[:, 0].double() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert float(tol.max() / ref.abs().min()) < 0.05  # the bound is a bound


# 600 requests of one row over the same pages: pieces of all lengths; one request of many rows: the large kernel
@pytest.mark.parametrize("requests,rows", [(600, 1), (1, 200)])
@pytest.mark.parametrize("size", [8, 20, 23, 28, 60, 100])
def test_equal_keys_weigh_the_same_however_large_their_scores(size, requests, rows):
    """Two equal keys, in different steps, lead all others by far: the output is the mean of their values, which is
    exact in 32 bits but for the weights' own rounding, the same for both; then one rounding of the output."""
    n, D = 256, 64
    k, v = torch.zeros(n, 1, D), torch.randn(n, 1, D, generator=torch.Generator().manual_seed(2))
    k[3, 0, 0] = k[3 + 128, 0, 0] = 6.0
    k[:, 0, 1] = -1.0
    cache, table, k, v = held(k.half(), v.half())
    q = torch.zeros(requests * rows, 1, D, dtype=torch.bfloat16)
    q[:, 0, 0] = 2.0 ** size
    args = (cache, table.expand(requests, -1).contiguous(), ints([n] * requests), ints(range(0, requests * rows + 1, rows)))
    want = ((v[3, 0].double() + v[3 + 128, 0].double()) / 2).expand(requests * rows, -1)
    for scale in (0.1, 0.77, 1 / 3):
        out = g.attn_cache4(q.cuda(), *args, scale, causal=False, max_tokens=rows)[:, 0].cpu().double()
        tol = HALF_STEP[torch.bfloat16] * 1.01 * want.abs() + 2.0 ** -20 * v.abs().max()
        off = (out - want).abs()
        assert (off <= tol).all(), (scale, float((off / tol).max()))


@pytest.mark.parametrize("page", [-1, -2 ** 25 - 3, -2 ** 31, 2 ** 25, 2 ** 25 + 1, 2 ** 26 + 2, 2 ** 31 - 1])
def test_plan_gives_no_slot_for_page_ids_beyond_slots(page):
    """An id whose slots have no 31 bits must not come out as the slot of another page, granted or held already."""
    held_by, free = [[page, 5, -1], [6, -1, -1]], [page, 9, page]
    tables, free_pages = ints(held_by), ints(free)
    plan = g.cache4_plan(tables, ints([64 + 60, 10]), ints([8, 64]), free_pages, ints([3]), 80)
    want = oracle.plan(held_by, [64 + 60, 10], [8, 64], free, 3, 80)
    assert plan.slots.tolist() == want["slots"] and plan.positions.tolist() == want["positions"]
    assert plan.added.tolist() == [8, 64] and tables.tolist() == want["tables"]
    # request 0: four tokens in page 5, four in the page granted first; request 1: 54 tokens in page 6, ten in page 9
    assert want["slots"] == [5 * 64 + 60 + i for i in range(4)] + [-1] * 4 \
        + [6 * 64 + 10 + i for i in range(54)] + [9 * 64 + i for i in range(10)] + [-1] * 8
    plan = g.cache4_plan(ints([[page]]), ints([3]), ints([2]), free_pages, ints([0]), 2)
    assert plan.slots.tolist() == [-1, -1] and plan.positions.tolist() == [3, 4]
    k = torch.ones(2, 1, 64, dtype=torch.float16, device="cuda")
    cache = g.cache4_alloc(4, 1, 64)
    g.cache4_write(k, k, cache, plan.slots)
    assert not cache.any()


def test_plan_of_the_largest_token_buffer():
    """Buffers near 2^31 tokens: every token behind the last is marked, none beyond the buffer is touched."""
    tokens = 2 ** 31 - 2
    plan = g.cache4_plan(ints([[0, 1]]), ints([3]), ints([5]), ints([2, 3]), ints([2]), tokens)
    assert plan.slots[:6].tolist() == [3, 4, 5, 6, 7, -1] and plan.free_count.item() == 2
    for x in (plan.slots, plan.positions):
        assert x.shape == (tokens,) and int(x[5:].max()) == -1 and int(x[5:].min()) == -1
    del plan, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [1, 32, 33, 100, 127, 128, 300])
def test_attention_without_requests(tokens):
    """No request, a token buffer of any size: zeros, or `out` as it was."""
    cache = g.cache4_alloc(2, 2, 64)
    q = torch.ones(tokens, 4, 64, dtype=torch.float16, device="cuda")
    for tables in (ints([]).reshape(0, 3), ints([]).reshape(0, 0)):
        args = (cache, tables, ints([]), ints([0]), 0.1)
        assert not g.attn_cache4(q, *args).any()
        out = torch.full_like(q, 7.0)
        g.attn_cache4(q, *args, out=out)
        assert (out == 7).all()


def check_rows(out, q, k, v, scale, causal, rows, heads, group):
    """Rows of one request of n = len(out) tokens: p's rounding and 32-bit scores, and one rounding of the output."""
    n, length = len(out), len(k)
    for i in rows:
        last = length - n + i + 1 if causal else length
        for h in heads:
            ref, size = oracle.attention(q[i, h][None], k[:last, h // group], v[:last, h // group], scale, False)
            tol = size * (2.0 ** -11 + 2.0 ** -12) + HALF_STEP[out.dtype] * ref.abs() * 1.01 \
                + last * 2.0 ** -32 * float(v.abs().max()) + 2.0 ** -25
            off = (out[i, h].cpu().double() - ref[0]).abs()
            assert (off <= tol[0]).all(), (i, h, float((off / tol[0]).max()))


@pytest.mark.parametrize("rows,length", [(1, 5000), (1, 31), (13, 1999), (60, 700)])
def test_attention_with_the_widest_table(rows, length):
    """A table of 2^25 - 1 pages, of which few are used: the call's size is that of the lengths."""
    H, D, width = 32, 64, 2 ** 25 - 1
    gen = torch.Generator().manual_seed(4)
    cache, table, k, v = held(*(torch.randn(length, H, D, generator=gen).half() for _ in range(2)))
    wide = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = torch.randn(rows, H, D, generator=gen).half()
    out = g.attn_cache4(q.cuda(), cache, wide, ints([length]), ints([0, rows]), 0.125, max_tokens=rows)
    check_rows(out, q, k, v, 0.125, True, range(0, rows, 7), [0, 1, 30, 31], 1)


@pytest.mark.parametrize("hint", [None, 1])
def test_attention_of_many_requests_with_wide_tables(hint):
    """4096 requests, 32 heads, room for 131072 tokens each."""
    R, H, D, width = 4096, 32, 64, 2048
    gen = torch.Generator().manual_seed(5)
    cache, table, k, v = held(*(torch.randn(300, H, D, generator=gen).half() for _ in range(2)))
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    tables[:, :table.shape[1]] = table
    lengths = [1 + 37 * r % 300 for r in range(R)]
    q = torch.randn(R, H, D, generator=gen).half()
    out = g.attn_cache4(q.cuda(), cache, tables, ints(lengths), ints(range(R + 1)), 0.125, max_tokens=hint)
    for r in (0, 1, 63, 64, 1000, 4095):
        check_rows(out[r:r + 1], q[r:r + 1], k[:lengths[r]], v[:lengths[r]], 0.125, True, [0], [0, 13, 31], 1)


def c_call(q, out, cache, tables, lengths, query_start, scale, causal=True, workspace=None):
    """(run, workspace) of one attention call through the C ABI on the current stream, which `run` launches."""
    lib = CABI(build.LIB_PATH)
    a = Cache4AttnArgs(q=q.data_ptr(), o=out.data_ptr(), cache=cache.data_ptr(), tables=tables.data_ptr(),
                       lengths=lengths.data_ptr(), query_start=query_start.data_ptr(), q_stride_t=q.stride(0),
                       q_stride_h=q.stride(1), o_stride_t=out.stride(0), o_stride_h=out.stride(1),
                       dtype=int(q.dtype == torch.bfloat16), tokens=q.shape[0], heads=q.shape[1],
                       kv_heads=cache.shape[1], D=q.shape[2], pages=cache.shape[0], requests=tables.shape[0],
                       width=tables.shape[1], max_tokens=q.shape[0], causal=int(causal), zero_rest=1, scale=scale)
    bytes_ = lib.dll.gfx906_b200_cache4_attn_workspace_size(ctypes.byref(a))
    ws = torch.empty(bytes_, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    assert ws.numel() == bytes_ and ws.data_ptr() % 256 == 0

    def run():
        rc = lib.dll.gfx906_b200_cache4_attn(ctypes.byref(a), ws.data_ptr(), ws.numel(),
                                             torch.cuda.current_stream().cuda_stream)
        assert rc == STATUS["OK"]
    return run, ws


def test_no_count_of_a_launch_is_left_for_its_replay():
    """Pieces of many rows are counted in the workspace's last words, two to an SM, under the launch's tag, which a
    replayed graph keeps. A CTA whose wait runs out marks its unit's word (bit 15): that unit is not joined, and the
    next replay finds nothing of it."""
    n, rows, gen = 4500, 600, torch.Generator().manual_seed(6)
    cache, table, k, v = held(*(torch.randn(n, 1, 64, generator=gen).half() for _ in range(2)))
    q = torch.randn(rows, 1, 64, generator=gen).half().cuda()
    args = (cache, table, ints([n]), ints([0, rows]), 0.125)
    want, out = g.attn_cache4(q, *args), torch.empty_like(q)
    run, ws = c_call(q, out, *args)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    words = ws[-(-(-16 * sms // 256) * 256):].view(torch.int64)[:2 * sms]  # the region is a multiple of 256 bytes
    ws.fill_(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lost in (None, 0, None, 3, None, None):
        if lost is not None:
            assert words[lost]  # tagged by the launch before
            words[lost] |= 0x8000
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert not (words & 0xffff).any()
        stored = (out == want).flatten(1).all(1)
        if lost is None:
            assert stored.all()
        else:  # one tile of 128 rows of a unit of 256, as it was
            assert int((~stored).sum()) in (128, rows % 256 % 128) and (out[~stored] == 7).all()


SHORT_WAITS = """
import torch, gfx906_b200 as g
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
cache = g.cache4_alloc(40, 1, 128)
k = torch.randn(2500, 1, 128, device="cuda").half()
g.cache4_write(k, k, cache, ints(range(2500)))
for rows in (1, 9, 400):
    q = torch.randn(rows, 1, 128, device="cuda").half()
    args = (cache, ints([list(range(40))]), ints([2500]), ints([0, rows]), 0.1)
    a, b = g.attn_cache4(q, *args, max_tokens=rows), g.attn_cache4(q, *args, max_tokens=rows)
    assert torch.equal(a, b) and a.isfinite().all() and a.any()
assert g.device_status() == 0
print("done")
"""


def test_attention_under_a_short_wait_limit():
    """No wait of a sound call comes near 20 milliseconds; a copy that did run out is waited for longer than that
    before its block ends."""
    got = subprocess.run([sys.executable, "-c", SHORT_WAITS], capture_output=True, text=True, timeout=120,
                         cwd=build.PKG_DIR.parent, env={**os.environ, "GFX906_B200_WAIT_TIMEOUT_MS": "20"})
    assert got.returncode == 0 and "done" in got.stdout, got.stderr


@pytest.mark.parametrize("rows", [1, 65])
def test_attention_to_the_longest_context(rows):
    """2^31 - 64 tokens, the most that a table can hold: all in one page but for the last 64, which outweigh them."""
    k, v = torch.zeros(128, 1, 64), torch.ones(128, 1, 64)
    k[64:, 0, 0], v[64:] = 6.0, 3.0
    cache, _, k, v = held(k.half(), v.half())
    tables = torch.zeros(1, 2 ** 25 - 1, dtype=torch.int32, device="cuda")
    tables[0, -1] = 1
    q = torch.zeros(rows, 1, 64, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 20.0
    out = g.attn_cache4(q, cache, tables, ints([2 ** 31 - 64]), ints([0, rows]), 0.5, causal=False, max_tokens=rows)
    assert (out == float(v[64, 0, 0])).all()  # the others weigh 2^31 e^-60 together


@pytest.mark.parametrize("tokens,heads", [(5, 1), (1, 3), (1, 1)])
def test_dimensions_of_one_entry_may_have_any_stride(tokens, heads):
    gen = torch.Generator().manual_seed(7)
    plain = [torch.randn(tokens, heads, 64, generator=gen).half().cuda() for _ in range(3)]
    if heads == 1:  # [tokens, 64, 1] seen as [tokens, 1, 64]: a stride of one from head to head
        odd = [x.transpose(1, 2).contiguous().transpose(1, 2).as_strided((tokens, 1, 64), (64, 1, 1)) for x in plain]
    else:  # [heads, 64, 1] seen as [1, heads, 64]: a stride of one from token to token
        odd = [x.as_strided((1, heads, 64), (1, 64, 1)) for x in plain]
    late = []  # the same, starting off 16 bytes
    for x in odd:
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].as_strided(x.shape, x.stride())
        late.append(y.copy_(x))
    slots, tables = ints(range(tokens)), ints([[0]])
    want = g.cache4_alloc(1, heads, 64)
    g.cache4_write(plain[0], plain[1], want, slots)
    args = (tables, ints([tokens]), ints([0, tokens]), 0.2)
    o = g.attn_cache4(plain[2], want, *args)
    for k, v, q in (odd, late):
        assert k.is_contiguous() and 1 in k.stride()[:2]
        cache = g.cache4_alloc(1, heads, 64)
        g.cache4_write(k, v, cache, slots)
        assert torch.equal(cache, want)
        assert torch.equal(g.attn_cache4(q, cache, *args), o)
    out = torch.zeros_like(o).as_strided(odd[2].shape, odd[2].stride())
    g.attn_cache4(odd[2], want, *args, out=out)
    assert torch.equal(out, o)


def test_out_shares_no_row_with_other_rows_of_q():
    T, H, D, gen = 6, 6, 64, torch.Generator().manual_seed(8)
    cache, table, _, _ = held(*(torch.randn(300, H, D, generator=gen).half() for _ in range(2)))
    q = torch.randn(T, H, D, generator=gen).half().cuda()
    args = (cache, table, ints([300]), ints([0, T]), 0.2)
    want = g.attn_cache4(q, *args)
    row = H * D
    memory = torch.empty(4 * T * row, dtype=torch.float16, device="cuda")

    def view(at, step_t, step_h):
        return memory.as_strided((T, H, D), (step_t, step_h, 1), at)

    fine = [(view(0, row, D), view(0, row, D)),                       # in place
            (view(0, row, D), view(T * row, row, D)),                 # one behind the other
            (view(row, 3 * row, D), view(0, 3 * row, D)),             # parts of a fused projection
            (view(0, 2 * row, 2 * D), view(D, 2 * row, 2 * D)),       # head by head
            (view(0, D, T * D), view(T * row, row, D)),               # two orders, apart
            (view(0, 2 * row, D), view(row, D, 2 * row)),             # two orders, interleaved
            (view(0, 4 * row, D), view(row + 8, 4 * row, D))]
    for x, out in fine:
        memory.zero_()
        x.copy_(q)
        g.attn_cache4(x, *args, out=out)
        assert torch.equal(out, want)
    bad = [(view(0, row, D), view(row, row, D)),                      # one token on
           (view(row, row, D), view(0, row, D)),
           (view(0, row, D), view(D, row, D)),                        # one head on
           (view(0, row, D), view(8, row, D)),                        # a part of a row
           (view(0, row, D), view((T - 1) * row + (H - 1) * D, row, D)),  # the last row alone
           (view(0, row, D), view(0, D, T * D)),                      # the same rows in another order
           (view(0, row, D), view(0, 2 * row, D)),
           (view(0, 2 * row, D), view(row - 8, D, 2 * row)),
           (view(0, row, D), view(3 * T * row // 2, D, D)),           # rows of out on top of each other
           (view(0, row, D), view(3 * T * row // 2, 0, D)),
           (view(0, row, D), view(3 * T * row // 2, 5 * D, D)),
           (view(0, row, D), view(3 * T * row // 2, D, 8))]
    for x, out in bad:
        with pytest.raises(RuntimeError, match="rows of its own"):
            g.attn_cache4(x, *args, out=out)
    # rows that the kernels cannot load are copied first, and out may be where they were
    spread = memory[:T * row * 2].view(T, H, D, 2)[..., 0]
    spread.copy_(q)
    out = view(0, row, D)
    g.attn_cache4(spread, *args, out=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_keys_and_values_read_have_memory_of_their_own(dtype):
    cache, _, _, _ = held(*(torch.randn(7, 3, 64).half() for _ in range(2)))
    for x in g.cache4_read(cache, ints(range(7)), dtype=dtype):
        assert x.untyped_storage().nbytes() == 7 * 3 * 64 * dtype.itemsize and x.storage_offset() == 0


@pytest.mark.parametrize("requests,heads", [(1, 1), (1, 7), (30, 5), (49, 3), (21, 7), (100, 4)])
def test_workspace_is_bounded_and_kept_to(requests, heads):
    """Units of many rows that are cut in 2 to 16 pieces: at most three pieces an SM, 256 rows of sums each."""
    n, rows, D, gen = 2300, 70, 128, torch.Generator().manual_seed(9)
    cache, table, _, _ = held(*(torch.randn(n, heads, D, generator=gen).half() for _ in range(2)))
    q = torch.randn(requests * rows, heads, D, generator=gen).half().cuda()
    args = (cache, table.expand(requests, -1).contiguous(), ints([n - 13 * r for r in range(requests)]),
            ints(range(0, requests * rows + 1, rows)), 0.09)
    want, out = g.attn_cache4(q, *args), torch.empty_like(q)
    run, ws = c_call(q, out, *args)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    few = sms * 3 * 2 * 16 * (D + 2) * 4  # sums of the other kernel's pieces: 16 rows, two a block
    assert ws.numel() <= 3 * sms * 256 * (D + 2) * 4 + few + 65536
    memory = torch.full((ws.numel() + 2 ** 20,), 0xa5, dtype=torch.uint8, device="cuda")
    run, _ = c_call(q, out, *args, workspace=memory[:ws.numel()])
    run()
    assert torch.equal(out, want) and (memory[ws.numel():] == 0xa5).all()


def test_calls_without_a_hint_are_sized_by_the_rows_there_are():
    """64 rows of four heads make three requests of more than 64 rows at most: four units, 16 pieces of each."""
    cache, table, _, _ = held(*(torch.randn(100, 1, 128).half() for _ in range(2)))
    q = torch.randn(64, 4, 128).half().cuda()
    args = (cache, table.expand(64, -1).contiguous(), ints([100] * 64), ints(range(65)), 0.09)
    out = torch.empty_like(q)
    run, ws = c_call(q, out, *args)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert ws.numel() <= 4 * 16 * 256 * (128 + 2) * 4 + sms * 3 * 2 * 16 * (128 + 2) * 4 + 65536
    run()
    assert torch.equal(out, g.attn_cache4(q, *args))


@pytest.mark.parametrize("rows", [1, 12, 130])
@pytest.mark.parametrize("power", [127, 126, -125, -126, -127, -130])
def test_the_largest_and_smallest_rows_of_bf16(power, rows):
    """Rows whose largest number is next to bf16's largest, or subnormal, under a factor that makes up for it."""
    n, D, gen = 300, 64, torch.Generator().manual_seed(10)
    cache, table, k, v = held(*(torch.randn(n, 1, D, generator=gen).half() for _ in range(2)))
    factor = 2.0 ** (-power if power > 0 else min(-power, 127))
    x = torch.randn(rows, 1, D, generator=gen)
    x = (x / x.abs().amax(-1, keepdim=True) * 1.9 * 2.0 ** power).to(torch.bfloat16)
    assert x.isfinite().all() and x.any()
    out = g.attn_cache4(x.cuda(), cache, table, ints([n]), ints([0, rows]), 1.0, causal=False, max_tokens=rows,
                        k_scale=torch.tensor([factor], device="cuda"))
    check_rows(out, x.double() * factor, k, v, 1.0, False, range(0, rows, 9), [0], 1)


@pytest.mark.parametrize("sms", [1, 2, 7, 147])
def test_attention_planned_for_fewer_sms(sms):
    """A cap on the SMs of other kernels changes how the work is cut, not what comes out."""
    n, H, D, gen = 1500, 2, 64, torch.Generator().manual_seed(11)
    cache, table, k, v = held(*(torch.randn(n, H, D, generator=gen).half() for _ in range(2)))
    counts = [1, 150, 0, 3, 300, 1]
    starts = [sum(counts[:r]) for r in range(len(counts) + 1)]
    lengths = [1500, 1400, 5, 3, 900, 0]
    q = torch.randn(starts[-1], H, D, generator=gen).half()
    with g.sm_limit(sms):
        out = g.attn_cache4(q.cuda(), cache, table.expand(len(counts), -1).contiguous(), ints(lengths), ints(starts), 0.125)
    for r, c in enumerate(counts):
        rows = [i for i in (0, 1, 2, 77, 128, 149, 255, 256, 299) if i < c]
        if lengths[r]:
            check_rows(out[starts[r]:starts[r + 1]], q[starts[r]:starts[r + 1]], k[:lengths[r]], v[:lengths[r]], 0.125, True,
                       rows, range(H), 1)
        else:
            assert not out[starts[r]:starts[r + 1]].any()
