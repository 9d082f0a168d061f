"""The 4-bit cache without a GPU: its byte layout, its oracle's rounding, refusals of the C ABI."""

import ctypes
import re

import numpy as np
import pytest
import torch

from gfx906_b200 import build
from gfx906_b200.cabi import CABI, STATUS, Cache4AttnArgs
from oracle import cache4 as oracle

HEADER = build.INCLUDE / "gfx906_b200_cache4.h"


@pytest.fixture(scope="module")
def lib():
    return CABI(build.build_library())


@pytest.mark.parametrize("D", [64, 128])
def test_layout_covers_a_page_exactly_once(D):
    seen = np.zeros(72 * D, dtype=int)
    for which in (0, 1):
        for t in range(64):
            for d in range(0, D, 2):
                at, high = oracle.byte_of(which, t, d, D)
                other, other_high = oracle.byte_of(which, t, d + 1, D)
                assert at == other and not high and other_high
                seen[at] += 1
            for g in range(D // 16):
                seen[oracle.scale_byte_of(which, t, g, D)] += 1
    assert (seen == 1).all()


def test_oracle_rounds_as_the_types_do():
    values = oracle.e4m3_values()
    ref = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(values, ref, equal_nan=True)
    x = torch.rand(20000, generator=torch.Generator().manual_seed(0)) * 448
    x[:127] = torch.from_numpy(values[:127]).float()
    x[127:253] = (x[:126] + x[1:127]) / 2  # ties
    assert np.array_equal(oracle.to_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, np.inf])
    assert oracle.to_e2m1(ties).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7]
    assert oracle.to_e2m1(-ties).tolist() == [8, 10, 10, 12, 12, 14, 14, 15, 15]


def test_header_symbols_are_exported(lib):
    names = re.findall(r"^GFX906_B200_API\s+[\w\s\*]*?\b(\w+)\s*\(", HEADER.read_text(), re.M)
    assert len(names) == 6
    for name in names:
        assert hasattr(lib.dll, name), name


def test_page_bytes(lib):
    assert [lib.dll.gfx906_b200_cache4_page_bytes(d) for d in (64, 128, 96, 0, 512)] == [72 * 64, 72 * 128, 0, 0, 0]


P, BAD = 4096, 4096 + 4  # never dereferenced: these calls return before any launch


def test_plan_refusals(lib):
    def call(requests=1, width=4, size=8, tokens=4, tables=P, query_start=P, slots=P):
        return lib.dll.gfx906_b200_cache4_plan(tables, P, P, P, P, requests, width, size, tokens, query_start, P, P,
                                               slots, P, P, None)

    for kw in ({"requests": -1}, {"requests": 8193}, {"width": -1}, {"width": 2 ** 31 // 64}, {"size": -1},
               {"tokens": -1}, {"tables": None}, {"query_start": None}, {"slots": None},
               {"requests": 8192, "width": 2 ** 19}):
        assert call(**kw) == STATUS["EINVAL"], kw
        assert lib.last_error() == STATUS["EINVAL"]


def test_write_and_read_refusals(lib):
    def write(k=P, dtype=0, stride=128, tokens=4, heads=2, D=128, cache=P, pages=3, slots=P):
        return lib.dll.gfx906_b200_cache4_write(k, P, dtype, stride, 128, 256, 128, tokens, heads, D, cache, pages,
                                                slots, None, None, None)

    def read(cache=P, dtype=0, tokens=4, heads=2, D=128, k=P, slots=P, pages=3):
        return lib.dll.gfx906_b200_cache4_read(cache, pages, slots, None, None, tokens, heads, D, k, P, dtype, None)

    for call in (write, read):
        assert call(D=96) == STATUS["EHEADDIM"]
        for kw in ({"dtype": -1}, {"dtype": 3}, {"tokens": -1}, {"heads": -1}, {"pages": -1}, {"k": None},
                   {"cache": None}, {"slots": None}):
            assert call(**kw) == STATUS["EINVAL"], (call, kw)
        assert call(k=BAD) == STATUS["EALIGN"] and call(cache=BAD) == STATUS["EALIGN"]
        assert call(tokens=0) == STATUS["OK"] and call(heads=0) == STATUS["OK"]
    assert write(dtype=2) == STATUS["EINVAL"] and write(stride=129) == STATUS["EALIGN"]
    assert write(pages=0) == STATUS["OK"]


def attn_args(**kw):
    a = Cache4AttnArgs(q=P, o=P, cache=P, tables=P, lengths=P, query_start=P, q_stride_t=256, q_stride_h=128,
                       o_stride_t=256, o_stride_h=128, dtype=0, tokens=3, heads=2, kv_heads=1, D=128, pages=2,
                       requests=1, width=2, max_tokens=3, causal=1, zero_rest=0, scale=0.1)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_attention_refusals(lib):
    def call(**kw):
        return lib.dll.gfx906_b200_cache4_attn(ctypes.byref(attn_args(**kw)), P, 0, None)

    assert lib.dll.gfx906_b200_cache4_attn(None, P, 0, None) == STATUS["EINVAL"]
    assert call(D=96) == STATUS["EHEADDIM"]
    for kw in ({"dtype": 2}, {"tokens": -1}, {"heads": 3, "kv_heads": 2}, {"kv_heads": 0}, {"requests": 8193},
               {"requests": -1}, {"width": -1}, {"width": 2 ** 31 // 64}, {"pages": -1}, {"max_tokens": -1},
               {"scale": float("inf")}, {"scale": float("nan")}, {"q": None}, {"o": None}, {"cache": None},
               {"tables": None}, {"lengths": None}, {"query_start": None},
               {"tokens": 2 ** 30, "heads": 8, "kv_heads": 1}):
        assert call(**kw) == STATUS["EINVAL"], kw
    for kw in ({"q": BAD}, {"o": BAD}, {"cache": BAD}, {"q_stride_t": 257}, {"o_stride_h": 4}):
        assert call(**kw) == STATUS["EALIGN"], kw
    assert call(tokens=0) == STATUS["OK"]
    assert lib.dll.gfx906_b200_cache4_attn_workspace_size(ctypes.byref(attn_args(D=96))) == 0


def test_operators_are_public_and_refuse_without_a_gpu():
    import gfx906_b200

    for name in ("cache4_alloc", "cache4_plan", "cache4_write", "cache4_read", "attn_cache4", "Cache4Plan"):
        assert name in gfx906_b200.__all__ and hasattr(gfx906_b200, name)
    with pytest.raises(RuntimeError, match="head_dim"):
        gfx906_b200.cache4_alloc(4, 2, 96, device="cpu")
    assert gfx906_b200.cache4_alloc(4, 2, 64, device="cpu").shape == (4, 2, 72 * 64)


def test_oracle_plan_grants_in_order_and_returns_first():
    got = oracle.plan([[5, 6, -1], [7, -1, -1], [-1, -1, -1]], [70, 64, 0], [-1, 1, 130], [0, 0, 0, 0, 0, 0], 0, 131)
    # pages 5 and 6 come back; request 1 gets the top one, request 2 needs three and is refused
    assert got["added"] == [0, 1, 0] and got["lengths"] == [0, 65, 0] and got["free_count"] == 1
    assert got["tables"][1][:2] == [7, 6] and got["slots"][0] == 6 * 64 and set(got["slots"][1:]) == {-1}


def test_torch_operators_refuse_host_tensors():
    from gfx906_b200 import gfx906_attn

    build.build_extension()
    mod = gfx906_attn.import_extension()
    i = torch.zeros(2, dtype=torch.int32)
    x, cache = torch.zeros(2, 1, 64).half(), torch.zeros(1, 1, 72 * 64, dtype=torch.uint8)
    for call in (lambda: mod.cache4_plan(i[None], i[:1], i[:1], i, i[:1], 1),
                 lambda: mod.cache4_write(x, x, cache, i, None, None), lambda: mod.cache4_read(cache, i, None, None, 0),
                 lambda: mod.attn_cache4(x, cache, i[None], i[:1], i, 0.1, True, None, None, None, None)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
