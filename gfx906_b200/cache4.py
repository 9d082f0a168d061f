"""A paged key/value cache held in 4 bits, and attention against it.

``gfx906_b200.attn`` attends to whole fp16 K and V. A program that generates
its positions a few at a time attends to a past instead, which these operators
keep in 4.5 bits a number:

* ``cache4_alloc`` makes the cache: pages of 64 tokens per kv head.
* ``cache4_plan`` does a step's page bookkeeping on the GPU, from the requests'
  lengths: which pages they get or return, and every new token's slot.
* ``cache4_write`` and ``cache4_read`` put keys and values into slots and take
  them out again (for ``attn`` on a prefix, or to move them elsewhere).
* ``attn_cache4`` is the attention of each request's new tokens against its
  pages, from one token to whole prompts.

A step of a generating program, all of it on the current stream and without
waiting for the GPU::

    plan = cache4_plan(tables, lengths, counts, free_pages, free_count, tokens)
    for layer in layers:
        q, k, v = layer.project(x, plan.positions)
        cache4_write(k, v, layer.cache, plan.slots, layer.k_scale, layer.v_scale)
        o = attn_cache4(q, layer.cache, tables, plan.lengths, plan.query_start, scale,
                        k_scale=layer.k_scale, v_scale=layer.v_scale, max_tokens=most)
    lengths, free_count = plan.lengths, plan.free_count

where ``most`` is the largest of the counts, which the program that sets them
knows.

A number is an e2m1 code times an e4m3 scale, shared by 16 neighbouring
channels of a token, times a float32 factor per kv head (``k_scale``,
``v_scale``, positive; 1 where they are None). The factor serves numbers whose scale
leaves e4m3's range: the largest magnitude of a head divided by 2688 keeps all
of it. The byte layout of a page is in ``csrc/cache4.cuh``.

Every operator raises RuntimeError on arguments it does not take, runs on its
tensors' device, and can be captured in a CUDA graph; like ``attn`` they record
no gradient. ``set_sm_limit`` does not hold for them: their blocks are many and
short, and go to any SM that is free. Index tensors are int32.
Page ids and slots come from device memory and are checked there: what lies
outside the cache is skipped.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

__all__ = ["Cache4Plan", "PAGE", "attn_cache4", "cache4_alloc", "cache4_plan", "cache4_read", "cache4_write"]

PAGE = 64  # tokens of a page

_READ_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class Cache4Plan(NamedTuple):
    """What ``cache4_plan`` found for a step: int32 CUDA tensors, parts of one allocation."""

    query_start: torch.Tensor  # [requests + 1] first token of each request in the packed batch, and their sum
    lengths: torch.Tensor      # [requests] tokens in the cache once the new ones are written
    added: torch.Tensor        # [requests] tokens appended (0: none, refused, or ended)
    slots: torch.Tensor        # [tokens] slot of each token, -1: none
    positions: torch.Tensor    # [tokens] position of each token in its request, -1: none
    free_count: torch.Tensor   # [1] free pages left


_loaded = None


def _module():
    """The operator module, or RuntimeError; kept, as these calls are as short as the look-up."""
    global _loaded
    if _loaded is None:
        from . import _module_or_raise

        _loaded = _module_or_raise()
    return _loaded


def cache4_alloc(pages, kv_heads, head_dim, device="cuda"):
    """A cache of ``pages`` pages for ``kv_heads`` heads of ``head_dim`` 64 or
    128: a uint8 tensor [pages, kv_heads, 72 * head_dim], zeroed."""
    if head_dim not in (64, 128):
        raise RuntimeError("cache4: head_dim must be 64 or 128")
    return torch.zeros(pages, kv_heads, 72 * head_dim, dtype=torch.uint8, device=device)


def cache4_plan(tables, lengths, counts, free_pages, free_count, tokens):
    """Page bookkeeping of one step; returns a ``Cache4Plan``.

    tables [requests, width]: the page ids of each request, one row each.
    lengths [requests]: tokens each holds. counts [requests]: tokens to append,
    or a negative number for a request that has ended. free_pages: a stack of
    page ids whose first free_count (a tensor [1]) are free; it has room for
    every page of the cache. tokens: size of the packed token buffer, at least
    the sum of the counts. A page belongs to one request at a time.

    Pages of ended requests go back first and may be granted in the same step.
    Then requests get pages in their order; one is refused -- ``added`` 0, slots
    -1, length unchanged -- when its tokens do not fit its row of tables, when
    they do not fit the buffer, or when the free pages do not cover it and all
    before it. Tokens in a page whose id is negative or beyond 2^25 - 1 get slot
    -1 as well.
    tables and free_pages are updated in place, only where the inputs do not
    use them: until lengths and free_count are replaced by the returned ones, a
    step may be planned again.
    """
    return Cache4Plan(*_module().cache4_plan(tables, lengths, counts, free_pages, free_count, int(tokens)))


def cache4_write(k, v, cache, slots, k_scale=None, v_scale=None):
    """Writes k and v [tokens, kv_heads, head_dim] (fp16 or bf16, any strides)
    into ``cache`` at ``slots`` [tokens], which are distinct; tokens with a slot
    outside the cache (-1) are skipped.

    Codes and scales are rounded to nearest even. The cache holds finite
    numbers only: infinities become the largest number of their head, NaN zero.
    """
    _module().cache4_write(k, v, cache, slots, k_scale, v_scale)


def cache4_read(cache, slots, k_scale=None, v_scale=None, dtype=torch.float16):
    """The keys and values at ``slots`` [tokens] as two contiguous tensors
    [tokens, kv_heads, head_dim] of fp16, bf16 or fp32; zeros where a slot lies
    outside the cache (-1). What a number was rounded up to in the cache may lie
    beyond fp16's range (6% at most for fp16 keys and values) and is then infinite."""
    if dtype not in _READ_DTYPES:
        raise RuntimeError("cache4: dtype must be float16, bfloat16 or float32")
    return _module().cache4_read(cache, slots, k_scale, v_scale, _READ_DTYPES[dtype])


def attn_cache4(q, cache, tables, lengths, query_start, scale, causal=True, k_scale=None, v_scale=None,
                max_tokens=None, out=None):
    """softmax(scale * q @ k^T) @ v of each request's rows of q against its
    tokens in the cache.

    q [tokens, heads, head_dim] is fp16 or bf16 with any strides; rows
    query_start[r] to query_start[r + 1] (which does not decrease; it starts at
    0) belong to request r, which attends to its first lengths[r] tokens in the
    pages tables[r]. heads is a multiple of
    the cache's kv heads; consecutive query heads share one. With ``causal`` a
    request's last row sees all its tokens and each row before it one token
    less; without, every row sees them all. Rows that see none are zero.

    max_tokens: no request has more rows than this, if known; it chooses the
    kernels (default: all rows of q may be one request's, which costs a step of
    64 single tokens half its time again). Too small a value costs time, not
    correctness.

    Scores, softmax sums and the output are held in 32 bits, and the output is
    rounded once. Weights are rounded to fp16 on their way to the tensor core:
    by 2^-11 of themselves down to 2^-21 of a row's largest, below that by 2^-32
    of it. Rows of bf16 go into fp16 divided by a power of two; their numbers
    below 2^-14 of the row's largest are rounded by up to 2^-25 of it. Returns a new tensor, with zeros in rows behind
    the last request, or ``out``, whose rows behind the last request are left
    as they were. ``out`` is q itself, or shares no row with q and no memory
    with the other arguments.
    """
    return _module().attn_cache4(q, cache, tables, lengths, query_start, float(scale), bool(causal), k_scale, v_scale,
                                 max_tokens, out)
