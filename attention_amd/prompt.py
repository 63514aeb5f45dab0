"""Prompts, and a paged K/V cache held in 8 bits.

    out = gqa_prefill(q, key, value, cu_seqlens)             # the prompts attend to themselves
    kv_append_q8(key, value, *cache, table, starts, cu_seqlens)
    ...
    kv_append_q8(key, value, *cache, table, positions)       # one token per sequence
    out = gqa_decode_q8(q, *cache, table, context_lens)

with ``cache = (k_cache, v_cache, k_scales, v_scales)``: caches ``[blocks,
block_size, Hkv, D]`` of ``torch.float8_e4m3fn`` or ``torch.int8``, and a
float32 scale per page and head, ``[blocks, Hkv]``; an element stands for itself
times its scale.  A later chunk of a prompt reads the cached tokens back with
:func:`kv_gather_q8` and attends with ``cu_seqlens_k``.

These have no counterpart in the reference; they forward to
``torch.ops.qd_serving.*`` of the in-tree HIP library.  There is no fallback, no
host synchronization and no gradient.  Metadata contents are caller-owned:
values out of range never leave a tensor.
"""
from __future__ import annotations

import math

import torch

from .core import _require_extension


def gqa_prefill(q, key, value, cu_seqlens, *, cu_seqlens_k=None, window=None, sinks=0, scale=None):
    """Causal attention over packed prompts.

    q ``[Tq, Hq, D]``, key and value ``[Tk, Hkv, D]``: tokens may lie any stride
    apart, as views of one projection's output do.  Sequence ``b`` has rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` of q (int32 ``[B + 1]``, the first 0)
    and of key and value, or there those of ``cu_seqlens_k``: its queries are then
    the last ones of its keys, query ``i`` of ``nq`` at position ``nk - nq + i``.  A
    query sees the keys up to its own position, or with ``window`` the last
    ``window`` of them and the first ``sinks`` of the sequence.  Returns ``[Tq, Hq,
    D]``; queries that see nothing, and rows behind the last sequence, give zeros.
    Sums are float32; float16 and bfloat16 round each softmax weight to the type
    once, where :func:`gqa_decode` keeps it in more bits.
    """
    _require_extension()
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if window is not None and window < 1:
        raise ValueError("window must be positive, or None")
    return torch.ops.qd_serving.gqa_prefill(q, key, value, cu_seqlens, cu_seqlens_k, float(scale), window or 0, sinks)


def kv_append_q8(key, value, k_cache, v_cache, k_scales, v_scales, block_table, positions, cu_seqlens=None):
    """Writes tokens to an 8-bit cache, in place.

    key and value ``[T, Hkv, D]`` (float32, float16 or bfloat16; tokens any stride
    apart).  Row ``cu_seqlens[b] + i`` becomes token ``positions[b] + i`` of sequence
    ``b`` (int32 ``[B]``); without ``cu_seqlens``, row ``b`` token ``positions[b]``.

    A page's scale of a head is the smallest power of two that holds its largest
    value: a page that the call begins takes the one of its new rows; one that it
    goes on with keeps the old one, or takes a larger one (in magnitude), and the rows
    before are rounded to it.  An Inf or NaN (or a scale past 2^100) makes the scale
    NaN, and with it every value of that page and head.  Sequences with a negative
    position write nothing, nor do tokens past the table or in pages outside the pool.
    Pages that are written to must be their sequence's own.
    """
    _require_extension()
    torch.ops.qd_serving.kv_append_q8(key, value, k_cache, v_cache, k_scales, v_scales, block_table, positions,
                                      cu_seqlens)


def kv_gather_q8(key, value, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, cu_seqlens):
    """Reads cached tokens back as packed rows: row ``cu_seqlens[b] + i`` of key and
    value ``[T, Hkv, D]`` becomes token ``i < context_lens[b]`` of sequence ``b``, in
    place.  Other rows are left as they were, such as those that hold a chunk's own
    tokens: with ``cu_seqlens`` over context and chunk, key and value are then what
    :func:`gqa_prefill` takes, with the same ``cu_seqlens_k``.
    """
    _require_extension()
    torch.ops.qd_serving.kv_gather_q8(key, value, k_cache, v_cache, k_scales, v_scales, block_table, context_lens,
                                      cu_seqlens)


def gqa_decode_q8(q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, *, scale=None):
    """:func:`gqa_decode` over an 8-bit cache: q ``[B, Hq, D]`` (float16 or
    bfloat16), scales of any magnitude from 2^-100 to 2^100, or 0.  Returns ``[B, Hq,
    D]``; a sequence of length 0 gives zeros.  Lengths are not read on the host: the
    width of ``block_table`` decides whether contexts may be split (with a second
    kernel that merges them), so trim it to the longest.  Sums are float32; weights
    times their values' scale are rounded to float16 once, and there is no ``window``
    as in :func:`gqa_decode_window`.
    """
    _require_extension()
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return torch.ops.qd_serving.gqa_decode_q8(q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens,
                                              float(scale))
