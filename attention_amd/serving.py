"""One decoding step with drafted tokens, or with a sliding window, on the
paged K/V cache of :func:`attention_amd.gqa_decode`.

    q = qk_norm_rope_write(q, key, value, ...)     # norms, rotation, cache write
    out = gqa_decode_tree(q, k_cache, ...)         # the drafted tokens attend
    kv_compact(caches, ...)                        # accepted rows move up

These have no counterpart in the reference; they forward to
``torch.ops.qd_serving.*`` of the in-tree HIP library.  There is no fallback,
no host synchronization and no gradient.  Metadata contents are caller-owned,
as for ``gqa_decode``.
"""
from __future__ import annotations

import math

import torch

from .core import _require_extension


def gqa_decode_window(q, k_cache, v_cache, block_table, context_lens, *, window, sinks=0, scale=None):
    """:func:`gqa_decode` over the last ``window`` tokens of each sequence
    (the current one among them) and its first ``sinks`` ones.

    q ``[B, Hq, D]``; caches ``[blocks, block_size, Hkv, D]``; int32
    ``block_table [B, max_pages]`` and ``context_lens [B]``.  Table entries of
    pages whose tokens are all out of sight are never read: the pages may have
    been freed.  Returns ``[B, Hq, D]``; a sequence of length 0 gives zeros.
    """
    _require_extension()
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return torch.ops.qd_serving.gqa_decode_window(q, k_cache, v_cache, block_table, context_lens, float(scale),
                                                  window, sinks)


def gqa_decode_tree(q, k_cache, v_cache, block_table, context_lens, tree_mask, *, window=None, sinks=0, scale=None):
    """Attention of up to 64 drafted tokens per sequence over the cache.

    q ``[B, T, Hq, D]``.  ``context_lens [B]`` counts the tokens before the
    drafted ones; drafted token ``j`` lies at token ``context_lens[b] + j`` of
    the cache (already written there).  Bit ``j`` of ``tree_mask[b, t]``
    (int64 ``[B, T]``): drafted token ``t`` sees drafted token ``j``, that is
    its ancestors and itself; lower-triangular masks make a chain.  A mask of 0
    marks padding of a ragged batch and gives a zero row.  Every other row sees
    all of its context, or with ``window`` what is less than ``window``
    positions before its own, ``context_lens[b] + popcount(mask) - 1``, and the
    first ``sinks`` tokens.  Returns ``[B, T, Hq, D]``.

    Without a window, how the work is cut follows from the width of
    ``block_table``, since lengths are not read on the host: short contexts are
    up to twice as fast with a table of the batch's longest context
    (``block_table[:, :pages].contiguous()``) as with one of the longest that a
    model allows.
    """
    _require_extension()
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if window is not None and window < 1:
        raise ValueError("window must be positive, or None")
    return torch.ops.qd_serving.gqa_decode_tree(q, k_cache, v_cache, block_table, context_lens, tree_mask,
                                                float(scale), window or 0, sinks)


def qk_norm_rope_write(q, key, value, cos_sin, positions, k_cache, v_cache, slot_mapping, *, q_weight=None,
                       k_weight=None, eps=1e-6, interleaved=False):
    """Normalizes (RMS, per head) and rotates queries and keys, writes keys and
    values to the cache, and returns the queries ``[N, Hq, D]``.

    q ``[N, Hq, D]``, key and value ``[N, Hkv, D]``: tokens may lie any stride
    apart, as views of one projection's output do.  ``cos_sin`` float32
    ``[max_positions, R]`` holds ``R/2`` cosines and then ``R/2`` sines of each
    position, ``R <= D`` even; the first ``R`` elements of a head are turned in
    pairs ``(i, i + R/2)``, or ``(2i, 2i + 1)`` if ``interleaved``.
    ``positions`` int32 ``[N]``.  ``slot_mapping`` int64 ``[N]`` are flat cache
    rows, as in :func:`latent_kv_write`: distinct, and one outside the cache
    (such as -1 for padding) is skipped.  A position outside the table gives a
    zero query and writes nothing.  The caches must not overlap each other (an
    error) or the inputs.  ``q_weight`` and ``k_weight`` ``[D]`` (q's dtype or
    float32) turn the norms on.  fp32 arithmetic, rounded once.
    """
    _require_extension()
    return torch.ops.qd_serving.qk_norm_rope_write(q, key, value, cos_sin, positions, k_cache, v_cache, slot_mapping,
                                                   q_weight, k_weight, float(eps), bool(interleaved))


def kv_compact(caches, block_table, context_lens, accepted):
    """Moves the cache rows of accepted drafted tokens next to the context.

    In every cache of ``caches`` (a list of ``[blocks, block_size, ...]``
    tensors of one shape and dtype that do not overlap: K and V of any number
    of layers, or latent caches) token ``context_lens[b] + accepted[b, i]``
    moves to token ``context_lens[b] + i``, as if all were read before any is
    written.  ``accepted`` int32 ``[B, A]``, ``A <= 64``: indices of drafted
    tokens, such as the path that was verified; negative entries move nothing.
    Tokens outside the table and pages outside the pool are skipped.  Rows
    that move must be their sequence's own: pages shared with other sequences
    may hold context, not drafted tokens.  One launch serves up to 128 caches.
    """
    _require_extension()
    torch.ops.qd_serving.kv_compact(list(caches), block_table, context_lens, accepted)
