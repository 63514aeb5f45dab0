"""CPU checks of the operators around drafted tokens and sliding windows:
argument checks in order with their messages, launch argument errors (before
anything is enqueued), plans, op schemas, and the oracle against closed forms
and the decode oracle.  No kernel runs here."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import attention_amd
from attention_amd import cabi, core
from attention_amd.cabi import desc
from oracle.gqa_oracle import oracle_decode
from oracle.serving_oracle import oracle_compact, oracle_tree, oracle_write, visible

F32, F16, BF16, I32, I64 = 0, 1, 2, 3, 4


def _edit(key, **kw):
    def f(d):
        old = d[key]
        if "sizes" in kw:
            old = desc(kw["sizes"], old.dtype, old.is_device, old.device_index, old.contiguous)
        for name, val in kw.items():
            if name != "sizes":
                setattr(old, name, val)
        d[key] = old
    return f


def _all(*edits):
    return lambda d: [e(d) for e in edits]


# ---- Attention ---------------------------------------------------------------


def tree_descs():
    return dict(q=desc([4, 5, 8, 64], F16), k=desc([57, 16, 2, 64], F16), v=desc([57, 16, 2, 64], F16),
                table=desc([4, 32], I32), lens=desc([4], I32), mask=desc([4, 5], I64))


def run_tree(d, **kw):
    return cabi.validate_gqa_decode_tree(d["q"], d["k"], d["v"], d["table"], d["lens"], d["mask"], **kw)


TREE_ORDER = [
    (_edit("q", is_device=0), "q must be a CUDA tensor"),
    (_edit("q", contiguous=0), "q must be contiguous"),
    (_edit("k", contiguous=0), "k_cache must be contiguous"),
    (_edit("lens", is_device=0), "context_lens must be a CUDA tensor"),
    (_edit("mask", is_device=0), "tree_mask must be a CUDA tensor"),
    (_edit("mask", contiguous=0), "tree_mask must be contiguous"),
    (_edit("q", sizes=[4, 8, 64]), "q must be [B, T, Hq, D]"),
    (_edit("k", sizes=[57, 16, 128]), "k_cache must be [Nblocks, BlockSize, Hkv, D]"),
    (_edit("v", sizes=[57, 16, 2, 32]), "v_cache shape mismatch"),
    (_edit("table", sizes=[4, 32, 1]), "block_table must be [B, MaxPages]"),
    (_edit("lens", sizes=[4, 1]), "context_lens must be [B]"),
    (_edit("mask", sizes=[4, 4]), "tree_mask must be int64 [B, T]"),
    (_edit("mask", dtype=I32), "tree_mask must be int64 [B, T]"),
    (_edit("mask", device_index=1), "all tensors must use one CUDA device"),
    (_edit("k", dtype=BF16), "q/k/v dtype must match"),
    (_all(_edit("q", dtype=-1), _edit("k", dtype=-1), _edit("v", dtype=-1)), "q/k/v must be float32/float16/bfloat16"),
    (_edit("table", dtype=I64), "block_table and context_lens must be int32"),
    (_edit("lens", sizes=[3]), "batch sizes must match"),
    (_all(_edit("q", sizes=[4, 65, 8, 64]), _edit("mask", sizes=[4, 65])),
     "supported drafted tokens per sequence are [1, 64]"),
    (_all(_edit("q", sizes=[4, 0, 8, 64]), _edit("mask", sizes=[4, 0])),
     "supported drafted tokens per sequence are [1, 64]"),
    (_edit("q", sizes=[4, 5, 8, 32]), "q head_dim and cache head_dim must match"),
    (_edit("q", sizes=[4, 5, 7, 64]), "Hq must be divisible by Hkv"),
    (_all(_edit("q", sizes=[4, 5, 8, 264]), _edit("k", sizes=[57, 16, 2, 264]), _edit("v", sizes=[57, 16, 2, 264])),
     "supported head_dim is [1, 256]"),
    (_all(_edit("k", sizes=[0, 16, 2, 64]), _edit("v", sizes=[0, 16, 2, 64])),
     "cache must have positive blocks and block_size"),
    (_edit("table", sizes=[4, 0]), "block_table must have at least one page"),
    (_all(_edit("q", sizes=[1 << 20, 5, 8, 64]), _edit("table", sizes=[1 << 20, 32]), _edit("lens", sizes=[1 << 20]),
          _edit("mask", sizes=[1 << 20, 5])), "tensor sizes exceed int32 CUDA launch limits"),
]


@pytest.mark.parametrize("i", range(len(TREE_ORDER)))
def test_tree_validation_order_and_messages(i):
    d = tree_descs()
    edit, message = TREE_ORDER[i]
    edit(d)
    assert run_tree(d) == (1, message)
    assert cabi.error_string(1) == message


def test_tree_validation_scalars():
    d = tree_descs()
    assert run_tree(d) == (0, "")
    assert run_tree(d, window=16, sinks=4) == (0, "")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert run_tree(d, scale=scale)[1] == "scale must be positive and finite"
    for window in (-1, 1 << 31):
        assert run_tree(d, window=window)[1] == "window must be in [1, 2^31)"
    for window, sinks in ((16, -1), (16, 1 << 31), (0, 4)):
        assert run_tree(d, window=window, sinks=sinks)[1] == "sinks must be in [0, 2^31) and need a window"


def test_window_validation():
    d = tree_descs()
    d.update(q=desc([4, 8, 64], F16), mask=None)
    assert run_tree(d, window=16) == (0, "")
    assert run_tree(d)[1] == "window must be in [1, 2^31)"
    d["q"] = desc([4, 5, 8, 64], F16)
    assert run_tree(d, window=16)[1] == "q must be [B, Hq, D]"


def tree_args():
    return dict(q=1, k=1, v=1, table=1, lens=1, mask=1, out=1, ws=16, ws_bytes=1 << 40, B=4, T=5, Hq=8, Hkv=2, D=64,
                P=16, maxP=32, N=57, dtype=BF16, scale=0.125, window=0, sinks=0, flags=0, stream=None)


@pytest.mark.parametrize("over, message", [
    (dict(T=65), "invalid dimensions"), (dict(T=0), "invalid dimensions"), (dict(Hq=7), "invalid dimensions"),
    (dict(D=257), "invalid dimensions"), (dict(P=0), "invalid dimensions"), (dict(maxP=0), "invalid dimensions"),
    (dict(N=0), "invalid dimensions"), (dict(dtype=I32), "invalid dimensions"), (dict(window=-1), "invalid dimensions"),
    (dict(sinks=4), "invalid dimensions"), (dict(mask=None), "invalid dimensions"), (dict(B=-1), "invalid dimensions"),
    (dict(B=1 << 24), "invalid dimensions"), (dict(scale=0.0), "scale must be positive and finite"),
    (dict(scale=float("nan")), "scale must be positive and finite"), (dict(q=None), "null tensor pointer"),
    (dict(out=None), "null tensor pointer"), (dict(lens=None), "null tensor pointer"),
    (dict(maxP=4096, ws=None), "workspace too small or not 16-byte aligned"),
    (dict(maxP=4096, ws=8), "workspace too small or not 16-byte aligned"),
    (dict(maxP=4096, ws_bytes=64), "workspace too small or not 16-byte aligned")])
def test_tree_launch_argument_errors(over, message):
    a = tree_args()
    a.update(over)
    assert cabi.lib().qd_gqa_decode_tree(*a.values()) == 1
    assert cabi.error_string(1) == message


def test_tree_launch_batch_zero_is_a_no_op():
    a = tree_args()
    a.update(B=0, q=None, ws=None, ws_bytes=0)
    assert cabi.lib().qd_gqa_decode_tree(*a.values()) == 0


SHAPES_OF_PLANS = [
    # B, T, Hq, Hkv, D, P, maxP, has_mask, window, sinks, dtype
    (1, 1, 1, 1, 8, 16, 1, 1, 0, 0, BF16),
    (64, 1, 32, 8, 128, 16, 512, 0, 1024, 4, BF16),
    (64, 1, 32, 8, 128, 16, 512, 0, 8192, 4, BF16),
    (32, 16, 32, 8, 128, 16, 257, 1, 0, 0, BF16),
    (8, 64, 64, 8, 128, 64, 257, 1, 0, 0, BF16),
    (5, 7, 32, 32, 80, 12, 60, 1, 0, 0, F16),
    (8, 8, 32, 8, 128, 16, 65, 1, 0, 0, F32),
    (2, 64, 71, 1, 256, 1, 4000, 1, 300, 64, BF16),
    (1025, 2, 4, 2, 64, 16, 2000, 1, 0, 0, F16),
    (4, 3, 4, 2, 33, 16, 2000, 1, 0, 0, F32),
    (1, 1, 8, 1, 128, 16, 1 << 27, 1, 0, 0, BF16),
    (1, 1, 8, 1, 128, 16, 1 << 27, 0, 2147483647, 2147483647, BF16),
]


@pytest.mark.parametrize("shape", SHAPES_OF_PLANS)
def test_plans_cover_all_rows_and_fit_their_workspace(shape):
    """Every row has a workgroup, one launch at most fills the card, and the
    workspace holds both kernels' partials."""
    B, T, Hq, Hkv, D, P, maxP, has_mask, window, sinks, dtype = shape
    kind, groups, rows = cabi.gqa_decode_tree_info(*shape)
    per_head = T * Hq // Hkv
    chunks = -(-per_head // rows)
    assert rows >= 1 and groups >= 1
    need = 0
    if kind == cabi.QD_TREE_VALU:
        assert D % 8 and rows == 1 and groups % (B * T * Hq) == 0
        splits = groups // (B * T * Hq)
        need = 4 * B * T * Hq * splits * (D + 2) if splits > 1 else 0
    elif kind == cabi.QD_TREE_MFMA:
        assert groups == B * Hkv * chunks
    else:
        assert B <= 1024 and groups <= 2 * 256
        need = 8 * B * Hkv * chunks + 4 * 2 * groups * rows * (D + 2)
    args = (B, T, Hq, Hkv, D, P, maxP, has_mask, window, sinks, dtype)
    valu = cabi.gqa_decode_tree_info(*args, cabi.QD_FLAG_FORCE_GENERIC)
    assert valu[0] == cabi.QD_TREE_VALU
    splits = valu[1] // (B * T * Hq)
    both = max(need, 4 * B * T * Hq * splits * (D + 2) if splits > 1 else 0)
    bytes_ = cabi.lib().qd_gqa_decode_tree_workspace_bytes(*args, 0)
    # A range has two partials, of whole blocks of 16 rows even for one row.
    assert both <= bytes_ <= 32 * both + 4096


@pytest.mark.parametrize("T,Hq,D,dtype", [(1, 8, 128, BF16), (2, 8, 128, BF16), (8, 8, 128, BF16), (16, 8, 128, BF16), (11, 8, 64, F16), (17, 8, 128, BF16), (64, 8, 128, BF16),
                                          (64, 64, 64, F16), (64, 71, 256, BF16), (64, 71, 128, F32),
                                          (64, 71, 256, F32), (3, 200, 192, F16)])
def test_rows_are_cut_evenly(T, Hq, D, dtype):
    """As many rows as the registers hold where the tiles fill the card (up to 128 rows of 256 bytes and short
    contexts: 64), fewer where they do not, 16 at least."""
    es = 4 if dtype == F32 else 2
    R = T * Hq
    most = 256 if D * es <= 256 else 128 if D * es <= 512 else 32

    def rows_of(B, maxP):
        kind, _, rows = cabi.gqa_decode_tree_info(B, T, Hq, 1, D, 16, maxP, dtype=dtype)
        assert kind != cabi.QD_TREE_VALU
        return rows

    def cut(most):
        return -(-R // -(-R // most))

    assert rows_of(256, 1000) == cut(most) <= most
    assert rows_of(1000, 64) == cut(min(most, 64) if R <= 128 else most)
    assert rows_of(1, 1) == cut(16) <= 16


def test_which_contexts_are_split():
    """One workgroup per item where that leaves little idle, equal ranges of all tiles elsewhere; more sequences
    than the split's prefix holds are not split."""
    def kind(B, maxP, window=0, mask=1):
        return cabi.gqa_decode_tree_info(B, 1, 32, 8, 128, 16, maxP, mask, window, 0, BF16)[0]

    assert kind(64, 512, 1024, 0) == cabi.QD_TREE_MFMA           # 512 items for 512 places
    assert kind(40, 512, 1024, 0) == cabi.QD_TREE_MFMA_SPLIT     # 320 items
    assert kind(4, 4) == cabi.QD_TREE_MFMA                       # one unit each
    assert kind(4, 512) == cabi.QD_TREE_MFMA_SPLIT
    assert kind(64, 64) == cabi.QD_TREE_MFMA                     # 16 units at most
    assert kind(64, 100) == cabi.QD_TREE_MFMA_SPLIT              # lengths may differ by 25 units
    assert kind(1024, 512) == cabi.QD_TREE_MFMA_SPLIT
    assert kind(1025, 512) == cabi.QD_TREE_MFMA


@pytest.mark.parametrize("P", [1 << 20, 1 << 24, 1 << 25, (1 << 25) + 5, (1 << 26) - 1])
@pytest.mark.parametrize("Hq", [1, 16, 1 << 10, 1 << 17, (1 << 18) - 1])
def test_plans_of_tables_past_the_clamp(P, Hq):
    """Lengths are clamped below 2^31 tokens, so wider tables change no plan (their items times tiles pass 2^63)."""
    tight = -(-(1 << 31) // P)
    for T, has_mask, window in ((64, 1, 0), (1, 0, 2147483647)):
        want = cabi.gqa_decode_tree_info(1, T, Hq, 1, 8, P, tight, has_mask, window, 0, BF16)
        assert want[0] != cabi.QD_TREE_VALU
        for maxP in (tight + 1, 1 << 20, 2147483647):
            args = (1, T, Hq, 1, 8, P, maxP, has_mask, window, 0, BF16)
            assert cabi.gqa_decode_tree_info(*args) == want
            assert cabi.lib().qd_gqa_decode_tree_workspace_bytes(*args, 0) == \
                cabi.lib().qd_gqa_decode_tree_workspace_bytes(1, T, Hq, 1, 8, P, tight, has_mask, window, 0, BF16, 0)


@pytest.mark.parametrize("over", [dict(B=1 << 30, T=64, Hq=1 << 30), dict(B=1 << 28, T=64, Hq=1 << 30),
                                  dict(B=1 << 24, T=1, Hq=2), dict(B=2, T=1, Hq=1 << 24),
                                  dict(B=0, T=64, Hq=1 << 30), dict(B=2147483647, T=64, Hq=2147483647)])
def test_tree_rows_are_counted_without_overflow(over):
    """Factors whose product wraps to a small number in 64 bits are refused everywhere."""
    a = tree_args()
    a.update(over, Hkv=1)
    assert cabi.lib().qd_gqa_decode_tree(*a.values()) == 1
    assert cabi.error_string(1) == "invalid dimensions"
    shape = (a["B"], a["T"], a["Hq"], 1, 64, 16, 32, 1, 0, 0, BF16)
    assert cabi.gqa_decode_tree_info(*shape)[0] == -1
    assert cabi.lib().qd_gqa_decode_tree_workspace_bytes(*shape, 0) == 0


@pytest.mark.parametrize("Hkv,D,P,valu", [
    (1 << 23, 256, 2147483647, True),        # 2^64 - 2^33 bytes, counted at 4 per element
    (1 << 23, 256, 1 << 30, True), (1 << 14, 256, 128, True),
    ((1 << 14) - 1, 256, 128, False), (1, 8, (1 << 26) - 1, False),
    (1, 8, 1 << 26, True), (1 << 17, 256, 1, True)])
def test_pages_past_32_bits_take_the_valu_kernel(Hkv, D, P, valu):
    """The matrix-core kernel's offsets within a page (of 16 tokens at least) are 32 bits wide."""
    assert (cabi.gqa_decode_tree_info(1, 1, Hkv, Hkv, D, P, 1, 1, 0, 0, BF16)[0] == cabi.QD_TREE_VALU) == valu


# ---- Norm, rotation and write ------------------------------------------------


def write_descs():
    return dict(q=desc([6, 8, 64], BF16), key=desc([6, 2, 64], BF16), value=desc([6, 2, 64], BF16),
                cos_sin=desc([100, 64], F32), positions=desc([6], I32), kc=desc([9, 16, 2, 64], BF16),
                vc=desc([9, 16, 2, 64], BF16), slots=desc([6], I64), qw=desc([64], BF16), kw=desc([64], BF16))


WRITE_ORDER = [
    (_edit("q", is_device=0), "all tensors must be CUDA tensors"),
    (_edit("qw", is_device=0), "all tensors must be CUDA tensors"),
    (_edit("slots", device_index=1), "all tensors must share a device"),
    (_edit("key", contiguous=0), "the heads of a token must be contiguous in q, key and value"),
    (_edit("kc", contiguous=0), "cos_sin, positions, caches, slots and weights must be contiguous"),
    (_edit("q", sizes=[6, 512]), "q must be [N, Hq, D]"),
    (_edit("key", sizes=[5, 2, 64]), "key/value must be [N, Hkv, D]"),
    (_edit("value", sizes=[6, 1, 64]), "key/value must be [N, Hkv, D]"),
    (_edit("kc", sizes=[9, 16, 128]), "cache must be [Nblocks, P, Hkv, D]"),
    (_edit("vc", sizes=[8, 16, 2, 64]), "cache must be [Nblocks, P, Hkv, D]"),
    (_all(_edit("kc", sizes=[9, 16, 3, 64]), _edit("vc", sizes=[9, 16, 3, 64])), "cache head shape mismatch"),
    (_all(_edit("kc", sizes=[0, 16, 2, 64]), _edit("vc", sizes=[0, 16, 2, 64])), "invalid dimensions"),
    (_edit("cos_sin", dtype=BF16), "cos_sin must be float32 [MaxPositions, R]"),
    (_edit("cos_sin", sizes=[100, 63]), "the rotary dim must be even and at most head_dim"),
    (_edit("cos_sin", sizes=[100, 66]), "the rotary dim must be even and at most head_dim"),
    (_edit("positions", dtype=I64), "positions must be int32 [N]"),
    (_edit("slots", dtype=I32), "slots must be int64 [N]"),
    (_edit("value", dtype=F16), "dtype mismatch"),
    (_edit("vc", dtype=F32), "dtype mismatch"),
    (_all(*(_edit(n, dtype=-1) for n in ("q", "key", "value", "kc", "vc"))), "unsupported dtype"),
    (_edit("qw", sizes=[32]), "weights must be [D]"),
    (_all(_edit("qw", dtype=F16), _edit("kw", dtype=F16)), "weights must have q's dtype or be float32"),
    (_edit("kw", dtype=F32), "q_weight and k_weight must have one dtype"),
    (_all(_edit("q", sizes=[1 << 24, 8, 64]), _edit("key", sizes=[1 << 24, 2, 64]),
          _edit("value", sizes=[1 << 24, 2, 64]), _edit("positions", sizes=[1 << 24]), _edit("slots", sizes=[1 << 24])),
     "tensor sizes exceed int32 CUDA launch limits"),
]


@pytest.mark.parametrize("i", range(len(WRITE_ORDER)))
def test_write_validation_order_and_messages(i):
    d = write_descs()
    edit, message = WRITE_ORDER[i]
    edit(d)
    assert cabi.validate_qk_norm_rope_write(*d.values()) == (1, message)


def test_write_validation_accepts():
    d = write_descs()
    assert cabi.validate_qk_norm_rope_write(*d.values()) == (0, "")
    d["kw"] = None
    assert cabi.validate_qk_norm_rope_write(*d.values()) == (0, "")
    d["qw"] = desc([64], F32)
    assert cabi.validate_qk_norm_rope_write(*d.values(), eps=0.0) == (0, "")
    for eps in (-1e-6, float("inf"), float("nan")):
        assert cabi.validate_qk_norm_rope_write(*d.values(), eps=eps)[1] == "eps must be finite and not negative"


def write_args():
    return dict(q=1, key=1, value=1, cos_sin=1, positions=1, kc=1, vc=1, slots=1, qw=1, kw=1, out=1, tokens=6, Hq=8, Hkv=2,
                D=64, rot=64, qs=768, ks=768, vs=768, max_positions=100, rows=144, dtype=BF16, wdtype=BF16, eps=1e-6,
                interleaved=0, stream=None)


@pytest.mark.parametrize("over, message", [
    (dict(tokens=-1), "tokens must be in [0, 2^24)"), (dict(tokens=1 << 24), "tokens must be in [0, 2^24)"),
    (dict(Hkv=0), "invalid dimensions"), (dict(rows=0), "invalid dimensions"), (dict(qs=-1), "invalid dimensions"),
    (dict(D=0), "supported head_dim is [1, 256]"), (dict(rot=66), "the rotary dim must be even and at most head_dim"),
    (dict(rot=31), "the rotary dim must be even and at most head_dim"), (dict(dtype=I32), "unsupported dtype"),
    (dict(wdtype=F16), "weights must have q's dtype or be float32"),
    (dict(eps=float("nan")), "eps must be finite and not negative"), (dict(out=None), "null tensor pointer"),
    (dict(cos_sin=None), "null tensor pointer")])
def test_write_launch_argument_errors(over, message):
    a = write_args()
    a.update(over)
    assert cabi.lib().qd_qk_norm_rope_write(*a.values()) == 1
    assert cabi.error_string(1) == message


def test_write_launch_without_tokens_is_a_no_op():
    a = write_args()
    a.update(tokens=0, q=None, out=None)
    assert cabi.lib().qd_qk_norm_rope_write(*a.values()) == 0


@pytest.mark.parametrize("dtype, kc, vc, rows", [
    (BF16, 4096, 4096, 144), (BF16, 4096, 4096 + 144 * 256 - 16, 144), (F32, 4096 + 144 * 512 - 16, 4096, 144),
    (F16, 4096, 1 << 47, 1 << 62)])
def test_write_refuses_overlapping_caches(dtype, kc, vc, rows):
    a = write_args()
    a.update(dtype=dtype, wdtype=dtype, kc=kc, vc=vc, rows=rows)
    assert cabi.lib().qd_qk_norm_rope_write(*a.values()) == 1
    assert cabi.error_string(1) == "k_cache and v_cache must not overlap"


# ---- Compaction --------------------------------------------------------------


def compact_descs():
    return dict(cache=desc([9, 16, 2, 64], BF16), table=desc([4, 3], I32), lens=desc([4], I32), accepted=desc([4, 8], I32))


COMPACT_ORDER = [
    (_edit("cache", is_device=0), "all tensors must be contiguous CUDA tensors"),
    (_edit("accepted", contiguous=0), "all tensors must be contiguous CUDA tensors"),
    (_edit("table", device_index=1), "all tensors must share a device"),
    (_edit("cache", sizes=[9, 16]), "cache must be [Nblocks, P, ...]"),
    (_edit("cache", sizes=[9, 0, 2, 64]), "invalid dimensions"),
    (_edit("accepted", sizes=[4]), "invalid metadata shape"),
    (_edit("lens", sizes=[3]), "invalid metadata shape"),
    (_edit("table", sizes=[4, 0]), "invalid metadata shape"),
    (_edit("accepted", dtype=I64), "metadata must be int32"),
    (_edit("accepted", sizes=[4, 65]), "at most 64 accepted tokens per sequence"),
    (_edit("cache", dtype=-1), "unsupported dtype"),
]


@pytest.mark.parametrize("i", range(len(COMPACT_ORDER)))
def test_compact_validation_order_and_messages(i):
    d = compact_descs()
    assert cabi.validate_kv_compact(*d.values()) == (0, "")
    edit, message = COMPACT_ORDER[i]
    edit(d)
    assert cabi.validate_kv_compact(*d.values()) == (1, message)


def _compact(pointers, n=None, count=8, batch=4, N=9, P=16, maxP=3, row=256, meta=16):
    array = (ctypes.c_void_p * max(1, len(pointers)))(*pointers)
    return cabi.lib().qd_kv_compact(array, len(pointers) if n is None else n, meta, meta, meta, batch, count, P, maxP, N,
                                    row, None)


def test_compact_launch_argument_errors():
    size = 9 * 16 * 256
    for call, message in [
            (lambda: _compact([4096, 4096]), "caches must not overlap"),
            (lambda: _compact([4096, 1 << 30, 4096 + size - 16]), "caches must not overlap"),
            (lambda: _compact([4097]), "caches must be aligned to their elements"),
            (lambda: _compact([None]), "null tensor pointer"),
            (lambda: _compact([4096], meta=None), "null tensor pointer"),
            (lambda: _compact([4096], count=65), "at most 64 accepted tokens per sequence"),
            (lambda: _compact([4096], row=3), "invalid dimensions"),
            (lambda: _compact([4096], N=1 << 60), "invalid dimensions"),
            (lambda: _compact([4096], P=0), "invalid dimensions"),
            (lambda: _compact([4096], batch=1 << 24), "caches and batch must be >= 0, batch below 2^24"),
            (lambda: _compact([4098], row=(1 << 24)), "tensor sizes exceed int32 CUDA launch limits")]:
        assert call() == 1
        assert cabi.error_string(1) == message
    assert _compact([]) == 0 and _compact([4096], batch=0) == 0 and _compact([4096], count=0) == 0


# ---- Torch ops and Python API --------------------------------------------------


def test_op_schemas():
    ops = torch.ops.qd_serving
    assert str(ops.gqa_decode_window.default._schema) == (
        "qd_serving::gqa_decode_window(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
        "Tensor context_lens, float scale, int window, int sinks) -> Tensor")
    assert str(ops.gqa_decode_tree.default._schema) == (
        "qd_serving::gqa_decode_tree(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
        "Tensor context_lens, Tensor tree_mask, float scale, int window, int sinks) -> Tensor")
    assert str(ops.qk_norm_rope_write.default._schema) == (
        "qd_serving::qk_norm_rope_write(Tensor q, Tensor key, Tensor value, Tensor cos_sin, Tensor positions, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, Tensor? q_weight, Tensor? k_weight, float eps, "
        "bool interleaved) -> Tensor")
    assert str(ops.kv_compact.default._schema) == (
        "qd_serving::kv_compact(Tensor(a!)[] caches, Tensor block_table, Tensor context_lens, Tensor accepted) -> ()")


def test_public_names_and_missing_extension(monkeypatch):
    for name in ("gqa_decode_window", "gqa_decode_tree", "qk_norm_rope_write", "kv_compact"):
        assert name in attention_amd.__all__
    q = torch.zeros(1, 2, 4)
    with pytest.raises(NotImplementedError):
        attention_amd.gqa_decode_window(q, q, q, q, q, window=4)
    with pytest.raises(ValueError, match="window must be positive, or None"):
        attention_amd.gqa_decode_tree(q, q, q, q, q, q, window=0)
    monkeypatch.setattr(core, "_LOAD_ERROR", OSError("missing"))
    for call in (lambda: attention_amd.gqa_decode_window(q, q, q, q, q, window=4),
                 lambda: attention_amd.gqa_decode_tree(q, q, q, q, q, q),
                 lambda: attention_amd.qk_norm_rope_write(q, q, q, q, q, q, q, q),
                 lambda: attention_amd.kv_compact([q], q, q, q)):
        with pytest.raises(RuntimeError, match=r"^qd_attention CUDA extension was not loaded$"):
            call()


# ---- The oracle ------------------------------------------------------------------


def _pool(rng, B, Hkv, D, P, width):
    N = B * width
    table = rng.permutation(N).reshape(B, width).astype(np.int32)
    return rng.standard_normal((N, P, Hkv, D)), rng.standard_normal((N, P, Hkv, D)), table


def test_oracle_wide_window_is_decode():
    rng = np.random.default_rng(0)
    k, v, table = _pool(rng, 3, 2, 8, 4, 5)
    q, lens = rng.standard_normal((3, 1, 4, 8)), np.array([0, 1, 19])
    got, _, _ = oracle_tree(q, k, v, table, lens, None, 20, 0, 0.3)
    want = oracle_decode(q[:, 0].astype(np.float32), k.astype(np.float32), v.astype(np.float32), table,
                         lens.astype(np.int32), scale=0.3)
    # The decode oracle is fp32: 8-term dots and 19-term sums of values below 5.
    assert np.abs(got[:, 0] - want).max() < 1e-4


def test_oracle_chain_is_one_query_at_a_time():
    rng = np.random.default_rng(1)
    k, v, table = _pool(rng, 2, 2, 8, 4, 5)
    q, lens = rng.standard_normal((2, 4, 4, 8)), np.array([0, 11])
    masks = [[(1 << t + 1) - 1 for t in range(4)]] * 2
    for window, sinks in ((0, 0), (3, 0), (3, 2), (9, 1)):
        got, _, _ = oracle_tree(q, k, v, table, lens, masks, window, sinks, 0.3)
        for t in range(4):
            one, _, _ = oracle_tree(q[:, t:t + 1], k, v, table, lens + t + 1, None, window or 99, sinks, 0.3)
            assert np.abs(got[:, t] - one[:, 0]).max() < 1e-12


def test_oracle_visibility():
    # Two branches below one root at context 5: window 2 keeps the token and its parent.
    masks = [0b1, 0b11, 0b101, 0]
    got = visible(5, masks, 4, 100, 2, 1)
    want = [[1, 0, 0, 0, 1, 1, 0, 0, 0], [1, 0, 0, 0, 0, 1, 1, 0, 0], [1, 0, 0, 0, 0, 1, 0, 1, 0], [0] * 9]
    assert np.array_equal(got, np.array(want, dtype=bool))
    # A table that ends after the first drafted token, and bits past the count.
    assert np.array_equal(visible(5, [0b1, 0b11111], 2, 6, 0, 0)[1], np.array([1, 1, 1, 1, 1, 1, 0], dtype=bool))


def test_oracle_write_and_compact_closed_forms():
    rng = np.random.default_rng(2)
    q, key, value = rng.standard_normal((3, 2, 6)), rng.standard_normal((3, 1, 6)), rng.standard_normal((3, 1, 6))
    kc = rng.standard_normal((2, 2, 1, 6))
    angle = np.arange(4)[:, None] * np.array([0.5, 0.1])
    cs = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    out, k2, v2 = oracle_write(q, key, value, cs, [0, 3, 9], kc, kc, [2, -1, 0], None, None, 0.0, False)
    assert np.array_equal(out[0], q[0]) and np.array_equal(out[2], 0 * q[2])        # position 0, position outside
    pair = (q[1, :, 0] + 1j * q[1, :, 2]) * np.exp(1j * angle[3, 0])                # rotation as a complex product
    assert np.allclose(out[1, :, 0] + 1j * out[1, :, 2], pair) and np.array_equal(out[1, :, 4:], q[1, :, 4:])
    assert np.array_equal(k2[1, 0], key[0]) and np.array_equal(v2[1, 0], value[0])
    k2[1, 0] = kc[1, 0]
    assert np.array_equal(k2, kc)                                                     # nothing else was written
    cache = np.arange(12.0).reshape(3, 4, 1)
    after = oracle_compact(cache, np.array([[2, 0]]), np.array([2]), np.array([[0, 3, 1, -1, 5, 7]]))
    # Tokens 2.. of pages 2, 0 are rows 10, 11, 0, 1, 2, 3; 5 is row 3, 7 lies past the table.
    want = np.arange(12.0)
    want[[10, 11, 0, 2]] = [10, 1, 11, 3]
    assert np.array_equal(after.reshape(-1), want)
