"""CPU checks of prompt attention and of 8-bit caches: argument checks in order
with their messages, launch argument errors (before anything is enqueued), plans,
op schemas, and the oracle against closed forms.  No kernel runs here."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_amd
from attention_amd import cabi, core
from attention_amd.cabi import desc
from oracle.prompt_oracle import oracle_append, oracle_decode, oracle_prefill, power_scale, round_to

F32, F16, BF16, I32, I64, E4M3, I8 = 0, 1, 2, 3, 4, 5, 6


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


def _in_order(validate, descs, order):
    """Each edit gives its message, also with every later edit's fault beside it."""
    assert validate(descs()) == (0, "")
    for i, (edit, message) in enumerate(order):
        d = descs()
        edit(d)
        assert validate(d) == (1, message), i


# ---- Prompt attention --------------------------------------------------------


def prefill_descs():
    return dict(q=desc([40, 8, 64], F16), k=desc([90, 2, 64], F16), v=desc([90, 2, 64], F16), cu=desc([4], I32),
                cu_k=desc([4], I32))


def run_prefill(d, **kw):
    return cabi.validate_gqa_prefill(d["q"], d["k"], d["v"], d["cu"], d["cu_k"], **kw)


PREFILL_ORDER = [
    (_edit("q", is_device=0), "all tensors must be CUDA tensors"),
    (_edit("k", device_index=1), "all tensors must share a device"),
    (_edit("v", contiguous=0), "the heads of a token must be contiguous in q, key and value"),
    (_edit("cu", contiguous=0), "cu_seqlens must be contiguous"),
    (_edit("cu_k", is_device=0), "all tensors must be CUDA tensors"),
    (_edit("q", sizes=[40, 512]), "q must be [Tq, Hq, D]"),
    (_edit("k", sizes=[90, 128]), "key/value must be [Tk, Hkv, D]"),
    (_edit("v", sizes=[91, 2, 64]), "key/value must be [Tk, Hkv, D]"),
    (_edit("q", sizes=[40, 8, 32]), "q and key head_dim must match"),
    (_edit("q", sizes=[40, 7, 64]), "Hq must be divisible by Hkv"),
    (_all(_edit("k", sizes=[90, 0, 64]), _edit("v", sizes=[90, 0, 64])), "Hq must be divisible by Hkv"),
    (_all(*(_edit(x, sizes=s) for x, s in (("q", [40, 8, 264]), ("k", [90, 2, 264]), ("v", [90, 2, 264])))),
     "supported head_dim is [1, 256]"),
    (_all(*(_edit(x, dtype=E4M3) for x in "qkv")), "q/key/value must be float32/float16/bfloat16"),
    (_edit("v", dtype=BF16), "q/key/value dtype must match"),
    (_edit("cu", dtype=I64), "cu_seqlens must be int32 [B + 1]"),
    (_edit("cu", sizes=[0]), "cu_seqlens must be int32 [B + 1]"),
    (_edit("cu_k", sizes=[5]), "cu_seqlens_k must be int32 [B + 1]"),
    (_edit("cu_k", defined=0), "without cu_seqlens_k there must be a key for every query"),
    (_edit("q", sizes=[1 << 28, 8, 64]), "tensor sizes exceed int32 CUDA launch limits"),
    (_all(_edit("k", sizes=[1 << 31, 2, 64]), _edit("v", sizes=[1 << 31, 2, 64])),
     "tensor sizes exceed int32 CUDA launch limits"),
]


def test_prefill_validation():
    _in_order(run_prefill, prefill_descs, PREFILL_ORDER)
    for kw, message in ((dict(scale=0.0), "scale must be positive and finite"),
                        (dict(scale=float("inf")), "scale must be positive and finite"),
                        (dict(window=-1), "window must be in [0, 2^31)"), (dict(window=1 << 31), "window must be in [0, 2^31)"),
                        (dict(sinks=1), "sinks must be in [0, 2^31) and need a window"),
                        (dict(window=5, sinks=-1), "sinks must be in [0, 2^31) and need a window")):
        assert run_prefill(prefill_descs(), **kw) == (1, message)
    assert run_prefill(prefill_descs(), window=5, sinks=9) == (0, "")


def prefill_args():
    return dict(q=16, k=16, v=16, cu=16, cu_k=16, out=16, ws=None, ws_bytes=0, B=3, Tq=40, Tk=90, Hq=8, Hkv=2, D=64,
                qs=512, ks=128, vs=128, dtype=BF16, scale=0.1, window=0, sinks=0, flags=0, stream=None)


@pytest.mark.parametrize("over, message", [
    (dict(B=-1), "invalid dimensions"), (dict(Tq=-1), "invalid dimensions"), (dict(Tq=1 << 28), "invalid dimensions"),
    (dict(Tk=2 ** 31 - 1), "invalid dimensions"), (dict(Hkv=3), "invalid dimensions"), (dict(Hkv=0), "invalid dimensions"),
    (dict(D=257), "invalid dimensions"), (dict(dtype=E4M3), "invalid dimensions"), (dict(qs=-1), "invalid dimensions"),
    (dict(cu_k=None), "invalid dimensions"), (dict(scale=0.0), "scale must be positive and finite"),
    (dict(window=-1), "sinks must not be negative and need a window"),
    (dict(sinks=4), "sinks must not be negative and need a window"), (dict(q=None), "null tensor pointer"),
    (dict(k=None), "null tensor pointer"), (dict(out=None), "null tensor pointer"), (dict(cu=None), "null tensor pointer")])
def test_prefill_launch_argument_errors(over, message):
    a = prefill_args()
    a.update(over)
    assert cabi.lib().qd_gqa_prefill(*a.values()) == 1
    assert cabi.error_string(1) == message


def test_prefill_without_queries_is_a_no_op():
    a = prefill_args()
    a.update(Tq=0, q=None, out=None)
    assert cabi.lib().qd_gqa_prefill(*a.values()) == 0


def test_prefill_plans_fit_the_launch():
    """Every row has a workgroup, and the grid fits, at the largest sizes too."""
    generic = cabi.QD_FLAG_FORCE_GENERIC
    assert cabi.gqa_prefill_info(1, 10, 10, 8, 2, 64, BF16, generic)[:2] == (0, 80)
    assert cabi.gqa_prefill_info(1, 10, 10, 7, 2, 64)[0] == -1
    assert cabi.gqa_prefill_info(1, 10, 10, 1 << 13, 8, 256, BF16)[0] == 1
    assert cabi.gqa_prefill_info(1, 10, 10, 1 << 14, 8, 256, BF16)[0] == 0  # a token's heads: 2^21 elements at most
    for B, Tq, Hq, Hkv, D in ((1, 1, 1, 1, 64), (16, 20000, 32, 8, 128), (1000, 7, 71, 1, 64), (3, 50, 4, 4, 256),
                              ((1 << 24) - 1, 1, 1, 1, 64), (1, (1 << 31) // 32 - 1, 32, 1, 128)):
        for dtype in (F32, F16, BF16):
            kind, grid, rows = cabi.gqa_prefill_info(B, Tq, Tq, Hq, Hkv, D, dtype)
            assert kind >= 0 and 0 < grid < 1 << 31
            if kind == 1:
                assert rows * (grid // Hkv) >= Tq * (Hq // Hkv)
            assert cabi.lib().qd_gqa_prefill_workspace_bytes(B, Tq, Tq, Hq, Hkv, D, dtype, 0, 0, 0) < 1 << 40


def test_prefill_splits_keys_of_few_rows():
    size = cabi.lib().qd_gqa_prefill_workspace_bytes
    assert cabi.gqa_prefill_info(1, 16, 30000, 8, 2, 128, BF16)[1] == 2 * 2 * 32
    row = 4 * 16 * 8 * 132                                        # bytes of a part
    assert size(1, 16, 30000, 8, 2, 128, BF16, 0, 0, 0) == 32 * row
    assert size(1, 16, 1000, 8, 2, 128, BF16, 0, 0, 0) == 7 * row    # of 128 keys or more
    assert size(1, 16, 391, 8, 2, 128, BF16, 0, 0, 0) == 0           # few keys
    assert size(1, 16, 391, 8, 2, 128, F32, 0, 0, 0) == 5 * row
    assert size(1, 16, 30000, 8, 2, 128, BF16, 300, 0, 0) == 0       # few that a row sees
    assert size(1, 16, 30000, 8, 2, 128, BF16, 900, 900, 0) == 14 * row
    assert size(1, 3100, 30000, 8, 2, 128, BF16, 0, 0, 0) == 2 * row * 3100 // 16  # two workgroups beside each other
    assert size(1, 3100, 30000, 8, 2, 256, BF16, 0, 0, 0) == 0       # too wide for that
    assert size(1, 1 << 14, 30000, 8, 2, 128, BF16, 0, 0, 0) == 0    # many rows
    assert size(1, 400, 400, 8, 2, 128, BF16, 0, 0, 0) == 0          # a prompt that sees itself
    assert size(1, 16, 30000, 8, 2, 128, BF16, 0, 0, cabi.QD_FLAG_FORCE_GENERIC) == 0
    a = prefill_args()
    a.update(B=1, Tq=16, Tk=30000, dtype=BF16, window=0, sinks=0)
    need = size(1, 16, 30000, a["Hq"], a["Hkv"], a["D"], BF16, 0, 0, 0)
    assert need > 0
    for over in (dict(ws=None, ws_bytes=need), dict(ws=24, ws_bytes=need), dict(ws=32, ws_bytes=need - 1)):
        a.update(over)
        assert cabi.lib().qd_gqa_prefill(*a.values()) == 1
        assert cabi.error_string(1) == "workspace too small or not 16-byte aligned"


# ---- 8-bit caches --------------------------------------------------------------


def rows_descs():
    return dict(key=desc([40, 2, 64], BF16), value=desc([40, 2, 64], BF16), kc=desc([9, 16, 2, 64], E4M3),
                vc=desc([9, 16, 2, 64], E4M3), ks=desc([9, 2], F32), vs=desc([9, 2], F32), table=desc([4, 3], I32),
                at=desc([4], I32), cu=desc([5], I32))


ROWS_ORDER = [
    (_edit("kc", is_device=0), "all tensors must be CUDA tensors"),
    (_edit("table", device_index=1), "all tensors must share a device"),
    (_edit("value", contiguous=0), "the heads of a token must be contiguous in key and value"),
    (_edit("vs", contiguous=0), "caches, scales and metadata must be contiguous"),
    (_edit("cu", contiguous=0), "caches, scales and metadata must be contiguous"),
    (_edit("key", sizes=[40, 128]), "key/value must be [T, Hkv, D]"),
    (_edit("value", sizes=[40, 2, 32]), "key/value must be [T, Hkv, D]"),
    (_edit("kc", sizes=[9, 16, 128]), "cache must be [Nblocks, P, Hkv, D]"),
    (_edit("vc", sizes=[9, 8, 2, 64]), "cache must be [Nblocks, P, Hkv, D]"),
    (_all(_edit("kc", sizes=[9, 16, 1, 64]), _edit("vc", sizes=[9, 16, 1, 64])), "cache head shape mismatch"),
    (_all(_edit("kc", sizes=[0, 16, 2, 64]), _edit("vc", sizes=[0, 16, 2, 64])), "invalid dimensions"),
    (_all(*(_edit(x, sizes=[40, 2, 257]) for x in ("key", "value")), *(_edit(x, sizes=[9, 16, 2, 257]) for x in ("kc", "vc"))),
     "supported head_dim is [1, 256]"),
    (_edit("ks", sizes=[9, 3]), "scales must be float32 [Nblocks, Hkv]"),
    (_edit("vs", dtype=BF16), "scales must be float32 [Nblocks, Hkv]"),
    (_edit("table", sizes=[3, 3]), "invalid metadata shape"),
    (_edit("at", sizes=[4, 1]), "invalid metadata shape"),
    (_edit("at", dtype=I64), "metadata must be int32"),
    (_edit("cu", sizes=[4]), "cu_seqlens must be int32 [B + 1]"),
    (_edit("key", dtype=E4M3), "unsupported dtype"),
    (_edit("value", dtype=F16), "dtype mismatch"),
    (_edit("vc", dtype=I8), "caches must both be float8_e4m3fn or int8"),
    (_all(_edit("kc", dtype=BF16), _edit("vc", dtype=BF16)), "caches must both be float8_e4m3fn or int8"),
    (_all(_edit("key", sizes=[1 << 31, 2, 64]), _edit("value", sizes=[1 << 31, 2, 64])),
     "tensor sizes exceed int32 CUDA launch limits"),
]


def test_rows_validation():
    _in_order(lambda d: cabi.validate_kv_append_q8(*d.values()), rows_descs, ROWS_ORDER)
    _in_order(lambda d: cabi.validate_kv_gather_q8(*d.values()), rows_descs, ROWS_ORDER)
    d = rows_descs()
    d["cu"] = None
    assert cabi.validate_kv_append_q8(*d.values()) == (1, "without cu_seqlens there must be one token per sequence")
    assert cabi.validate_kv_gather_q8(*d.values()) == (1, "cu_seqlens must be int32 [B + 1]")
    d["key"], d["value"] = desc([4, 2, 64], BF16), desc([4, 2, 64], BF16)
    assert cabi.validate_kv_append_q8(*d.values()) == (0, "")


def rows_args():
    return dict(key=1 << 20, value=1 << 21, kc=1 << 22, vc=1 << 23, ks=1 << 24, vs=1 << 25, table=16, at=16, cu=16, B=4,
                T=40, Hkv=2, D=64, P=16, maxP=3, N=9, k_stride=128, v_stride=128, dtype=BF16, cache=E4M3, stream=None)


@pytest.mark.parametrize("over, message", [
    (dict(B=1 << 24), "batch and tokens must be >= 0, batch below 2^24"),
    (dict(T=-1), "batch and tokens must be >= 0, batch below 2^24"), (dict(Hkv=0), "invalid dimensions"),
    (dict(P=0), "invalid dimensions"), (dict(N=0), "invalid dimensions"), (dict(N=1 << 31), "invalid dimensions"),
    (dict(k_stride=-1), "invalid dimensions"), (dict(D=0), "supported head_dim is [1, 256]"),
    (dict(dtype=I8), "unsupported dtype"), (dict(cache=BF16), "unsupported dtype"), (dict(key=None), "null tensor pointer"),
    (dict(vs=None), "null tensor pointer"), (dict(table=None), "null tensor pointer")])
def test_rows_launch_argument_errors(over, message):
    a = rows_args()
    a.update(over)
    for call in (cabi.lib().qd_kv_append_q8, cabi.lib().qd_kv_gather_q8):
        assert call(*a.values()) == 1
        assert cabi.error_string(1) == message


def test_append_refuses_overlap_and_missing_rows():
    pool = 9 * 16 * 2 * 64
    for over, message in ((dict(vc=1 << 22), "k_cache and v_cache must not overlap"),
                          (dict(vc=(1 << 22) + pool - 1), "k_cache and v_cache must not overlap"),
                          (dict(kc=(1 << 23) + pool - 1), "k_cache and v_cache must not overlap"),
                          (dict(vs=(1 << 24) + 68), "k_scales and v_scales must not overlap"),
                          (dict(cu=None), "without cu_seqlens there must be one token per sequence"),
                          (dict(T=2 ** 31 - 1, P=1), "tensor sizes exceed int32 CUDA launch limits")):
        a = rows_args()
        a.update(over)
        assert cabi.lib().qd_kv_append_q8(*a.values()) == 1
        assert cabi.error_string(1) == message
    a = rows_args()
    a.update(cu=None)
    assert cabi.lib().qd_kv_gather_q8(*a.values()) == 1 and cabi.error_string(1) == "null tensor pointer"
    for over in (dict(T=0), dict(B=0)):
        a = rows_args()
        a.update(over, key=None, kc=None)
        assert cabi.lib().qd_kv_append_q8(*a.values()) == 0 and cabi.lib().qd_kv_gather_q8(*a.values()) == 0


def test_gather_refuses_rows_that_overlap():
    for over in (dict(k_stride=0), dict(v_stride=127), dict(k_stride=64)):
        a = rows_args()
        a.update(over)
        assert cabi.lib().qd_kv_gather_q8(*a.values()) == 1
        assert cabi.error_string(1) == "rows of key and value must not overlap"


def test_launches_beyond_the_grid_are_refused():
    text = "tensor sizes exceed int32 CUDA launch limits"
    a = prefill_args()
    a.update(Tq=1 << 22, Tk=1 << 22, cu_k=None, flags=cabi.QD_FLAG_FORCE_GENERIC)   # 2^25 rows
    assert cabi.lib().qd_gqa_prefill(*a.values()) == 1 and cabi.error_string(1) == text
    a = prefill_args()
    a.update(B=1 << 23, Tq=1 << 23, Tk=1 << 23, cu_k=None)
    assert cabi.lib().qd_gqa_prefill(*a.values()) == 1 and cabi.error_string(1) == text
    a = rows_args()
    a.update(T=1 << 30, P=16)
    assert cabi.lib().qd_kv_append_q8(*a.values()) == 1 and cabi.error_string(1) == text
    assert cabi.lib().qd_kv_gather_q8(*a.values()) == 1 and cabi.error_string(1) == text


def decode_descs():
    return dict(q=desc([4, 8, 64], F16), kc=desc([9, 16, 2, 64], I8), vc=desc([9, 16, 2, 64], I8), ks=desc([9, 2], F32),
                vs=desc([9, 2], F32), table=desc([4, 3], I32), lens=desc([4], I32))


DECODE_ORDER = [
    (_edit("q", is_device=0), "q must be a CUDA tensor"), (_edit("q", contiguous=0), "q must be contiguous"),
    (_edit("ks", is_device=0), "k_scales must be a CUDA tensor"), (_edit("vs", contiguous=0), "v_scales must be contiguous"),
    (_edit("lens", contiguous=0), "context_lens must be contiguous"),
    (_edit("q", sizes=[4, 512]), "q must be [B, Hq, D]"),
    (_edit("kc", sizes=[9, 16, 128]), "k_cache must be [Nblocks, BlockSize, Hkv, D]"),
    (_edit("vc", sizes=[9, 16, 2, 32]), "v_cache shape mismatch"),
    (_edit("ks", sizes=[9, 1]), "scales must be float32 [Nblocks, Hkv]"),
    (_edit("vs", dtype=F16), "scales must be float32 [Nblocks, Hkv]"),
    (_edit("table", sizes=[4]), "block_table must be [B, MaxPages]"), (_edit("lens", sizes=[4, 1]), "context_lens must be [B]"),
    (_edit("table", device_index=1), "all tensors must use one CUDA device"),
    (_edit("q", dtype=F32), "q must be float16/bfloat16"),
    (_edit("kc", dtype=E4M3), "caches must both be float8_e4m3fn or int8"),
    (_all(_edit("kc", dtype=F16), _edit("vc", dtype=F16)), "caches must both be float8_e4m3fn or int8"),
    (_edit("lens", dtype=I64), "block_table and context_lens must be int32"), (_edit("lens", sizes=[3]), "batch sizes must match"),
    (_edit("q", sizes=[4, 8, 32]), "q head_dim and cache head_dim must match"),
    (_edit("q", sizes=[4, 7, 64]), "Hq must be divisible by Hkv"),
    (_edit("table", sizes=[4, 0]), "block_table must have at least one page"),
    (_all(_edit("q", sizes=[1 << 22, 8, 64]), _edit("table", sizes=[1 << 22, 3]), _edit("lens", sizes=[1 << 22])),
     "tensor sizes exceed int32 CUDA launch limits"),
]


def test_decode_validation():
    _in_order(lambda d: cabi.validate_gqa_decode_q8(*d.values()), decode_descs, DECODE_ORDER)
    for scale in (0.0, -1.0, float("nan")):
        assert cabi.validate_gqa_decode_q8(*decode_descs().values(), scale=scale) == (1, "scale must be positive and finite")


def decode_args():
    return dict(q=16, kc=16, vc=16, ks=16, vs=16, table=16, lens=16, out=16, ws=16, ws_bytes=1 << 40, B=4, Hq=8, Hkv=2,
                D=64, P=16, maxP=300, N=9, dtype=F16, cache=E4M3, scale=0.1, flags=0, stream=None)


@pytest.mark.parametrize("over, message", [
    (dict(B=-1), "invalid dimensions"), (dict(B=1 << 22), "invalid dimensions"), (dict(Hkv=3), "invalid dimensions"),
    (dict(dtype=F32), "invalid dimensions"), (dict(cache=F16), "invalid dimensions"), (dict(N=0), "invalid dimensions"),
    (dict(N=1 << 31), "invalid dimensions"), (dict(D=257), "invalid dimensions"), (dict(maxP=0), "invalid dimensions"),
    (dict(scale=float("nan")), "scale must be positive and finite"), (dict(vs=None), "null tensor pointer"),
    (dict(ws=None), "workspace too small or not 16-byte aligned"), (dict(ws=24), "workspace too small or not 16-byte aligned"),
    (dict(ws_bytes=8), "workspace too small or not 16-byte aligned")])
def test_decode_launch_argument_errors(over, message):
    a = decode_args()
    a.update(over)
    assert cabi.lib().qd_gqa_decode_q8(*a.values()) == 1
    assert cabi.error_string(1) == message


def test_decode_without_sequences_is_a_no_op():
    a = decode_args()
    a.update(B=0, q=None)
    assert cabi.lib().qd_gqa_decode_q8(*a.values()) == 0


def test_decode_plans_at_the_largest_sizes():
    """Workspaces and grids stay within what a launch takes, whatever the table's width."""
    for B, Hq, Hkv, D in ((1, 1, 1, 64), (1, 32, 8, 128), (64, 64, 8, 128), (1 << 20, 8, 8, 64), (300, 40, 1, 256)):
        for P, maxP in ((16, 1), (16, 4096), (1, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (48, 1000)):
            for flags in (0, cabi.QD_FLAG_FORCE_GENERIC):
                kind, grid = cabi.gqa_decode_q8_info(B, Hq, Hkv, D, P, maxP, BF16, flags)
                assert kind >= 0 and 0 < grid < 1 << 31
                assert cabi.lib().qd_gqa_decode_q8_workspace_bytes(B, Hq, Hkv, D, P, maxP, BF16, flags) < 1 << 36
    assert cabi.gqa_decode_q8_info(4, 7, 2, 64, 16, 3)[0] == -1


# ---- Torch ops and Python API --------------------------------------------------


def test_op_schemas():
    ops = torch.ops.qd_serving
    assert str(ops.gqa_prefill.default._schema) == (
        "qd_serving::gqa_prefill(Tensor q, Tensor key, Tensor value, Tensor cu_seqlens, Tensor? cu_seqlens_k, "
        "float scale, int window, int sinks) -> Tensor")
    assert str(ops.kv_append_q8.default._schema) == (
        "qd_serving::kv_append_q8(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, "
        "Tensor(c!) k_scales, Tensor(d!) v_scales, Tensor block_table, Tensor positions, Tensor? cu_seqlens) -> ()")
    assert str(ops.kv_gather_q8.default._schema) == (
        "qd_serving::kv_gather_q8(Tensor(a!) key, Tensor(b!) value, Tensor k_cache, Tensor v_cache, Tensor k_scales, "
        "Tensor v_scales, Tensor block_table, Tensor context_lens, Tensor cu_seqlens) -> ()")
    assert str(ops.gqa_decode_q8.default._schema) == (
        "qd_serving::gqa_decode_q8(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, "
        "Tensor block_table, Tensor context_lens, float scale) -> Tensor")


def test_public_names_and_missing_extension(monkeypatch):
    for name in ("gqa_prefill", "kv_append_q8", "kv_gather_q8", "gqa_decode_q8"):
        assert name in attention_amd.__all__
    q = torch.zeros(1, 2, 4)
    with pytest.raises(NotImplementedError):
        attention_amd.gqa_prefill(q, q, q, q)
    with pytest.raises(ValueError, match="window must be positive, or None"):
        attention_amd.gqa_prefill(q, q, q, q, window=0)
    monkeypatch.setattr(core, "_LOAD_ERROR", OSError("missing"))
    for call in (lambda: attention_amd.gqa_prefill(q, q, q, q), lambda: attention_amd.kv_append_q8(*[q] * 8),
                 lambda: attention_amd.kv_gather_q8(*[q] * 9), lambda: attention_amd.gqa_decode_q8(*[q] * 7)):
        with pytest.raises(RuntimeError, match=r"^qd_attention CUDA extension was not loaded$"):
            call()


def test_other_operators_refuse_8_bit_caches():
    """Rows of a cache with scales per page cannot move between pages: kv_compact has no dtype code for them."""
    assert cabi.validate_kv_compact(desc([9, 16, 2, 64], E4M3), desc([4, 3], I32), desc([4], I32), desc([4, 8], I32))[0] == 1
    assert cabi.validate_kv_compact(desc([9, 16, 2, 64], I8), desc([4, 3], I32), desc([4], I32), desc([4, 8], I32))[0] == 1


# ---- The oracle ------------------------------------------------------------------


def test_oracle_rounding_is_torchs():
    x = np.concatenate([np.linspace(-448, 448, 20001), np.ldexp(1.0, np.arange(-12, 9)), [0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0]])
    want = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(round_to(x.astype(np.float32), "e4m3"), want)
    assert np.array_equal(round_to([0.5, 1.5, -2.5, 126.5], "int8"), [0, 2, -2, 126])
    assert power_scale(448.0, "e4m3") == 1 and power_scale(448.1, "e4m3") == 2 and power_scale(0.0, "int8") == 2.0 ** -100
    assert power_scale(127.0, "int8") == 1 and power_scale(63.0, "int8") == 0.5 and np.isnan(power_scale(np.inf, "int8"))


def test_oracle_prefill_closed_forms():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((5, 2, 4)), rng.standard_normal((5, 1, 4)), rng.standard_normal((5, 1, 4))
    out, _, _ = oracle_prefill(q, k, v, [0, 2, 5], None, 0, 0, 0.5)
    assert np.array_equal(out[0], np.repeat(v[0], 2, 0)) and np.array_equal(out[2], np.repeat(v[2], 2, 0))
    out, _, _ = oracle_prefill(q, k, v, [0, 2, 5], None, 1, 0, 0.5)
    assert np.allclose(out, np.repeat(v, 2, 1))                       # a window of one: the own value
    out, _, _ = oracle_prefill(0 * q, k, v, [0, 5], None, 2, 1, 0.5)
    assert np.allclose(out[4, 0], (v[0] + v[3] + v[4])[0] / 3)       # two last ones and the first, equal scores
    out, _, _ = oracle_prefill(q, k, v, [0, 3], [0, 1], 0, 0, 0.5)
    assert not out[:2].any() and np.allclose(out[2], np.repeat(v[0], 2, 0)) and not out[3:].any()
    # Torch's own product of the same.
    mask = torch.ones(5, 5, dtype=torch.bool).tril()
    want = torch.nn.functional.scaled_dot_product_attention(
        *(torch.from_numpy(np.repeat(x, 2 // x.shape[1], 1).transpose(1, 0, 2).copy()) for x in (q, k, v)), attn_mask=mask, scale=0.5)
    out, _, _ = oracle_prefill(q, k, v, [0, 5], None, 0, 0, 0.5)
    assert np.allclose(out, want.numpy().transpose(1, 0, 2))


def test_oracle_append_and_decode():
    rng = np.random.default_rng(1)
    rows = rng.standard_normal((6, 1, 4))
    cache, scales = np.zeros((3, 4, 1, 4)), np.zeros((3, 1))
    table = np.array([[2, 0]])
    for kind, part in (("int8", 0.5 / 63), ("e4m3", 2.0 ** -4)):
        kc, vc, ks, vs = oracle_append(rows, rows * 8, cache, cache, scales, scales, table, [0], [0, 6], kind)
        values = (kc * ks[:, :, None, None]).reshape(-1, 4)
        got = values[[8, 9, 10, 11, 0, 1]]
        assert np.abs(got - rows[:, 0]).max() <= part * np.abs(rows).max() and not kc[1].any() and not kc[0, 2:].any()
        assert np.array_equal(kc * ks[:, :, None, None] * 8, vc * vs[:, :, None, None])   # a power of two apart
        out, _, _, _ = oracle_decode(np.zeros((1, 2, 4)), kc, vc, ks, vs, table, [6], 1.0)
        assert np.allclose(out[0, 0], got.mean(0) * 8)
        # One more token, nine times as large: the page's rows go to the larger scale.
        k2, _, k2s, _ = oracle_append(90 * rows[:1], rows[:1], kc, vc, ks, vs, table, [6], None, kind)
        assert k2s[0, 0] > ks[0, 0] and np.array_equal(k2[2], kc[2]) and np.array_equal(k2s[1:], ks[1:])
        moved = np.abs(k2[0, :2] * k2s[0, 0] - kc[0, :2] * ks[0, 0]).max()
        assert moved <= k2s[0, 0] * (0.5 if kind == "int8" else 2.0 ** -10) + (kind == "e4m3") * 2.0 ** -4 * np.abs(rows).max()
