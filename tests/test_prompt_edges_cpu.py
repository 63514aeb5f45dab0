"""CPU checks of prompt attention and of 8-bit caches at the ends of their ranges.  No
kernel runs here."""
from __future__ import annotations

import os

import pytest

from attention_amd import _build, cabi
from tests.test_prompt_boundary_cpu import rows_args


def test_append_refuses_runs_past_32_bits():
    """A wave counts a run's rows in 32 bits, in steps of up to 8 x 64: heads of one element, one page."""
    for over in (dict(T=2 ** 31 - 500, P=2 ** 31 - 1), dict(T=2 ** 31 - 400, P=2 ** 31 - 500)):
        a = rows_args()
        a.update(over, B=1, Hkv=1, D=1, maxP=1, N=1, k_stride=1, v_stride=1, vc=1 << 40, vs=1 << 41)
        assert cabi.lib().qd_kv_append_q8(*a.values()) == 1
        assert cabi.error_string(1) == "tensor sizes exceed int32 CUDA launch limits"


INCLUDED = {"packed.h": {"prefill", "prefill_mfma_bf16", "prefill_mfma_f16", "prefill_mfma_f32", "cache_q8", "decode_q8"},
            "prefill_kernels.h": {"prefill", "prefill_mfma_bf16", "prefill_mfma_f16", "prefill_mfma_f32"},
            "tree_kernels.h": {"tree_decode", "tree_mfma_bf16", "tree_mfma_f16", "tree_mfma_f32"},
            "torch_desc.h": {"torch_ops", "serving_ops", "prompt_ops"}}
INCLUDED["tile_device.h"] = INCLUDED["prefill_kernels.h"] | INCLUDED["tree_kernels.h"]
INCLUDED["qd_attention.h"] = set(_build.HIP_SOURCES) | set(_build.TORCH_SOURCES)
INCLUDED["qd_device.h"] = set(_build.HIP_SOURCES) - {"kv_append", "validate"}


@pytest.mark.parametrize("header", INCLUDED)
def test_a_changed_header_rebuilds_what_includes_it(monkeypatch, tmp_path, header):
    """An incremental build compiles every source again that includes a changed header, directly or through another."""
    monkeypatch.setattr(_build, "OBJ_DIR", str(tmp_path))
    for name in _build.HIP_SOURCES + _build.TORCH_SOURCES:
        (tmp_path / f"{name}.o").write_bytes(b"")
    monkeypatch.setattr(_build.os.path, "getmtime",
                        lambda p: {".o": 1.0}.get(os.path.splitext(p)[1], 2.0 if os.path.basename(p) == header else 0.0))
    stale = {n for n in _build.HIP_SOURCES if _build._stale(n)} | {n for n in _build.TORCH_SOURCES if _build._torch_stale(n)}
    assert stale == INCLUDED[header]
