"""CPU checks of prompt attention and of 8-bit caches at the ends of their ranges.  No
kernel runs here."""
from __future__ import annotations

from attention_amd import cabi
from tests.test_prompt_boundary_cpu import rows_args


def test_append_refuses_runs_past_32_bits():
    """A wave counts a run's rows in 32 bits, in steps of up to 8 x 64: heads of one element, one page."""
    for over in (dict(T=2 ** 31 - 500, P=2 ** 31 - 1), dict(T=2 ** 31 - 400, P=2 ** 31 - 500)):
        a = rows_args()
        a.update(over, B=1, Hkv=1, D=1, maxP=1, N=1, k_stride=1, v_stride=1, vc=1 << 40, vs=1 << 41)
        assert cabi.lib().qd_kv_append_q8(*a.values()) == 1
        assert cabi.error_string(1) == "tensor sizes exceed int32 CUDA launch limits"
