"""GPU parity of prompt attention and of 8-bit caches (append, gather, decode)
against the float64 oracle, and what a caller can run into: sequences without
tokens, more queries than keys, hidden tokens that hold NaN, strided views, pages
that end inside a tile, other streams, captured graphs, unaligned tensors, pools
past 2^32 bytes.  Every case prints its name first.

Tolerances, u = 2^-24 and h = half a step of the output type relative to the
value (fp32 2^-24, fp16 2^-11, bf16 2^-8):
  prefill    a score of D terms is off by at most (D + 4) u S, S its sum of
             |q k| scale; a softmax weight by twice that and 8 u of the two
             exponentials, relatively; n summed terms by n u; 16-bit weights are
             rounded once, by h.  fp16 weights lie on a grid of 2^-24, with the
             largest at least 2^7: n 2^-32 of the largest value.  Times
             sum(weight |v|), plus the output's rounding h |out|.
  decode     the same over cached values; weights go in as fp16, times the scale
             of their page, the largest such product at least 2^7: rounded by
             2^-11, and n 2^-32 of that product times the type's largest element.
             bf16 queries go in as fp16 with the largest in [2^14, 2^15): off by
             2^-25 of 2^14 each, D 2^-39 max|q| max|k| scale of a score.
  append     elements and scales are determined: equal.
  gather     one rounding of element times scale: equal.
Below the smallest normal number the rounding step is fixed: 2^-25 for fp16.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_amd
from attention_amd import cabi
from oracle.prompt_oracle import TOP, cached_rows, oracle_append, oracle_decode, oracle_prefill

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
HALF = {FP: 2.0 ** -24, HF: 2.0 ** -11, BF: 2.0 ** -8}
WEIGHT = {FP: 0.0, HF: 2.0 ** -11, BF: 2.0 ** -8}
TINY = {FP: 2.0 ** -149, HF: 2.0 ** -25, BF: 2.0 ** -133}
CACHE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def say(msg):
    print(f"[case] {msg}", flush=True)


def f64(x):
    return x.detach().cpu().double().numpy()


def starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)


def worst_of(got, want, tol, what):
    assert np.isfinite(got).all(), f"{what}: not finite"
    worst = (np.abs(got - want) / tol).max() if got.size else 0.0
    say(f"{what}: {worst:.3f} of the tolerance")
    assert worst <= 1.0, what


# ---- Prompt attention --------------------------------------------------------


def prefill_case(dtype, nq, nk, Hq, Hkv, D, *, seed=0, spare=3, k_scale=1.5):
    """nk None: as many keys as queries.  ``spare`` rows follow the last sequence."""
    gen = torch.Generator().manual_seed(seed)
    cu, cu_k = starts(nq), None if nk is None else starts(nk)
    Tq = int(cu[-1]) + spare
    Tk = Tq if nk is None else int(cu_k[-1]) + spare
    q = torch.randn(Tq, Hq, D, generator=gen).to(dtype)
    k = (k_scale * torch.randn(Tk, Hkv, D, generator=gen)).to(dtype)
    v = torch.randn(Tk, Hkv, D, generator=gen).to(dtype)
    return q, k, v, cu, cu_k


def prefill(gpu, case, window=0, sinks=0, flags=None, scale=None):
    d = [x if x is None else x.to(gpu) for x in case]
    if flags is not None:
        out = torch.full_like(d[0], float("nan"))
        rc = cabi.gqa_prefill(*d, out, scale=scale or 1 / math.sqrt(out.shape[-1]), window=window, sinks=sinks, flags=flags)
        assert rc == 0, cabi.error_string(rc)
    else:
        out = attention_amd.gqa_prefill(*d[:4], cu_seqlens_k=d[4], window=window or None, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    return out


def prefill_tolerance(case, want, spread, size):
    q, k, v, cu, cu_k = case
    n, D = int((cu if cu_k is None else cu_k).diff().max()), q.shape[-1]
    rel = 2 * (D + 4) * U * size[..., None] + 8 * U + 2 * n * U + WEIGHT[q.dtype]
    grid = n * 2.0 ** -32 * v[v.isfinite()].abs().max().item() if q.dtype == HF else 0.0
    return HALF[q.dtype] * np.abs(want) + rel * spread + grid + TINY[q.dtype]


def check_prefill(gpu, case, window=0, sinks=0, flags=None, what="", scale=None):
    q, k, v, cu, cu_k = case
    want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), None if cu_k is None else cu_k.tolist(),
                                        window, sinks, scale or 1 / math.sqrt(q.shape[-1]))
    out = prefill(gpu, case, window, sinks, flags, scale)
    assert out.dtype == q.dtype and out.is_contiguous()
    worst_of(f64(out), want, prefill_tolerance(case, want, spread, size), what)
    return out


PREFILL = [
    # dtype, queries, keys (None: the same), Hq, Hkv, D, window, sinks
    (BF, [1], None, 1, 1, 64, 0, 0),
    (BF, [2, 1, 0, 3], None, 4, 2, 128, 0, 0),
    (BF, [100], None, 8, 2, 128, 0, 0),
    (HF, [63, 65, 1], None, 8, 2, 128, 0, 0),
    (BF, [128, 129], None, 4, 4, 64, 0, 0),
    (HF, [200], None, 2, 1, 64, 0, 0),
    (BF, [70, 0, 31], None, 5, 1, 96, 0, 0),
    (HF, [90], None, 14, 2, 80, 0, 0),
    (BF, [65], None, 6, 2, 72, 0, 0),
    (BF, [75, 20], None, 4, 1, 256, 0, 0),
    (HF, [66], None, 2, 2, 192, 0, 0),
    (BF, [40, 33], None, 4, 2, 8, 0, 0),
    (FP, [70, 5], None, 4, 2, 128, 0, 0),
    (FP, [33], None, 2, 1, 64, 0, 0),
    (FP, [20, 40], None, 3, 1, 256, 0, 0),
    (FP, [25], None, 2, 1, 20, 0, 0),
    (BF, [30], None, 3, 1, 33, 0, 0),            # rows of no whole 16 bytes
    (HF, [17], None, 2, 1, 1, 0, 0),
    (BF, [1], None, 71, 1, 64, 0, 0),            # a group wider than a tile's rows of one token
    (BF, [3, 40], None, 40, 1, 128, 0, 0),
    (BF, [10, 3, 70], [100, 200, 70], 8, 2, 128, 0, 0),       # chunks after a context
    (HF, [1, 1, 1], [1, 64, 300], 8, 2, 64, 0, 0),
    (BF, [50, 4], [20, 0], 4, 2, 128, 0, 0),     # more queries than keys: the first see nothing
    (FP, [30], [7], 2, 1, 64, 0, 0),
    (BF, [150], None, 4, 2, 128, 32, 0),
    (BF, [150, 90], None, 4, 2, 128, 1, 0),
    (HF, [200], None, 4, 2, 64, 64, 4),
    (BF, [260], None, 2, 1, 128, 50, 70),
    (HF, [20, 130], [300, 131], 6, 2, 96, 100, 3),
    (FP, [100], None, 2, 1, 64, 30, 2),
    (BF, [80], [200], 4, 1, 256, 65, 1),
    (BF, [90], None, 4, 2, 128, 1 << 30, 5),
]


@pytest.mark.parametrize("i", range(len(PREFILL)))
@pytest.mark.parametrize("flags", [None, cabi.QD_FLAG_FORCE_GENERIC])
def test_prefill(gpu, i, flags):
    dtype, nq, nk, Hq, Hkv, D, window, sinks = PREFILL[i]
    say(f"prefill {i} {PREFILL[i]} flags {flags}")
    out = check_prefill(gpu, prefill_case(dtype, nq, nk, Hq, Hkv, D, seed=i), window, sinks, flags, f"prefill {i}")
    assert not out[sum(nq):].any()  # behind the last sequence


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_prefill_projection_views(gpu, dtype):
    say(f"views {dtype}")
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(150, 8 + 2 + 2, 64, generator=gen).to(dtype).to(gpu)
    q, k, v = qkv.split([8, 2, 2], dim=1)
    cu = starts([70, 80]).to(gpu)
    got = attention_amd.gqa_prefill(q, k, v, cu)
    want = attention_amd.gqa_prefill(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(got, want)
    one = qkv[:1].expand(150, -1, -1)  # stride 0: one token for all
    got = attention_amd.gqa_prefill(*one.split([8, 2, 2], dim=1), cu)
    assert torch.allclose(got.float(), one[:, 10:].repeat_interleave(4, 1).float(), rtol=2 * HALF[dtype] + WEIGHT[dtype] + 200 * U, atol=1e-30)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_prefill_unaligned(gpu, dtype):
    say(f"unaligned {dtype}")
    case = prefill_case(dtype, [40, 9], None, 4, 2, 64, seed=8)
    q, k, v, cu, _ = (x if x is None else x.to(gpu) for x in case)
    want = attention_amd.gqa_prefill(q, k, v, cu)
    shifted = []
    for x in (q, k, v):
        buf = torch.zeros(x.numel() + 1, dtype=dtype, device=gpu)
        buf[1:] = x.reshape(-1)
        shifted.append(buf[1:].view(x.shape))
    got = attention_amd.gqa_prefill(*shifted, cu)
    assert torch.allclose(got.float(), want.float(), rtol=4 * HALF[dtype], atol=2 * WEIGHT[dtype] + 1e-5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype, D, Hq", [(BF, 128, 4), (HF, 64, 2), (FP, 64, 2), (BF, 256, 1)])
@pytest.mark.parametrize("flags", [None, cabi.QD_FLAG_FORCE_GENERIC])
def test_prefill_hidden_values(gpu, bad, dtype, D, Hq, flags):
    """A value that is not finite reaches the rows that see it, and no other."""
    say(f"hidden {bad} {dtype} {D} flags {flags}")
    for window, sinks in ((0, 0), (20, 0), (20, 3)):
        case = prefill_case(dtype, [130, 70], None, Hq, 1, D, seed=3)
        q, k, v, cu, _ = case
        want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), None, window, sinks, 1 / math.sqrt(D))
        for token, col in ((60, 0), (129, 5), (2, 7), (131, D - 1)):
            v[token, 0, col] = bad
        k[128, 0, 1] = bad     # a key: every element of the rows that see it
        out = f64(prefill(gpu, case, window, sinks, flags))
        hit = np.zeros_like(want, dtype=bool)
        for t in range(200):
            b, i = (0, t) if t < 130 else (130, t - 130)
            sees = lambda j: b <= j <= t and (not window or j > t - window or j - b < sinks)  # noqa: E731
            for token, col in ((60, 0), (129, 5), (2, 7), (131, D - 1)):
                hit[t, :, col] |= sees(token)
            hit[t] |= sees(128)
        assert np.isfinite(out[~hit]).all()
        if not math.isnan(bad):  # an infinite key may hide itself: a score of -inf has no weight
            hit[128:130] = False
            assert not np.isfinite(out[hit]).any()
        else:
            assert np.isnan(out[hit]).all()
        clear = ~hit
        clear[128:130] = False
        tol = prefill_tolerance(case, want, spread, size)
        assert (np.abs(out - want)[clear] <= tol[clear]).all()


SPLIT = [
    # As above: few rows with many keys, whose keys several workgroups share.
    (BF, [16], [3000], 4, 2, 128, 0, 0),
    (HF, [5, 0, 7], [4000, 900, 10], 8, 2, 64, 0, 0),      # one sequence with all of the keys
    (BF, [40, 3], [20, 6000], 4, 4, 128, 0, 0),            # rows that see nothing beside a long one
    (BF, [3], [1200], 71, 1, 96, 0, 0),
    (HF, [30], [2500], 4, 1, 256, 1500, 40),
    (BF, [20], [9000], 2, 1, 128, 2000, 2100),             # more sinks than a part has keys
    (HF, [1, 1], [1024, 5000], 2, 2, 192, 1100, 0),
    (BF, [700, 20], [900, 1400], 16, 4, 128, 0, 0),        # two workgroups per CU
    (FP, [7], [1500], 4, 2, 64, 0, 0),
    (FP, [20, 3], [900, 700], 3, 1, 128, 300, 5),
    (FP, [1], [2000], 2, 1, 256, 0, 0),
]


@pytest.mark.parametrize("i", range(len(SPLIT)))
def test_prefill_split_keys(gpu, i):
    dtype, nq, nk, Hq, Hkv, D, window, sinks = SPLIT[i]
    say(f"split {i} {SPLIT[i]}")
    case = prefill_case(dtype, nq, nk, Hq, Hkv, D, seed=50 + i)
    bytes_ = cabi.lib().qd_gqa_prefill_workspace_bytes(len(nq), case[0].shape[0], case[1].shape[0], Hq, Hkv, D,
                                                       cabi.DTYPE[dtype], window, sinks, 0)
    assert bytes_ > 0
    torch.full((bytes_ // 4,), float("nan"), device=gpu)  # what the workspace holds before
    out = check_prefill(gpu, case, window, sinks, None, f"split {i}")
    assert not out[sum(nq):].any()


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prefill_split_hidden_values(gpu, bad, dtype):
    """As test_prefill_hidden_values, where the keys are split."""
    for window, sinks in ((0, 0), (1500, 2)):
        say(f"split hidden {dtype} {bad} window {window}")
        case = prefill_case(dtype, [6], [3000], 4, 2, 128, seed=9)
        q, k, v, cu, cu_k = case
        want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), cu_k.tolist(), window, sinks, 128 ** -0.5)
        places = ((2997, 0), (1497, 1), (1, 2), (700, 3))
        for token, col in places:
            v[token, :, col] = bad
        out = f64(prefill(gpu, case, window, sinks))
        hit = np.zeros_like(want, dtype=bool)
        for t in range(6):
            at = 2994 + t
            for token, col in places:
                hit[t, :, col] |= token <= at and (not window or token > at - window or token < sinks)
        assert hit.any() and not np.isfinite(out[hit]).any()
        tol = prefill_tolerance(case, want, spread, size)
        assert (np.abs(out - want)[~hit] <= tol[~hit]).all()


def test_prefill_split_bad_metadata_stays_inside(gpu):
    say("split bad metadata")
    q, k, v, _, _ = (x if x is None else x.to(gpu) for x in prefill_case(BF, [10], [3000], 4, 2, 64))
    for cu, cu_k in (([0, 500], [0, 1 << 30]), ([0, -5], [0, -9]), ([7, 9], [5, 2 ** 31 - 1]), ([-(1 << 31), 2 ** 31 - 1], [9, -(1 << 31)])):
        cu, cu_k = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in (cu, cu_k))
        assert cabi.gqa_prefill(q, k, v, cu, cu_k, torch.zeros_like(q), scale=0.1) == 0
    torch.cuda.synchronize()


def test_prefill_large_rows_of_64(gpu):
    """As many rows as make heads of 64 take twice the rows per wave; parity with the
    plain kernel, which the oracle has checked."""
    say("heads of 64, 256 rows")
    for dtype, window, sinks in ((BF, 0, 0), (HF, 100, 5)):
        counts = [3000, 1, 0, 1095]
        case = prefill_case(dtype, counts, None, 64, 8, 64, seed=12, spare=1)
        assert cabi.gqa_prefill_info(4, 4097, 4097, 64, 8, 64, cabi.DTYPE[dtype])[2] == 256
        out = prefill(gpu, case, window, sinks)
        plain = prefill(gpu, case, window, sinks, cabi.QD_FLAG_FORCE_GENERIC)
        # Both within their tolerance of the truth: spread at most the largest value,
        # scores of 64 terms at most 64 * 4.5 * 7 / 8.
        top = float(case[2].abs().max())
        tol = 2 * (HALF[dtype] + 2 * 68 * U * 252 + 8 * U + 6000 * U + WEIGHT[dtype]) * top + 3000 * 2.0 ** -32 * top
        assert (out.float() - plain.float()).abs().max().item() <= tol
        assert not out[4096:].any()
        # One sequence's rows against the oracle.
        part = tuple(x[3001:4096] for x in case[:3]) + (torch.tensor([0, 1095], dtype=torch.int32), None)
        want, spread, size = oracle_prefill(*(f64(x) for x in part[:3]), [0, 1095], None, window, sinks, 0.125)
        worst_of(f64(out[3001:4096]), want, prefill_tolerance(part, want, spread, size), "the last sequence")


def test_prefill_scores_of_all_sizes(gpu):
    """Scores far apart, rising and falling along the keys: the reference maximum moves."""
    for dtype in (BF, HF, FP):
        for sign in (1, -1):
            say(f"slopes {dtype} {sign}")
            q, k, v, cu, _ = prefill_case(dtype, [300], None, 2, 1, 64, seed=4)
            q[:] = 0
            q[:, :, 0] = 8
            k[:, :, 0] = (sign * torch.linspace(-60, 60, k.shape[0])[:, None]).to(dtype)
            check_prefill(gpu, (q, k, v, cu, None), what=f"slopes {dtype} {sign}", scale=1.0)


def test_prefill_bad_metadata_stays_inside(gpu):
    say("bad metadata")
    q, k, v, _, _ = (x if x is None else x.to(gpu) for x in prefill_case(BF, [100], None, 4, 2, 64))
    for cu, cu_k in (([0, 500, 1 << 30], None), ([0, -5, 103], None), ([7, 90, 20], None),
                     ([0, 50, 103], [0, 1 << 30, -9]), ([-(1 << 31), 2 ** 31 - 1, 0], [0, 2 ** 31 - 1, 4])):
        cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
        cu_k = None if cu_k is None else torch.tensor(cu_k, dtype=torch.int32, device=gpu)
        for flags in (0, cabi.QD_FLAG_FORCE_GENERIC):
            out = torch.zeros_like(q)
            assert cabi.gqa_prefill(q, k, v, cu, cu_k, out, scale=0.1, flags=flags) == 0
    torch.cuda.synchronize()


def test_prefill_empty(gpu):
    say("empty")
    q, k = torch.zeros(0, 4, 64, device=gpu, dtype=BF), torch.zeros(0, 2, 64, device=gpu, dtype=BF)
    cu = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert attention_amd.gqa_prefill(q, k, k, cu).shape == (0, 4, 64)
    q = torch.ones(5, 4, 64, device=gpu, dtype=BF)
    kk = torch.ones(5, 2, 64, device=gpu, dtype=BF)
    assert not attention_amd.gqa_prefill(q, kk, kk, cu).any()       # no sequences
    cu2 = torch.tensor([0, 5], dtype=torch.int32, device=gpu)
    none = torch.zeros(2, dtype=torch.int32, device=gpu)
    assert not attention_amd.gqa_prefill(q, k, k, cu2, cu_seqlens_k=none).any()   # no keys


def test_prefill_many_sequences(gpu):
    say("many sequences")
    gen = torch.Generator().manual_seed(6)
    counts = torch.randint(0, 6, (5000,), generator=gen).tolist()
    case = prefill_case(BF, counts, None, 2, 1, 64, seed=6)
    check_prefill(gpu, case, what="5000 sequences")


# ---- 8-bit caches --------------------------------------------------------------


def table_of(gen, used, spare):
    """Pages of their own for every sequence, scattered; ``spare`` more columns of -1."""
    width, total = max(max(used), 1) + spare, sum(used)
    ids = torch.randperm(total + 3, generator=gen)[:total].tolist()
    rows = []
    for n in used:
        rows.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
    return torch.tensor(rows, dtype=torch.int32), total + 3


def held(gen, kind, shape):
    x = torch.randn(*shape, generator=gen)
    return (x * 90).clamp(-448, 448).to(CACHE[kind]) if kind == "e4m3" else (x * 30).round().clamp(-127, 127).to(torch.int8)


def cache_case(kind, lens, more, Hkv, D, P, *, seed=0, power=True, spare=1):
    """Caches that hold ``lens`` tokens per sequence, with room for ``more`` each."""
    gen = torch.Generator().manual_seed(seed)
    table, N = table_of(gen, [-(-(max(n, 0) + m) // P) for n, m in zip(lens, more)], spare)
    kc, vc = held(gen, kind, (N, P, Hkv, D)), held(gen, kind, (N, P, Hkv, D))
    ks, vs = (torch.exp2(torch.randint(-9, -4, (N, Hkv), generator=gen).float()) for _ in range(2))
    if not power:
        ks, vs = ks * (1 + torch.rand(N, Hkv, generator=gen)), vs * (1 + torch.rand(N, Hkv, generator=gen))
    return kc, vc, ks, vs, table, gen


def bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def check_append(gpu, key, value, kc, vc, ks, vs, table, positions, cu, kind, what):
    d = [x.to(gpu) for x in (kc, vc, ks, vs)]
    attention_amd.kv_append_q8(key.to(gpu), value.to(gpu), *d, table.to(gpu), positions.to(gpu),
                               None if cu is None else cu.to(gpu))
    torch.cuda.synchronize()
    want = oracle_append(f64(key), f64(value), f64(kc), f64(vc), f64(ks), f64(vs), table.numpy(), positions.tolist(),
                         None if cu is None else cu.tolist(), kind)
    for name, x, y, scales in zip(("k", "v", "k_scales", "v_scales"), d, want, [*want[2:], None, None]):
        x = f64(x)
        same = (x == y) | (np.isnan(x) & np.isnan(y))
        if scales is not None:  # elements without a scale are unspecified
            same |= np.isnan(scales)[:, None, :, None]
        off = np.argwhere(~same)
        assert not len(off), f"{what}: {name} differs at {off[:4].tolist()}: {x[tuple(off[0])]} for {y[tuple(off[0])]}"
    return d


APPEND = [
    # dtype, kind, positions, tokens (None: one each, without cu), Hkv, D, P
    (BF, "e4m3", [0, 5, 16, 31], None, 2, 128, 16),
    (HF, "int8", [0, 1, 15], None, 1, 64, 16),
    (FP, "e4m3", [3, 64, 127], None, 3, 64, 64),
    (FP, "int8", [3, 64, 127], None, 2, 128, 64),
    (BF, "int8", [0, 7, 0, 33], [50, 1, 0, 70], 2, 64, 16),
    (BF, "e4m3", [0, 7, 30, 33], [100, 9, 2, 200], 2, 128, 32),
    (HF, "e4m3", [5, 0], [300, 129], 1, 96, 128),
    (HF, "int8", [5, 0], [3, 20], 5, 72, 7),
    (FP, "e4m3", [2, 0], [10, 20], 2, 20, 4),
    (BF, "e4m3", [0, 3], [5, 6], 2, 33, 16),     # element by element
    (HF, "int8", [0, 3], [25, 6], 1, 1, 16),
    (BF, "int8", [9, 0, 2], [4, 5, 6], 2, 80, 1),
    (BF, "e4m3", [10, 0], [700, 300], 1, 256, 256),  # runs longer than the registers hold
    (FP, "int8", [100, 0], [300, 500], 1, 256, 512),
    (BF, "e4m3", [5, 0, 127], [300, 128, 2], 2, 128, 128),  # twice the pieces per lane
    (FP, "int8", [3, 64], [100, 1], 2, 128, 64), (HF, "int8", [0, 70], [64, 200], 1, 256, 64),
]


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append(gpu, i):
    dtype, kind, at, counts, Hkv, D, P = APPEND[i]
    say(f"append {i} {APPEND[i]}")
    more = [1] * len(at) if counts is None else counts
    kc, vc, ks, vs, table, gen = cache_case(kind, at, more, Hkv, D, P, seed=i)
    cu = None if counts is None else starts(counts)
    rows = sum(more) + (2 if cu is not None else 0)
    size = torch.exp2(torch.randint(-4, 5, (rows, 1, 1), generator=gen).float())
    kv = (torch.randn(rows, 2 * Hkv, D, generator=gen) * size).to(dtype)
    key, value = kv.split([Hkv, Hkv], dim=1)
    check_append(gpu, key, value, kc, vc, ks, vs, table, torch.tensor(at, dtype=torch.int32), cu, kind, f"append {i}")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_append_edges_of_scales(gpu, kind, dtype):
    """Largest values next to the borders between scales, zeros, subnormal and largest numbers; ties."""
    say(f"edges {kind} {dtype}")
    gen = torch.Generator().manual_seed(1)
    top = TOP[kind]
    most = [0.0, top, top * 2, np.nextafter(np.float32(top), np.float32(1e9)), np.nextafter(np.float32(top), np.float32(0)),
            1.0, 0.875, 1.75, 127 / 128, 0.5, 2.0 ** -20, 1e-38, 1e-45, 2.0 ** -14, 2.0 ** -24, 6e4, 3e38, 2.0 ** -110]
    n = len(most)
    x = torch.tensor(np.array(most, dtype=np.float32)).to(dtype)[:, None, None] * torch.ones(1, 2, 64, dtype=dtype)
    x = torch.where(torch.isfinite(x), x, torch.tensor(1.0, dtype=dtype))
    steps = torch.randint(-512, 513, (n, 2, 64), generator=gen).to(dtype) / 512
    key, value = x.clone(), x.clone()
    key[:, :, 1:] = (x * steps)[:, :, 1:]
    value[:, :, 2:] = (x * steps)[:, :, 2:].flip(-1)
    kc, vc, ks, vs, table, _ = cache_case(kind, [0] * n, [1] * n, 2, 64, 16)
    check_append(gpu, key, value, kc, vc, ks, vs, table, torch.zeros(n, dtype=torch.int32), None, kind, "edges")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_not_finite(gpu, kind):
    say(f"not finite {kind}")
    kc, vc, ks, vs, table, gen = cache_case(kind, [3, 3, 0], [2, 2, 2], 2, 64, 16)
    key = torch.randn(6, 2, 64, generator=gen).to(BF)
    value = key.clone()
    key[0, 0, 3], key[3, 1, 5], value[5, 1, 63] = float("nan"), float("inf"), -float("inf")
    d = [x.to(gpu) for x in (kc, vc, ks, vs)]
    attention_amd.kv_append_q8(key.to(gpu), value.to(gpu), *d, table.to(gpu),
                               torch.tensor([3, 3, 0], dtype=torch.int32, device=gpu), starts([2, 2, 2]).to(gpu))
    torch.cuda.synchronize()
    nan = [torch.isnan(x).nonzero().tolist() for x in d[2:]]
    p = table[:, 0].tolist()
    assert sorted(nan[0]) == sorted([[p[0], 0], [p[1], 1]]) and nan[1] == [[p[2], 1]]
    # It stays while the page is gone on with, and goes when it is begun anew.
    one = torch.ones(3, 2, 64, device=gpu, dtype=BF)
    attention_amd.kv_append_q8(one, one, *d, table.to(gpu), torch.tensor([5, 0, 2], dtype=torch.int32, device=gpu))
    assert torch.isnan(d[2]).nonzero().tolist() == [[p[0], 0]] and torch.isnan(d[3]).nonzero().tolist() == [[p[2], 1]]
    lens = torch.tensor([6, 1, 3], dtype=torch.int32, device=gpu)
    q = torch.ones(3, 4, 64, device=gpu, dtype=BF)
    for flags in (0, cabi.QD_FLAG_FORCE_GENERIC):
        out = torch.zeros_like(q)
        assert cabi.gqa_decode_q8(q, *d, table.to(gpu), lens, out, scale=0.1, flags=flags) == 0
        bad = torch.isnan(out).all(-1)
        assert bad.tolist() == [[True, True, False, False], [False] * 4, [False, False, True, True]], flags
        assert torch.isfinite(out[~bad]).all()


def test_append_leaves_the_rest(gpu):
    """Padding, tokens past the table, pages outside the pool and other rows."""
    say("append leaves the rest")
    kc, vc, ks, vs, table, gen = cache_case("int8", [0, 0, 0, 0], [40, 40, 40, 40], 2, 64, 16, spare=0)
    table[1, 1], table[2, 2] = -7, 10 ** 6
    key = torch.randn(150, 2, 64, generator=gen).to(HF)
    cu = starts([30, 40, 60, 10])
    check_append(gpu, key, key, kc, vc, ks, vs, table, torch.tensor([-1, 3, 0, 45], dtype=torch.int32), cu, "int8", "rest")
    for bad in ([0, 10 ** 9, 5, 7, 2 ** 31 - 1], [-4, -3, -2, 2 ** 31 - 1, -1], [0, 150, 100, 50, 0]):
        d = [x.to(gpu) for x in (kc, vc, ks, vs)]
        attention_amd.kv_append_q8(key.to(gpu), key.to(gpu), *d, table.to(gpu),
                                   torch.tensor([2 ** 31 - 1, 2 ** 31 - 40, 0, 5], dtype=torch.int32, device=gpu),
                                   torch.tensor(bad, dtype=torch.int32, device=gpu))
        attention_amd.kv_gather_q8(key.to(gpu), key.to(gpu), *d, table.to(gpu),
                                   torch.tensor([2 ** 31 - 1, -5, 40, 7], dtype=torch.int32, device=gpu),
                                   torch.tensor(bad, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()


def test_append_own_scales(gpu):
    """Scales of the caller's that are no powers of two stay while they hold the values."""
    say("own scales")
    for kind in ("e4m3", "int8"):
        kc, vc, ks, vs, table, gen = cache_case(kind, [9, 20], [5, 5], 2, 64, 16, power=False)
        key = torch.randn(10, 2, 64, generator=gen).to(BF)
        d = check_append(gpu, key, key * 0.01, kc, vc, ks, vs, table, torch.tensor([9, 20], dtype=torch.int32),
                         starts([5, 5]), kind, "own scales")
        assert torch.equal(d[3].cpu(), vs)


def test_append_token_by_token(gpu):
    """A page filled one token at a time holds every value to one step of its last scale."""
    for kind in ("e4m3", "int8"):
        say(f"token by token {kind}")
        kc, vc, ks, vs, table, gen = cache_case(kind, [0, 0], [48, 48], 2, 64, 16)
        rows = torch.randn(48, 2, 2, 64, generator=gen) * torch.exp2(torch.linspace(-6, 3, 48))[:, None, None, None]
        d = [x.to(gpu) for x in (kc, vc, ks, vs)]
        for t in range(48):
            attention_amd.kv_append_q8(rows[t].to(BF).to(gpu), rows[t].to(BF).to(gpu), *d, table.to(gpu),
                                       torch.tensor([t, t], dtype=torch.int32, device=gpu))
        for b in range(2):
            got, scales = cached_rows(f64(d[0]), f64(d[2]), table[b].numpy(), 48)
            want = f64(rows[:, b].to(BF))
            step = scales[:, :, None] if kind == "int8" else np.maximum(2.0 ** -3 * np.abs(want), scales[:, :, None] * 2.0 ** -9)
            assert (np.abs(got - want) <= step).all(), kind


def check_gather(gpu, case, lens, cu, dtype, what, rows=None):
    kc, vc, ks, vs, table, _ = case
    Hkv, D = kc.shape[2:]
    rows = int(cu[-1]) + 2 if rows is None else rows
    buf = torch.full((rows, 2 * Hkv + 1, D), 7.0, device=gpu, dtype=dtype)
    key, value = buf[:, :Hkv], buf[:, Hkv:2 * Hkv]
    attention_amd.kv_gather_q8(key, value, *(x.to(gpu) for x in (kc, vc, ks, vs, table)), lens.to(gpu), cu.to(gpu))
    torch.cuda.synchronize()
    for got, cache, scales in ((key, kc, ks), (value, vc, vs)):
        want = torch.full((rows, Hkv, D), 7.0, dtype=torch.float64)
        for b in range(len(lens)):
            n = min(max(int(lens[b]), 0), int(cu[b + 1] - cu[b]), table.shape[1] * kc.shape[1])
            want[cu[b]:cu[b] + n] = torch.from_numpy(cached_rows(f64(cache), f64(scales), table[b].numpy(), n)[0])
        # element times scale is exact in float64: one rounding.
        assert torch.equal(got.cpu(), want.float().to(dtype)), what
    assert (buf[:, 2 * Hkv:] == 7.0).all()


GATHER = [
    (BF, "e4m3", [5, 0, 100, 64], [8, 3, 100, 70], 2, 128, 16), (HF, "int8", [33, 1], [33, 1], 3, 64, 16),
    (FP, "int8", [300], [310], 2, 128, 64), (FP, "e4m3", [40, 50], [30, 60], 2, 72, 7), (HF, "e4m3", [70], [70], 1, 256, 32),
    (BF, "int8", [40, 9], [40, 9], 2, 33, 16), (BF, "int8", [20], [20], 5, 80, 1), (HF, "int8", [10], [12], 1, 1, 4),
    (BF, "e4m3", [90, 77], [95, 80], 40, 128, 16), (BF, "int8", [9] * 90, [10] * 90, 1, 64, 16)]


@pytest.mark.parametrize("i", range(len(GATHER)))
@pytest.mark.parametrize("power", [True, False])
def test_gather(gpu, i, power):
    dtype, kind, lens, counts, Hkv, D, P = GATHER[i]
    say(f"gather {i} {GATHER[i]} {power}")
    case = cache_case(kind, lens, [0] * len(lens), Hkv, D, P, seed=i, power=power)
    if not power and dtype != FP:
        case = (*case[:2], case[2].bfloat16().float(), case[3].bfloat16().float(), *case[4:])  # products exact in fp32
    check_gather(gpu, case, torch.tensor(lens, dtype=torch.int32), starts(counts), dtype, f"gather {i}")


# ---- Decode over an 8-bit cache -------------------------------------------------


def decode_case(dtype, kind, lens, Hq, Hkv, D, P, *, seed=0, power=True, spare=1):
    case = cache_case(kind, lens, [0] * len(lens), Hkv, D, P, seed=seed, power=power, spare=spare)
    q = (2 * torch.randn(len(lens), Hq, D, generator=case[5])).to(dtype)
    return q, *case[:5], torch.tensor(lens, dtype=torch.int32)


def decode(gpu, case, flags=None, scale=None):
    d = [x.to(gpu) for x in case]
    if flags is not None:
        out = torch.full_like(d[0], float("nan"))
        rc = cabi.gqa_decode_q8(*d, out, scale=scale or 1 / math.sqrt(out.shape[-1]), flags=flags)
        assert rc == 0, cabi.error_string(rc)
    else:
        out = attention_amd.gqa_decode_q8(*d, scale=scale)
    torch.cuda.synchronize()
    return out


def check_decode(gpu, case, flags=None, what="", scale=None):
    q, kc, vc, ks, vs, table, lens = case
    D, kind = q.shape[-1], "int8" if kc.dtype == torch.int8 else "e4m3"
    scale = scale or 1 / math.sqrt(D)
    want, spread, size, top = oracle_decode(f64(q), f64(kc), f64(vc), f64(ks), f64(vs), table.numpy(), lens.numpy(), scale)
    n = max(1, int(lens.max()))
    kmax = TOP[kind] * ks.abs().max().item()
    err = (D + 4) * U * size + D * 2.0 ** -39 * f64(q).__abs__().max(-1) * kmax * scale
    rel = 2 * err[..., None] + 8 * U + 2 * n * U + 2.0 ** -11
    tol = HALF[q.dtype] * np.abs(want) + rel * spread + n * 2.0 ** -32 * top[..., None] * TOP[kind] + TINY[q.dtype]
    out = decode(gpu, case, flags, scale)
    assert out.dtype == q.dtype
    worst_of(f64(out), want, tol, what)
    return out


DECODE = [
    # dtype, kind, lens, Hq, Hkv, D, P
    (BF, "e4m3", [0, 1, 16, 17], 8, 2, 128, 16), (HF, "int8", [5, 300], 8, 2, 128, 16),
    (BF, "int8", [64, 129, 700], 32, 8, 128, 16), (HF, "e4m3", [1000, 3], 4, 4, 64, 32),
    (BF, "e4m3", [333], 40, 8, 128, 64), (HF, "int8", [90, 191], 15, 3, 96, 16), (BF, "int8", [130], 7, 1, 80, 48),
    (BF, "e4m3", [200, 40], 8, 1, 256, 16), (HF, "e4m3", [129], 4, 2, 192, 16), (BF, "e4m3", [77], 4, 2, 72, 16),
    (BF, "int8", [50, 333], 4, 4, 64, 7), (HF, "e4m3", [70], 6, 2, 64, 1), (HF, "int8", [240], 4, 2, 128, 12),
    (BF, "int8", [40], 3, 1, 33, 16), (HF, "e4m3", [9], 2, 1, 1, 16), (BF, "e4m3", [80, 81], 40, 1, 128, 16),
    (BF, "int8", [333], 71, 1, 64, 16), (BF, "e4m3", [5000], 8, 8, 128, 16), (HF, "int8", [3000, 20], 64, 8, 128, 64),
    (BF, "e4m3", [100] * 70, 8, 2, 128, 16), (HF, "int8", [20] * 1100, 2, 1, 64, 16), (BF, "e4m3", [64, 65], 12, 3, 128, 256),
    (BF, "e4m3", [33], 24, 3, 64, 16), (HF, "int8", [450, 449, 448], 16, 16, 64, 16), (BF, "int8", [600], 160, 10, 128, 16),
]


@pytest.mark.parametrize("i", range(len(DECODE)))
@pytest.mark.parametrize("flags", [None, cabi.QD_FLAG_FORCE_GENERIC])
def test_decode(gpu, i, flags):
    dtype, kind, lens, Hq, Hkv, D, P = DECODE[i]
    say(f"decode {i} {dtype} {kind} {lens[:4]} {Hq} {Hkv} {D} {P} flags {flags}")
    check_decode(gpu, decode_case(dtype, kind, lens, Hq, Hkv, D, P, seed=i, power=i % 2 == 0), flags, f"decode {i}")


@pytest.mark.parametrize("i", range(len(DECODE)))
def test_decode_split(gpu, i):
    """The same in tables wide enough for contexts to be split."""
    dtype, kind, lens, Hq, Hkv, D, P = DECODE[i]
    say(f"decode split {i} {dtype} {kind} {lens[:4]} {Hq} {Hkv} {D} {P}")
    case = decode_case(dtype, kind, lens, Hq, Hkv, D, P, seed=i, power=i % 2 == 1, spare=-(-3000 // P))
    if D % 16 == 0 and P % 16 == 0 and len(lens) <= 1024:
        assert cabi.gqa_decode_q8_info(len(lens), Hq, Hkv, D, P, case[5].shape[1], cabi.DTYPE[dtype])[0] == 2
    check_decode(gpu, case, None, f"decode split {i}")


def test_decode_wide_table(gpu):
    """Short contexts in a table of many pages: the ranges are cut by its width."""
    say("wide table")
    for spare in (1, 60, 4000):
        check_decode(gpu, decode_case(BF, "e4m3", [100, 0, 40, 513], 8, 2, 128, 16, seed=2, spare=spare), None, f"spare {spare}")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_decode_scales_far_apart(gpu, kind):
    """Pages whose scales differ by many powers of two, zeros among them, with and against the weights."""
    for dtype in (BF, HF):
        for sign in (1, -1):
            say(f"scales {kind} {dtype} {sign}")
            q, kc, vc, ks, vs, table, lens = decode_case(dtype, kind, [320, 100], 4, 1, 64, 16, seed=9)
            q = q * 0.1
            first = {int(p): i for row in table for i, p in enumerate(row.tolist()) if p >= 0}
            for p, i in first.items():
                vs[p] = 2.0 ** (sign * (2 * i - 20)) if dtype == BF else 2.0 ** (sign * (0.5 * i - 5) - 4)
                ks[p] = 2.0 ** (-9 + i % 5)
            vs[table[0, 3]] = 0.0
            vs[table[0, 5]] *= -1
            check_decode(gpu, (q, kc, vc, ks, vs, table, lens), None, f"scales {kind} {dtype} {sign}")
            vs[:] = 2.0 ** -100
            ks[:] = 2.0 ** -100
            check_decode(gpu, (q, kc, vc, ks, vs, table, lens), None, "smallest scales")
            if dtype == BF:
                vs[:] = 2.0 ** 100
                check_decode(gpu, (q, kc, vc, ks, vs, table, lens), None, "largest scales")


def test_decode_hidden_bytes(gpu):
    """Rows behind the last token, pages outside the table and their scales do not matter, NaN bytes included."""
    say("hidden bytes")
    q, kc, vc, ks, vs, table, lens = decode_case(BF, "e4m3", [37, 5, 0, 64], 8, 2, 128, 16, seed=3)
    want = decode(gpu, (q, kc, vc, ks, vs, table, lens))
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for t in range(n):
            used[table[b, t // 16], t % 16] = True
    for c in (kc, vc):
        c.view(torch.uint8)[~used] = 0x7F
    for s in (ks, vs):
        s[~used.any(1)] = float("nan")
    assert torch.equal(decode(gpu, (q, kc, vc, ks, vs, table, lens)), want)


def test_decode_bad_pages(gpu):
    say("bad pages")
    q, kc, vc, ks, vs, table, lens = decode_case(HF, "int8", [300, 40], 8, 2, 64, 16, seed=4)
    table[0, 2], table[0, 4], table[1, 0] = -9, 1 << 30, 2 ** 31 - 1
    for flags in (None, cabi.QD_FLAG_FORCE_GENERIC):
        check_decode(gpu, (q, kc, vc, ks, vs, table, lens), flags, "clamped pages")
    lens2 = torch.tensor([2 ** 31 - 1, -4], dtype=torch.int32)
    case = (q, kc, vc, ks, vs, table, lens2)
    full = torch.tensor([table.shape[1] * 16, 0], dtype=torch.int32)
    assert torch.equal(decode(gpu, case), decode(gpu, (q, kc, vc, ks, vs, table, full)))


def test_decode_unaligned(gpu):
    say("unaligned")
    case = decode_case(BF, "e4m3", [100, 20], 8, 2, 64, 16, seed=5)
    want = decode(gpu, case)
    d = [x.to(gpu) for x in case]
    for j in range(3):
        x = d[j]
        buf = torch.zeros(x.numel() + 1, dtype=torch.uint8 if x.element_size() == 1 else x.dtype, device=gpu)
        buf[1:] = bits(x).reshape(-1)
        moved = buf[1:].view(x.shape) if x.element_size() > 1 else buf[1:].view(x.dtype).view(x.shape)
        got = attention_amd.gqa_decode_q8(*d[:j], moved, *d[j + 1:])
        assert torch.allclose(got.float(), want.float(), rtol=4 * HALF[BF], atol=2.0 ** -10)


def test_large_pool(gpu):
    """Pages past 2^32 bytes of the cache, written, read back and attended to."""
    say("large pool")
    P, Hkv, D = 64, 8, 128
    N = (1 << 32) // (P * Hkv * D) + 40
    kc = torch.zeros(N, P, Hkv, D, device=gpu, dtype=torch.int8)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.ones(N, Hkv, device=gpu) for _ in range(2))
    table = torch.tensor([[N - 1, N - 7, N - 30, 3], [N - 20, 2, N - 40, 1]], dtype=torch.int32, device=gpu)
    gen = torch.Generator().manual_seed(0)
    lens = [250, 130]
    rows = torch.randn(sum(lens), 2 * Hkv, D, generator=gen).to(BF)
    key, value = rows.to(gpu).split([Hkv, Hkv], dim=1)
    cu, zero = starts(lens).to(gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    attention_amd.kv_append_q8(key, value, kc, vc, ks, vs, table, zero, cu)
    back = torch.zeros_like(rows, device=gpu)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    attention_amd.kv_gather_q8(*back.split([Hkv, Hkv], dim=1), kc, vc, ks, vs, table, n, cu)
    err = (back.float().cpu() - rows.float()).abs().amax()
    assert 0 < err < 5 / 127  # values below 5: a step is at most 5 * 2 / 127, off by half of it
    q = torch.randn(2, 32, D, generator=gen).to(BF).to(gpu)
    got = attention_amd.gqa_decode_q8(q, kc, vc, ks, vs, table, n)
    want, spread, size = oracle_prefill(f64(q), *(f64(x) for x in back.split([Hkv, Hkv], dim=1)), [0, 1, 2], cu.tolist(), 0,
                                        0, 1 / math.sqrt(D))
    tol = HALF[BF] * np.abs(want) + (2 * (D + 4) * U * size[..., None] + 600 * U + 2.0 ** -11) * spread + 2.0 ** -20
    worst_of(f64(got), want, tol, "large pool")
    assert int(kc[:N - 40].any()) and not kc[4:N - 40].any()


# ---- Together --------------------------------------------------------------------


def test_serving_run(gpu):
    """Prompts, a second chunk of them that reads the cache back, and decoding steps, against attention over the
    cached values in float64."""
    for dtype, kind in ((BF, "e4m3"), (HF, "int8")):
        say(f"serving run {dtype} {kind}")
        Hq, Hkv, D, P = 8, 2, 64, 16
        gen = torch.Generator().manual_seed(7)
        first, second, steps = [37, 5, 90], [20, 33, 1], 4
        total = [a + b + steps for a, b in zip(first, second)]
        table, N = table_of(gen, [-(-n // P) for n in total], 0)
        table = table.to(gpu)
        cache = [torch.zeros(N, P, Hkv, D, device=gpu, dtype=CACHE[kind]) for _ in range(2)]
        cache += [torch.zeros(N, Hkv, device=gpu) for _ in range(2)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731

        def project(n):
            return torch.randn(n, Hq + 2 * Hkv, D, generator=gen).to(dtype).to(gpu).split([Hq, Hkv, Hkv], dim=1)

        q, k, v = project(sum(first))
        cu = starts(first).to(gpu)
        out = attention_amd.gqa_prefill(q, k, v, cu)
        want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), None, 0, 0, 1 / math.sqrt(D))
        case = (q.cpu(), k.cpu(), v.cpu(), cu.cpu(), None)
        worst_of(f64(out), want, prefill_tolerance(case, want, spread, size), "first chunk")
        attention_amd.kv_append_q8(k, v, *cache, table, i32([0, 0, 0]), cu)
        # The second chunk sees the first as the cache holds it, and itself.
        q, k, v = project(sum(second))
        cu, both = starts(second).to(gpu), starts([a + b for a, b in zip(first, second)]).to(gpu)
        key, value = (torch.zeros(int(both[-1]), Hkv, D, device=gpu, dtype=dtype) for _ in range(2))
        own = torch.cat([torch.arange(both[b] + first[b], both[b + 1]) for b in range(3)]).to(gpu)
        key[own], value[own] = k, v
        attention_amd.kv_gather_q8(key, value, *cache, table, i32(first), both)
        out = attention_amd.gqa_prefill(q, key, value, cu, cu_seqlens_k=both)
        want, spread, size = oracle_prefill(f64(q), f64(key), f64(value), cu.tolist(), both.tolist(), 0, 0, 1 / math.sqrt(D))
        case = (q.cpu(), key.cpu(), value.cpu(), cu.cpu(), both.cpu())
        worst_of(f64(out), want, prefill_tolerance(case, want, spread, size), "second chunk")
        assert torch.equal(key[own], k)
        attention_amd.kv_append_q8(k, v, *cache, table, i32(first), cu)
        for step in range(steps):
            q, k, v = project(3)
            at = [a + b + step for a, b in zip(first, second)]
            attention_amd.kv_append_q8(k, v, *cache, table, i32(at))
            check_decode(gpu, (q.cpu(), *(x.cpu() for x in cache), table.cpu(), torch.tensor(at, dtype=torch.int32) + 1),
                         None, f"step {step}")


def test_streams_and_graphs(gpu):
    """Calls on a side stream, two at once, and captured ones: every replay as the eager call."""
    say("streams and graphs")
    pre = [x if x is None else x.to(gpu) for x in prefill_case(BF, [150, 70], None, 8, 2, 128, seed=1)]
    dec = [x.to(gpu) for x in decode_case(BF, "e4m3", [900, 40, 3], 8, 2, 128, 16, seed=1)]
    app = [x.to(gpu) for x in cache_case("int8", [9, 4], [1, 1], 2, 128, 16, seed=2)[:5]]
    rows = torch.randn(2, 2, 128, device=gpu, dtype=BF)
    at = torch.tensor([9, 4], dtype=torch.int32, device=gpu)
    back = torch.zeros(40, 2, 128, device=gpu, dtype=BF)
    cu = torch.tensor([0, 20, 40], dtype=torch.int32, device=gpu)

    def step():
        attention_amd.kv_append_q8(rows, rows, *app, at)
        attention_amd.kv_gather_q8(back, back.clone(), *app, at + 1, cu)
        return (attention_amd.gqa_prefill(*pre[:4]), attention_amd.gqa_decode_q8(*dec), back.clone(), *(x.clone() for x in app[:4]))

    want = step()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append((attention_amd.gqa_prefill(*pre[:4]), attention_amd.gqa_decode_q8(*dec)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want[:2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        dec[0].mul_(1.0 if i % 2 else -1.0)
        rows.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in out]
        eager = step()
        for x, y in zip(replayed, eager):
            assert torch.equal(bits(x), bits(y)), i


@pytest.mark.parametrize("dtype", [BF, FP])
def test_split_prompts_on_streams_and_in_graphs(gpu, dtype):
    """Two calls at once whose keys are split, and captured ones that share nothing but the graphs' memory."""
    say(f"split prompts, streams and graphs {dtype}")
    a, b = ([x.to(gpu) for x in prefill_case(dtype, nq, nk, 8, 2, 64, seed=s)] for nq, nk, s in (([9, 2], [2000, 1500], 1), ([3], [2500], 2)))
    run = lambda c: attention_amd.gqa_prefill(*c[:4], cu_seqlens_k=c[4])  # noqa: E731
    want = [run(a), run(b)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, c in zip(side, (a, b)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, out = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, c in zip(graphs, (a, b)):
        with torch.cuda.graph(g):
            out.append(run(c))
    for i in range(3):
        a[0].mul_(-1)
        b[2].mul_(0.5)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in out]
        assert all(torch.equal(x, y) for x, y in zip(replayed, (run(a), run(b)))), i


def test_decode_short_tables_in_a_graph(gpu):
    """The launch without a merge, captured; lengths change between replays."""
    say("short tables in a graph")
    case = [x.to(gpu) for x in decode_case(HF, "int8", [90, 0, 33], 8, 2, 128, 16, seed=4)]
    assert cabi.gqa_decode_q8_info(3, 8, 2, 128, 16, case[5].shape[1], cabi.DTYPE[HF])[0] == 1
    graph = torch.cuda.CUDAGraph()
    attention_amd.gqa_decode_q8(*case)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = attention_amd.gqa_decode_q8(*case)
    for lens in ([90, 0, 33], [1, 96, 0], [0, 0, 0], [50, 51, 52]):
        case[6].copy_(torch.tensor(lens, dtype=torch.int32))
        case[5].clamp_(min=0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, attention_amd.gqa_decode_q8(*case)), lens
        assert not replayed[[i for i, n in enumerate(lens) if n == 0]].any()
