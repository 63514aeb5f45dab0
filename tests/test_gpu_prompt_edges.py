"""GPU tests of prompt attention and of 8-bit caches where scores, scales, values and
sizes are far from ordinary.  Every case prints its name first."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_amd
from attention_amd import cabi
from oracle.prompt_oracle import TOP, cached_rows, oracle_prefill
from tests.test_gpu_prompt import (BF, CACHE, DECODE, FP, HALF, HF, SPLIT, TINY, U, WEIGHT, cache_case, check_append,
                                   check_gather, decode, decode_case, f64, prefill, prefill_case, prefill_tolerance, say,
                                   starts)

pytestmark = pytest.mark.gpu


def split_bytes(case, window=0, sinks=0):
    q, k, _, cu, _ = case
    return cabi.lib().qd_gqa_prefill_workspace_bytes(cu.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2],
                                                     cabi.DTYPE[q.dtype], window, sinks, 0)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("flags", [None, cabi.QD_FLAG_FORCE_GENERIC])
def test_prefill_split_nan_scores(gpu, dtype, flags):
    """A NaN query, and NaN keys that are all that a row sees of a part, give NaN rows, and no others."""
    say(f"split NaN scores {dtype} flags {flags}")
    case = prefill_case(dtype, [6], [3000], 4, 2, 128, seed=31)
    assert split_bytes(case) > 0
    q, k, v, cu, cu_k = case
    want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), cu_k.tolist(), 0, 0, 128 ** -0.5)
    tol = prefill_tolerance(case, want, spread, size)
    q[2, 1, 77] = float("nan")
    for keys in (None, slice(0, 1000), slice(1500, 2990), slice(2995, 2996)):
        kk = k.clone()
        hit = np.zeros((q.shape[0], 4), dtype=bool)
        hit[2, 1] = True
        if keys is not None:
            kk[keys, 1, 5] = float("nan")
            hit[max(0, keys.start - 2994):6, 2:] = True  # query i sees the keys up to 2994 + i
        out = f64(prefill(gpu, (q, kk, v, cu, cu_k), flags=flags))
        assert np.isnan(out[hit]).all(), keys
        assert (np.abs(out - want)[~hit] <= tol[~hit]).all(), keys


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_prefill_split_one_nan_key(gpu, dtype):
    """One NaN key.  For one row it is the only key that it sees of its part: parts begin at token 1344, and the
    first ends with token 1471 (fp32: 1407), which is the first that query 98 (34) sees."""
    case = prefill_case(dtype, [128], [3000], 2, 2, 64, seed=32)
    assert split_bytes(case, 1500) > 0
    q, k, v, cu, cu_k = case
    want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), cu_k.tolist(), 1500, 0, 0.125)
    tol = prefill_tolerance(case, want, spread, size)
    for token in (1407, 1471):
        say(f"split, one NaN key {dtype} {token}")
        kk = k.clone()
        kk[token, 1, 3] = float("nan")
        out = f64(prefill(gpu, (q, kk, v, cu, cu_k), window=1500))
        hit = np.zeros((q.shape[0], 2), dtype=bool)
        hit[:token - 1373 + 1, 1] = True  # query i sees the keys from 1373 + i on
        assert np.isnan(out[hit]).all(), token
        assert (np.abs(out - want)[~hit] <= tol[~hit]).all(), token


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("flags", [0, cabi.QD_FLAG_FORCE_GENERIC])
@pytest.mark.parametrize("D", [64, 33])
def test_prefill_no_sequences(gpu, dtype, flags, D):
    """Only rows behind the last sequence, whatever lies behind the one entry of cu_seqlens."""
    say(f"no sequences {dtype} flags {flags} {D}")
    q, k = torch.ones(5, 4, D, device=gpu, dtype=dtype), torch.ones(5, 2, D, device=gpu, dtype=dtype)
    cu, cu_k = (torch.tensor([0, 5, 5], dtype=torch.int32, device=gpu)[:1] for _ in range(2))
    for ends in (None, cu_k):
        out = torch.full_like(q, float("nan"))
        assert cabi.gqa_prefill(q, k, k, cu, ends, out, scale=0.1, flags=flags) == 0
        assert not out.any()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_goes_on_with_scales_below_zero(gpu, kind):
    """A page's scale may be negative: it stays while its magnitude holds the new rows, and is replaced else."""
    say(f"scales below zero {kind}")
    kc, vc, ks, vs, table, gen = cache_case(kind, [9, 20, 3, 40], [5, 5, 1, 30], 2, 64, 16, power=False)
    key = torch.randn(41, 2, 64, generator=gen).to(BF)
    ks, vs = -32 * ks, -vs
    at, cu = torch.tensor([9, 20, 3, 40], dtype=torch.int32), starts([5, 5, 1, 30])
    d = check_append(gpu, key * 100, key * 0.001, kc, vc, ks, vs, table, at, cu, kind, "small and large scales below zero")
    assert (d[3] < 0).any() and (d[2] < 0).any() and (d[2] > 0).any()


LEVELS = {
    "same": lambda j, n: 0 * j + 5, "negative": lambda j, n: 0 * j - 7, "rising": lambda j, n: -60 + j * 120 // n,
    "falling": lambda j, n: 60 - j * 120 // n, "mixed": lambda j, n: (j * 37) % 101 - 50,
}


def far_case(dtype, nq, nk, Hq, Hkv, D, level):
    """Scores that are exact in float32: 8 times a small whole number that each key has."""
    q, k, v, cu, cu_k = prefill_case(dtype, nq, nk, Hq, Hkv, D, seed=41)
    q[:], k[:] = 0, 0
    q[:, :, 0] = 8
    levels = LEVELS[level](torch.arange(k.shape[0]), k.shape[0])
    k[:, :, 0] = levels[:, None].to(dtype)
    return (q, k, v, cu, cu_k), levels.numpy()


def far_want(case, levels):
    """Only the largest scores that a query sees have a weight, all the same: the mean of their values."""
    q, k, v, cu, cu_k = case
    cu_k = cu if cu_k is None else cu_k
    want, spread = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(cu) - 1):
        q0, q1, k0, k1 = int(cu[b]), int(cu[b + 1]), int(cu_k[b]), int(cu_k[b + 1])
        for i in range(q1 - q0):
            seen = levels[k0:k1 - (q1 - q0) + i + 1]
            top = f64(v)[k0 + np.flatnonzero(seen == seen.max())]
            want[q0 + i] = np.repeat(top.mean(0), q.shape[1] // k.shape[1], 0)
            spread[q0 + i] = np.repeat(np.abs(top).mean(0), q.shape[1] // k.shape[1], 0)
    return want, spread


FAR = [([300], None, 2, 1, 64), ([200, 3], None, 4, 2, 128), ([6], [3000], 4, 2, 128), ([70], None, 2, 1, 96), ([100], None, 2, 2, 256)]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("i", range(len(FAR)))
@pytest.mark.parametrize("level", LEVELS)
def test_prefill_far_scores(gpu, dtype, i, level):
    """Scores of 2^16 to 2^109.  They are exact and at least 2^16 apart: weights are 0 or all the same.  Their sum of
    n terms is off by 2 n u, their exponentials by 8 u, and both halves of the quotient are rounded as always; the
    grid of fp16 weights is 2^-32 of the largest."""
    case, levels = far_case(dtype, *FAR[i], level)
    want, spread = far_want(case, levels)
    n = case[1].shape[0]
    tol = HALF[dtype] * np.abs(want) + (WEIGHT[dtype] + 2 * n * U + 8 * U) * spread + TINY[dtype]
    if dtype == HF:
        tol = tol + n * 2.0 ** -32 * case[2].abs().max().item()
    for e in (13, 17, 18, 22, 25, 28, 33, 60, 100):
        say(f"far scores {dtype} {FAR[i]} {level} 2^{e}")
        for flags in (None, cabi.QD_FLAG_FORCE_GENERIC):
            out = f64(prefill(gpu, case, flags=flags, scale=2.0 ** e))
            assert (np.abs(out - want) <= tol).all(), (e, flags)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_prefill_far_scores_of_64_rows(gpu, dtype):
    """The same, where a wave has 64 rows: rising scores, whose last key alone has a weight."""
    case = prefill_case(dtype, [1000] * 4, None, 66, 2, 64, seed=42, spare=0)
    q, k, v, cu, _ = case
    assert cabi.gqa_prefill_info(4, 4000, 4000, 66, 2, 64, cabi.DTYPE[dtype])[2] == 256
    q[:], k[:] = 0, 0
    q[:, :, 0] = 8
    k[:, :, 0] = torch.arange(1, 1001).repeat(4)[:, None] // 8
    k[:, :, 1] = torch.arange(1, 1001).repeat(4)[:, None] % 8
    q[:, :, 1] = 1  # scores 1, 2, .. of a sequence's keys
    for e in (10, 17, 25, 33, 60, 90):
        say(f"far scores, 64 rows {dtype} 2^{e}")
        out = prefill(gpu, case, scale=2.0 ** e).cpu()
        assert torch.equal(out, v.repeat_interleave(33, 1)), e


FAR_DECODE = [
    # lens, Hq, Hkv, D, P, spare pages
    ([300, 1, 77], 8, 2, 64, 16, 0), ([300, 129], 8, 4, 128, 16, 200), ([2000], 4, 1, 128, 64, 0), ([100, 500], 6, 3, 256, 16, 0),
    ([700], 40, 8, 128, 32, 100),
]


@pytest.mark.parametrize("dtype, values", [(HF, 1.0), (BF, 1.0), (BF, 2.0 ** 40), (BF, 2.0 ** -40)])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("i", range(len(FAR_DECODE)))
@pytest.mark.parametrize("flags", [0, cabi.QD_FLAG_FORCE_GENERIC])
def test_decode_far_scores(gpu, dtype, values, kind, i, flags):
    """Scores of 2^16 to 2^100, exact and at least 2^16 apart: only the largest have a weight, all the same.
    Tolerance: weights once to fp16 with the scale of their page, on a grid of 2^-32 of the largest such
    product; n terms by 2 n u, exponentials by 8 u, the output's rounding."""
    lens, Hq, Hkv, D, P, spare = FAR_DECODE[i]
    q, kc, vc, ks, vs, table, n = decode_case(dtype, kind, lens, Hq, Hkv, D, P, seed=51 + i, spare=spare)
    q[:] = 0
    q[:, :, 0] = 8
    ks[:], vs = 0.5, vs * values
    for level in LEVELS:
        levels = LEVELS[level](torch.arange(max(lens)), max(lens)) // 5  # -12 to 12: both types hold them
        k = torch.zeros(kc.shape)
        want, tol = np.zeros(q.shape), np.zeros(q.shape)
        for b, len_ in enumerate(lens):
            for t in range(len_):
                k[table[b, t // P], t % P, :, 0] = levels[t].float()
            v, scales = cached_rows(f64(vc), f64(vs), table[b].numpy(), len_)
            top = np.flatnonzero(levels[:len_] == levels[:len_].max())
            mean, spread = v[top].mean(0), np.abs(v[top]).mean(0)
            err = (HALF[dtype] * np.abs(mean) + (2.0 ** -11 + 2 * len_ * U + 8 * U) * spread
                   + len_ * 2.0 ** -32 * TOP[kind] * scales[top].max(0)[:, None] / len(top) + TINY[dtype])
            want[b], tol[b] = np.repeat(mean, Hq // Hkv, 0), np.repeat(err, Hq // Hkv, 0)
        for e in (14, 20, 24, 26, 28, 33, 60, 94):
            say(f"far decode {dtype} {values} {kind} {FAR_DECODE[i]} {level} 2^{e} flags {flags}")
            out = f64(decode(gpu, (q, k.to(CACHE[kind]), vc, ks, vs, table, n), flags, 2.0 ** e))
            assert (np.abs(out - want) <= tol).all(), (level, e)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("last", [True, False])
def test_decode_long_stretch_of_zero_values(gpu, kind, last):
    """65552 tokens, of which only 16 have values, with the others' scales as kv_append_q8 writes them (2^-100).
    All scores are the same but for the first 32, which are lower."""
    say(f"zero values {kind} {last}")
    B, P, pages = 512, 16, 4097
    kc, vc = torch.zeros(4, P, 4, 64), torch.zeros(4, P, 4, 64)
    kc[1:, :, :, 0] = 8
    vc[2] = torch.randint(-15, 16, (P, 4, 64), generator=torch.Generator().manual_seed(3)).float()
    ks, vs = torch.full((4, 4), 0.125), torch.full((4, 4), 2.0 ** -100)
    vs[2] = 0.25
    row = [0, 0] + [1] * (pages - 2)
    row[-1 if last else 2000] = 2
    table = torch.tensor([row] * B, dtype=torch.int32)
    q = torch.zeros(B, 4, 64, dtype=BF)
    q[:, :, 0] = 5.25  # scores 5.25, or 0: 7.57 binary places apart
    out = decode(gpu, (q, kc.to(CACHE[kind]), vc.to(CACHE[kind]), ks, vs, table, torch.full((B,), P * pages, dtype=torch.int32)),
                 scale=1.0)
    v = f64(vc[2]) * 0.25
    total = 32 * np.exp(-5.25) + P * (pages - 2)
    want = (v.sum(0) / total)[None]
    # Weights are rounded once, to fp16 with the scale of their page, on a grid of 2^-32 of the largest such product;
    # n terms are off by 2 n u, exponentials by 8 u, the output by half a step.  The largest weight times scale is
    # 0.25 / total, the values at most 15 steps of it.
    tol = (HALF[BF] * np.abs(want) + (2.0 ** -11 + 2 * P * pages * U + 8 * U) * (np.abs(v).sum(0) / total)[None]
           + P * pages * 2.0 ** -32 * 0.25 * 15 / total)
    assert (np.abs(f64(out) - want) <= tol).all()


# ---- What a workspace holds before a call, lookups of many sequences ---------------


@pytest.mark.parametrize("i", range(len(SPLIT)))
def test_prefill_split_reads_what_it_wrote(gpu, i):
    """Whatever the workspace holds before the call."""
    dtype, nq, nk, Hq, Hkv, D, window, sinks = SPLIT[i]
    say(f"split workspace {i} {SPLIT[i]}")
    case = prefill_case(dtype, nq, nk, Hq, Hkv, D, seed=50 + i)
    d = [x if x is None else x.to(gpu) for x in case]
    bytes_ = split_bytes(case, window, sinks)
    assert bytes_ > 0
    outs = []
    for fill in (0x00, 0xFF, 0x7F):  # zeros, NaN, the largest numbers
        ws = torch.full((bytes_ + 256,), fill, dtype=torch.uint8, device=gpu)
        out = torch.full_like(d[0], float("nan"))
        assert cabi.gqa_prefill(*d, out, scale=1 / math.sqrt(D), window=window, sinks=sinks, workspace=ws[:bytes_]) == 0
        outs.append(out)
        assert (ws[bytes_:] == fill).all()
    assert torch.isfinite(outs[0]).all() and all(torch.equal(x, outs[0]) for x in outs)


@pytest.mark.parametrize("i", range(len(DECODE)))
def test_decode_split_reads_what_it_wrote(gpu, i):
    dtype, kind, lens, Hq, Hkv, D, P = DECODE[i]
    say(f"decode workspace {i} {dtype} {kind} {lens[:4]} {Hq} {Hkv} {D} {P}")
    case = [x.to(gpu) for x in decode_case(dtype, kind, lens, Hq, Hkv, D, P, seed=i, spare=-(-3000 // P))]
    bytes_ = cabi.lib().qd_gqa_decode_q8_workspace_bytes(len(lens), Hq, Hkv, D, P, case[5].shape[1], cabi.DTYPE[dtype], 0)
    outs = []
    for fill in (0x00, 0xFF, 0x7F):
        ws = torch.full((bytes_ + 256,), fill, dtype=torch.uint8, device=gpu)
        out = torch.full_like(case[0], float("nan"))
        assert cabi.gqa_decode_q8(*case, out, scale=1 / math.sqrt(D), workspace=ws[:bytes_]) == 0
        outs.append(out)
        assert (ws[bytes_:] == fill).all()
    assert torch.isfinite(outs[0]).all() and all(torch.equal(x, outs[0]) for x in outs)


@pytest.mark.parametrize("B", [62, 63, 64, 65, 200, 4100])
@pytest.mark.parametrize("P", [1, 7, 16])
def test_append_many_sequences(gpu, B, P):
    """Runs are found by one round trip up to 63 sequences and by searches from 64 on; empty sequences, and runs
    begun anywhere in a page."""
    say(f"append {B} sequences, pages of {P}")
    gen = torch.Generator().manual_seed(B)
    counts = torch.randint(0, 40, (B,), generator=gen).tolist()
    for b in (0, B // 2, B - 1):
        counts[b] = 0
    at = torch.randint(0, 30, (B,), generator=gen).tolist()
    kc, vc, ks, vs, table, gen = cache_case("int8" if P == 7 else "e4m3", at, counts, 1, 16, P, seed=B)
    rows = torch.randn(sum(counts) + 2, 2, 16, generator=gen).to(BF)
    check_append(gpu, rows[:, :1], rows[:, 1:], kc, vc, ks, vs, table, torch.tensor(at, dtype=torch.int32), starts(counts),
                 "int8" if P == 7 else "e4m3", f"{B} sequences")


@pytest.mark.parametrize("B", [62, 63, 64, 65, 1000])
def test_gather_many_sequences(gpu, B):
    say(f"gather {B} sequences")
    gen = torch.Generator().manual_seed(B)
    counts = torch.randint(0, 70, (B,), generator=gen)
    lens = torch.minimum(counts, torch.randint(0, 70, (B,), generator=gen))
    counts[0], lens[0], lens[B - 1] = 0, 0, 0
    case = cache_case("e4m3", lens.tolist(), [0] * B, 1, 16, 16, seed=B)
    check_gather(gpu, case, lens.int(), starts(counts.tolist()), BF, f"{B} sequences")


# ---- Values that are not finite, where a wave has 64 rows and where heads are padded ----


def bad_values(case, places, bad):
    q, k, v, cu, cu_k = case
    v = v.clone()
    for token, col in places:
        v[token, :, col] = bad
    return q, k, v, cu, cu_k


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype, D", [(HF, 80), (BF, 96), (BF, 72), (HF, 192), (BF, 160), (FP, 80), (FP, 200)])
def test_prefill_hidden_values_of_padded_heads(gpu, bad, dtype, D):
    """A value that is not finite reaches the rows that see it, and no other; the last column of a head too."""
    say(f"hidden, padded heads {bad} {dtype} {D}")
    for window, sinks in ((0, 0), (20, 3)):
        case = prefill_case(dtype, [130, 70], None, 2, 1, D, seed=61)
        q, k, v, cu, _ = case
        want, spread, size = oracle_prefill(f64(q), f64(k), f64(v), cu.tolist(), None, window, sinks, 1 / math.sqrt(D))
        tol = prefill_tolerance(case, want, spread, size)
        places = ((60, 0), (129, D - 1), (2, D // 2), (131, D - 1))
        out = f64(prefill(gpu, bad_values(case, places, bad), window, sinks))
        hit = np.zeros_like(want, dtype=bool)
        for t in range(200):
            b = 0 if t < 130 else 130
            for token, col in places:
                hit[t, :, col] |= b <= token <= t and (not window or token > t - window or token - b < sinks)
        assert not np.isfinite(out[hit]).any() and (np.abs(out - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
@pytest.mark.parametrize("dtype, window, sinks", [(BF, 0, 0), (HF, 100, 5)])
def test_prefill_hidden_values_of_64_rows(gpu, bad, dtype, window, sinks):
    """The same where a wave has 64 rows, against the call without such values: rows that see none are as there."""
    say(f"hidden, 64 rows {bad} {dtype} {window}")
    counts = [3000, 1, 0, 1095]
    case = prefill_case(dtype, counts, None, 64, 8, 64, seed=62, spare=1)
    assert cabi.gqa_prefill_info(4, 4097, 4097, 64, 8, 64, cabi.DTYPE[dtype])[2] == 256
    places = ((3, 0), (700, 63), (2999, 5), (3000, 6), (3500, 7))
    want = prefill(gpu, case, window, sinks)
    got = prefill(gpu, bad_values(case, places, bad), window, sinks)
    t = torch.arange(4097)
    begin = torch.where(t < 3000, 0, torch.where(t < 3001, 3000, torch.where(t < 4096, 3001, 4096)))
    hit = torch.zeros(4097, 64, 64, dtype=torch.bool)
    for token, col in places:
        sees = (begin <= token) & (token <= t)
        if window:
            sees &= (token > t - window) | (token - begin < sinks)
        hit[sees, :, col] = True
    hit = hit.to(gpu)
    assert not got[hit].isfinite().any()
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D", [8, 64, 128, 256])
@pytest.mark.parametrize("flags", [0, cabi.QD_FLAG_FORCE_GENERIC])
def test_prefill_rows_of_scores_without_weight(gpu, dtype, D, flags):
    """A query all of whose scores are -inf gets zeros, whatever the values hold; others are as ever."""
    say(f"scores of -inf {dtype} {D} flags {flags}")
    case = prefill_case(dtype, [70, 3], None, 2, 1, D, seed=71)
    q, k, v, cu, _ = case
    q[:, :, 3] = 1
    want, spread, size = oracle_prefill(f64(q[70:73]), f64(k[70:73]), f64(v[70:73]), [0, 3], None, 0, 0, 1 / math.sqrt(D))
    for bad in (float("nan"), float("inf"), -float("inf")):
        kk, vv = k.clone(), v.clone()
        kk[:70, 0, 3] = -float("inf")
        vv[:66, 0, 5] = bad
        vv[69, 0, 1] = bad
        out = prefill(gpu, (q, kk, vv, cu, None), flags=flags)
        assert not out[:70].any()
        tol = prefill_tolerance((q, k, v, cu, None), want, spread, size)
        assert (np.abs(f64(out[70:73]) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_prefill_past_2_32_bytes(gpu, dtype):
    """Queries, keys, values and output of one projection of 5.6 GB: sequences at both ends against the oracle."""
    say(f"past 2^32 bytes {dtype}")
    Hq, Hkv, D, T = 32, 4, 128, 550_000
    counts = [37] + [499] * 1102 + [0, 55, 3]
    cu = starts(counts)
    assert 0 < T - int(cu[-1]) < 500
    qkv = torch.empty(T, Hq + 2 * Hkv, D, dtype=dtype, device=gpu)
    qkv[:] = torch.randn(997, Hq + 2 * Hkv, D, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)).to(dtype).repeat(552, 1, 1)[:T]
    q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
    out = attention_amd.gqa_prefill(q, k, v, cu.to(gpu))
    assert out.numel() * 2 > 2 ** 32 and qkv.numel() * 2 > 2 ** 32
    assert not out[int(cu[-1]):].any()
    for b in (0, len(counts) - 2, len(counts) - 1):
        part = tuple(x[cu[b]:cu[b + 1]].cpu() for x in (q, k, v)) + (torch.tensor([0, counts[b]], dtype=torch.int32), None)
        want, spread, size = oracle_prefill(*(f64(x) for x in part[:3]), [0, counts[b]], None, 0, 0, D ** -0.5)
        tol = prefill_tolerance(part, want, spread, size)
        assert (np.abs(f64(out[cu[b]:cu[b + 1]]) - want) <= tol).all(), b
