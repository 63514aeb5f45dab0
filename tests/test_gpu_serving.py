"""GPU parity of the operators around drafted tokens and sliding windows
(norm, rotation and cache write; window and tree attention; compaction)
against the float64 oracle, and what a caller can run into: hidden tokens
that hold NaN, freed pages, ragged batches, other streams, captured graphs,
unaligned tensors, pools past 2^32 bytes.  Every case prints its name first.

Tolerances, u = 2^-24 and h = half a step of the output type relative to the
value (fp32 2^-24, fp16 2^-11, bf16 2^-8):
  attention  a score of D terms is off by at most (D + 4) u S, S its sum of
             |q k| scale; a softmax weight by twice that and 8 u of the two
             exponentials, relatively; n summed terms by n u; weights kept as
             two 16-bit parts by 2^-15 (bf16, 16 bits, cut) and 2^-20 (fp16).
             Times sum(weight |v|), plus the output's rounding h |out|.
  write      y = x r w: the sum of squares is off by D u, its root and
             reciprocal by a few u: (D + 16) u (|a| + |b|) of the rotated
             pair, plus h |y|.
Below the smallest normal number the rounding step is fixed: 2^-25 for fp16.
"""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import attention_amd
from attention_amd import cabi
from oracle.serving_oracle import oracle_compact, oracle_tree, oracle_write

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
WEIGHT = {torch.float32: 0.0, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -15}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def say(msg):
    print(f"[case] {msg}", flush=True)


def f64(x):
    return x.detach().cpu().double().numpy()


# ---- Attention -------------------------------------------------------------------


def tree_masks(gen, B, T, branch, ragged):
    """Ancestor masks of random trees; the rows past a sequence's last drafted token are 0."""
    masks = []
    for b in range(B):
        count = int(torch.randint(1, T + 1, (1,), generator=gen)) if ragged else T
        row = []
        for j in range(count):
            parent = j - int(torch.randint(1, branch + 1, (1,), generator=gen))
            row.append((row[parent] if parent >= 0 else 0) | 1 << j)
        masks.append(row + [0] * (T - count))
    return masks


def signed(masks):
    return torch.tensor([[m - (1 << 64) if m >> 63 else m for m in row] for row in masks], dtype=torch.int64)


def attention_case(dtype, B, T, Hq, Hkv, D, P, lens, *, branch=2, ragged=True, window=0, seed=0, spare=2, k_scale=2.0):
    """T = 0: one query per sequence, no masks.  Every sequence has pages of
    its own, ``spare`` more than it needs."""
    gen = torch.Generator().manual_seed(seed)
    width = max(-(-(max(n, 0) + T) // P) for n in lens) + spare
    N = B * width + 3
    table = torch.randperm(N, generator=gen)[:B * width].view(B, width).int().contiguous()
    q = torch.randn(*((B, T) if T else (B,)), Hq, D, generator=gen).to(dtype)
    k = (k_scale * torch.randn(N, P, Hkv, D, generator=gen)).to(dtype)
    v = torch.randn(N, P, Hkv, D, generator=gen).to(dtype)
    masks = tree_masks(gen, B, T, branch, ragged) if T else None
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32), masks


def attention_want(q, k, v, table, lens, masks, window, sinks, scale):
    q4 = f64(q) if masks is not None else f64(q)[:, None]
    out, spread, size = oracle_tree(q4, f64(k), f64(v), table.cpu().numpy(), lens.cpu().numpy(), masks, window, sinks,
                                    scale)
    if masks is None:
        out, spread, size = out[:, 0], spread[:, 0], size[:, 0]
    return out, spread, size


def attention_check(got, want, spread, size, dtype, D, n, what):
    """n: the most tokens that a row sums."""
    assert got.dtype == dtype
    got = f64(got)
    assert np.isfinite(got).all(), f"{what}: not finite"
    rel = 2 * (D + 4) * U * size[..., None] + 8 * U + 2 * n * U + WEIGHT[dtype]
    tol = HALF[dtype] * np.abs(want) + rel * spread + TINY[dtype]
    worst = (np.abs(got - want) / tol).max() if got.size else 0.0
    print(f"[case] {what}: {worst:.3f} of the tolerance", flush=True)
    assert worst <= 1.0, what


def attend(gpu, case, window=0, sinks=0, flags=None, scale=None):
    q, k, v, table, lens, masks = case
    d = [x.to(gpu) for x in (q, k, v, table, lens)]
    m = signed(masks).to(gpu) if masks is not None else None
    if flags is not None:
        out = torch.full_like(d[0], float("nan"))
        rc = cabi.gqa_decode_tree(*d, m, out, scale=scale or 1 / math.sqrt(q.shape[-1]), window=window, sinks=sinks,
                                  flags=flags)
        assert rc == 0, cabi.error_string(rc)
    elif masks is None:
        out = attention_amd.gqa_decode_window(*d, window=window, sinks=sinks, scale=scale)
    else:
        out = attention_amd.gqa_decode_tree(*d, m, window=window or None, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    return out


def check_case(gpu, case, window=0, sinks=0, flags=None, what="", scale=None):
    q, k, v, table, lens, masks = case
    want, spread, size = attention_want(q, k, v, table, lens, masks, window, sinks, scale or 1 / math.sqrt(q.shape[-1]))
    out = attend(gpu, case, window, sinks, flags, scale)
    attention_check(out, want, spread, size, q.dtype, q.shape[-1], int(max(lens)) + 64, what)
    return out


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

TREE_SHAPES = [
    # dtype, B, T, Hq, Hkv, D, P, lens, branch, window, sinks
    (BF, 1, 1, 1, 1, 8, 16, [0], 1, 0, 0),
    (BF, 2, 1, 8, 2, 64, 16, [1, 130], 1, 0, 0),
    (BF, 3, 7, 8, 2, 128, 16, [0, 63, 300], 2, 0, 0),
    (HF, 2, 16, 8, 2, 128, 16, [64, 129], 3, 0, 0),
    (BF, 2, 16, 32, 4, 128, 32, [700, 5], 3, 0, 0),
    (BF, 2, 64, 8, 2, 128, 16, [100, 257], 8, 0, 0),
    (HF, 1, 64, 16, 1, 64, 64, [640], 4, 0, 0),
    (BF, 2, 33, 15, 3, 96, 12, [90, 191], 2, 0, 0),
    (HF, 3, 5, 4, 4, 80, 7, [1, 50, 333], 1, 0, 0),
    (BF, 1, 3, 6, 2, 72, 1, [70], 2, 0, 0),
    (HF, 2, 9, 4, 2, 112, 8, [17, 240], 2, 0, 0),
    (BF, 2, 4, 8, 1, 256, 16, [40, 200], 2, 0, 0),
    (BF, 1, 24, 8, 1, 192, 16, [129], 3, 0, 0),
    (HF, 1, 12, 2, 1, 160, 16, [66], 3, 0, 0),
    (BF, 2, 3, 40, 1, 128, 16, [80, 81], 2, 0, 0),
    (BF, 1, 2, 71, 1, 64, 16, [333], 2, 0, 0),
    (BF, 2, 3, 256, 1, 64, 16, [50, 200], 2, 0, 0),     # workgroups within one query
    (FP, 2, 8, 8, 2, 128, 16, [64, 300], 3, 0, 0),
    (FP, 2, 5, 4, 2, 64, 16, [0, 77], 2, 0, 0),
    (FP, 1, 20, 4, 1, 96, 8, [150], 3, 0, 0),
    (FP, 1, 6, 4, 1, 256, 16, [100], 2, 0, 0),
    (FP, 1, 64, 4, 1, 80, 16, [60], 4, 0, 0),
    # head_dims and pages of no vector width
    (BF, 2, 3, 4, 2, 17, 5, [9, 40], 2, 0, 0),
    (HF, 1, 2, 2, 1, 1, 3, [10], 2, 0, 0),
    (FP, 2, 3, 2, 2, 33, 4, [9, 70], 2, 0, 0),
    (BF, 1, 4, 2, 1, 100, 16, [70], 2, 0, 0),
    # windows: shorter than a path, inside a tile, across tiles, with first tokens
    (BF, 2, 16, 8, 2, 128, 16, [200, 3], 1, 1, 0),
    (BF, 2, 16, 8, 2, 128, 16, [200, 3], 1, 5, 2),
    (HF, 2, 64, 8, 2, 64, 16, [300, 40], 1, 40, 3),
    (BF, 3, 12, 8, 2, 128, 16, [500, 70, 0], 2, 100, 4),
    (BF, 2, 8, 16, 2, 96, 12, [400, 150], 3, 128, 64),
    (FP, 2, 7, 4, 2, 128, 16, [300, 20], 2, 33, 5),
    (HF, 1, 64, 32, 1, 128, 16, [700], 2, 200, 70),
    (BF, 1, 4, 8, 2, 256, 8, [300], 2, 64, 1),
]


@pytest.mark.parametrize("shape", TREE_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-T{s[2]}-{s[3]}x{s[4]}x{s[5]}-P{s[6]}-w{s[9]}-s{s[10]}")
def test_tree_matches_oracle(gpu, shape):
    dtype, B, T, Hq, Hkv, D, P, lens, branch, window, sinks = shape
    say(f"tree {shape}")
    case = attention_case(dtype, B, T, Hq, Hkv, D, P, lens, branch=branch, seed=B + T + D)
    check_case(gpu, case, window, sinks, what="default")
    check_case(gpu, case, window, sinks, flags=cabi.QD_FLAG_FORCE_GENERIC, what="VALU kernel")


WINDOW_SHAPES = [
    # dtype, B, Hq, Hkv, D, P, lens, window, sinks
    (BF, 4, 8, 2, 128, 16, [0, 1, 64, 700], 128, 0),
    (BF, 4, 8, 2, 128, 16, [5, 131, 133, 700], 128, 4),
    (HF, 3, 8, 2, 64, 16, [17, 300, 512], 128, 4),
    (HF, 3, 4, 4, 80, 12, [17, 300, 512], 65, 63),
    (BF, 2, 40, 1, 128, 16, [400, 90], 1, 0),
    (BF, 2, 16, 1, 256, 16, [400, 90], 100, 2),
    (FP, 2, 8, 2, 128, 16, [400, 90], 100, 2),
    (FP, 2, 4, 2, 256, 4, [200, 10], 33, 2),
    (FP, 2, 3, 3, 33, 5, [200, 10], 33, 2),
    (BF, 2, 6, 2, 192, 1, [150, 10], 2147483647, 0),
    (BF, 2, 6, 2, 96, 64, [150, 10], 40, 2147483647),
    (HF, 1, 1, 1, 8, 16, [1], 1, 0),
]


@pytest.mark.parametrize("shape", WINDOW_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-{s[2]}x{s[3]}x{s[4]}-P{s[5]}-w{s[7]}-s{s[8]}")
def test_window_matches_oracle(gpu, shape):
    dtype, B, Hq, Hkv, D, P, lens, window, sinks = shape
    say(f"window {shape}")
    case = attention_case(dtype, B, 0, Hq, Hkv, D, P, lens, seed=B + D)
    check_case(gpu, case, window, sinks, what="default")
    check_case(gpu, case, window, sinks, flags=cabi.QD_FLAG_FORCE_GENERIC, what="VALU kernel")


LONG_SHAPES = [
    # dtype, B, T, Hq, Hkv, D, P, lens, window, sinks: contexts that are split over workgroups
    (BF, 2, 4, 8, 1, 128, 16, [9000, 37], 0, 0),
    (BF, 3, 16, 8, 2, 64, 16, [4000, 0, 2500], 0, 0),
    (HF, 2, 64, 8, 2, 128, 16, [3000, 5000], 0, 0),
    (BF, 1, 40, 8, 1, 256, 16, [3000], 0, 0),
    (FP, 2, 6, 8, 2, 128, 16, [3000, 700], 0, 0),
    (BF, 2, 5, 8, 2, 128, 16, [9000, 4000], 3001, 130),
    (BF, 2, 0, 8, 2, 128, 16, [9000, 4000], 5000, 4),
    (HF, 5, 0, 4, 1, 96, 12, [6000, 1, 0, 3000, 2999], 2900, 65),
]


@pytest.mark.parametrize("shape", LONG_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-T{s[2]}-{s[3]}x{s[4]}x{s[5]}-w{s[8]}")
def test_long_contexts_match_oracle(gpu, shape):
    dtype, B, T, Hq, Hkv, D, P, lens, window, sinks = shape
    say(f"long {shape}")
    case = attention_case(dtype, B, T, Hq, Hkv, D, P, lens, seed=D + T, k_scale=1.5)
    check_case(gpu, case, window, sinks, what="default")


def shared_pages_case(dtype, B, T, Hq, Hkv, D, P, lens, width, *, branch=2, seed=0):
    """Many or long sequences on a small pool: their tables name the same pages in different orders."""
    gen = torch.Generator().manual_seed(seed)
    pool = 40 if P > 1 else 400
    table = torch.randint(0, pool, (B, width), generator=gen, dtype=torch.int32)
    q = torch.randn(*((B, T) if T else (B,)), Hq, D, generator=gen).to(dtype)
    k, v = (torch.randn(pool, P, Hkv, D, generator=gen).to(dtype) for _ in range(2))
    masks = tree_masks(gen, B, T, branch, True) if T else None
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32), masks


def lengths(B, hi, *long):
    return list(long) + [(37 * i) % (hi + 1) for i in range(B - len(long))]


MANY_SHAPES = [
    # dtype, B, T, Hq, Hkv, D, P, lens, width, window, sinks, kind
    # the prefix of the costs in a wave's lanes, all of them used, and in LDS
    (BF, 64, 2, 4, 2, 64, 16, lengths(64, 60, 1900, 0, 700), 130, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    (BF, 65, 2, 4, 2, 64, 16, lengths(65, 60, 1900, 0, 700), 130, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    (HF, 300, 1, 4, 1, 64, 16, lengths(300, 90, 0, 0, 1500), 130, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    (FP, 90, 2, 2, 1, 128, 8, lengths(90, 40, 900), 250, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    (BF, 1024, 1, 2, 1, 64, 16, lengths(1024, 30, 3000), 250, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    (BF, 1024, 0, 2, 1, 64, 16, lengths(1024, 30, 3000), 250, 2000, 4, cabi.QD_TREE_MFMA),
    (BF, 70, 2, 2, 1, 64, 16, [0] * 70, 130, 0, 0, cabi.QD_TREE_MFMA_SPLIT),
    # more sequences than the split takes; a workgroup's page list is refilled: one
    # id for a token (pages of 12, 1) and for 16 (pages of 32)
    (BF, 1030, 1, 2, 1, 64, 12, lengths(1030, 20, 2500, 1024, 1025, 0, 2049), 220, 0, 0, cabi.QD_TREE_MFMA),
    (FP, 1030, 1, 2, 1, 64, 1, lengths(1030, 20, 2500, 1024, 1025, 0, 2049), 2600, 0, 0, cabi.QD_TREE_MFMA),
    (BF, 1030, 2, 2, 1, 128, 32, lengths(1030, 20, 16500, 16384, 33000, 0), 1040, 0, 0, cabi.QD_TREE_MFMA),
    (HF, 1030, 0, 2, 1, 64, 1, lengths(1030, 20, 2500, 1024), 2600, 1500, 33, cabi.QD_TREE_MFMA),
]


@pytest.mark.parametrize("shape", MANY_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-T{s[2]}-{s[5]}-P{s[6]}-w{s[9]}-n{max(s[7])}")
def test_many_sequences_match_oracle(gpu, shape):
    dtype, B, T, Hq, Hkv, D, P, lens, width, window, sinks, kind = shape
    say(f"many {shape[:7]} {width} {window} {sinks}")
    assert cabi.gqa_decode_tree_info(B, max(T, 1), Hq, Hkv, D, P, width, int(T > 0), window, sinks,
                                     cabi.DTYPE[dtype])[0] == kind
    case = shared_pages_case(dtype, B, T, Hq, Hkv, D, P, lens, width, seed=B + D)
    check_case(gpu, case, window, sinks, what="default")


REFILL_SHAPES = [
    # dtype, B, T, Hq, Hkv, D, P, longest, window, sinks: ranges of more tokens than a page list holds (1024 ids,
    # of one token or of 16)
    (BF, 200, 1, 2, 1, 64, 12, 5200, 0, 0),
    (FP, 100, 3, 2, 1, 64, 1, 12000, 0, 0),
    (BF, 60, 2, 24, 2, 72, 12, 9000, 0, 0),
    (BF, 200, 0, 2, 1, 64, 12, 9000, 5200, 70),
    (BF, 64, 1, 1, 1, 8, 16, 190000, 0, 0),
    (FP, 40, 2, 2, 1, 8, 64, 300000, 0, 0),
    (BF, 64, 0, 1, 1, 8, 32, 220000, 190000, 33),
]


@pytest.mark.parametrize("shape", REFILL_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-T{s[2]}-{s[3]}x{s[4]}x{s[5]}-P{s[6]}-w{s[8]}")
def test_ranges_that_refill_their_page_list(gpu, shape):
    """Split contexts whose ranges begin inside an item and pass the end of a page list.  About every 50th page
    holds keys that count, one of 30 such pages; the keys of all others score e^-100 of them, so that each page
    listed wrongly shows.  Sums round only where something is added: the tokens that count."""
    dtype, B, T, Hq, Hkv, D, P, longest, window, sinks = shape
    say(f"refill {shape}")
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(longest * 4 // 5, longest + 1, (B,), generator=gen, dtype=torch.int32)
    width = -(-(longest + T) // P) + 1
    kind, groups, _ = cabi.gqa_decode_tree_info(B, max(T, 1), Hq, Hkv, D, P, width, int(T > 0), window, sinks,
                                                cabi.DTYPE[dtype])
    assert kind == cabi.QD_TREE_MFMA_SPLIT
    seen = sum(min(n, window + sinks) if window else n for n in lens.tolist())
    assert Hkv * seen / groups > 1.1 * 1024 * (16 if P % 16 == 0 else 1)
    counts = torch.rand(B, width, generator=gen) < 0.02
    table = torch.where(counts, torch.randint(1, 31, (B, width), generator=gen), 0).int().contiguous()
    q = (0.5 + torch.rand(*((B, T) if T else (B,)), Hq, D, generator=gen)).to(dtype)
    k = torch.randn(31, P, Hkv, D, generator=gen).to(dtype)
    v = torch.randn(31, P, Hkv, D, generator=gen).to(dtype)
    k[0], v[0] = -105 / math.sqrt(D), 5.0               # a score of -105 times q's mean, about 1
    masks = [[(2 << t) - 1 for t in range(T)] for _ in range(B)] if T else None
    want, spread, size = attention_want(q, k, v, table, lens, masks, window, sinks, 1 / math.sqrt(D))
    out = attend(gpu, (q, k, v, table, lens, masks), window, sinks)
    most = int(counts.sum(1).max()) * P
    attention_check(out, want, spread, size, dtype, D, most, f"{groups} ranges, {most} tokens that count")


def test_launch_limit_of_sequences(gpu):
    """Almost 2^24 rows in one call, a workgroup for each: parts of the batch by themselves are bitwise the same."""
    say("2^24 rows")
    B = 4_000_000
    gen = torch.Generator(device=gpu).manual_seed(0)
    q = torch.randn(B, 4, 8, generator=gen, device=gpu).to(BF)
    k, v = (torch.randn(50, 16, 4, 8, generator=gen, device=gpu).to(BF) for _ in range(2))
    table = torch.randint(0, 50, (B, 1), generator=gen, device=gpu, dtype=torch.int32)
    lens = torch.randint(0, 17, (B,), generator=gen, device=gpu, dtype=torch.int32)
    whole = attention_amd.gqa_decode_window(q, k, v, table, lens, window=12, sinks=2)
    for at in (0, 1_500_000, B - 2000):
        part = slice(at, at + 2000)
        assert torch.equal(whole[part], attention_amd.gqa_decode_window(q[part], k, v, table[part], lens[part], window=12,
                                                                        sinks=2))


@pytest.mark.parametrize("seed", range(4))
def test_random_calls_match_oracle(gpu, seed):
    """Types, heads, pages, lengths, trees and windows at random; what one random query does not see holds NaN, Inf
    or large values."""
    from oracle.serving_oracle import visible
    rng = random.Random(seed)
    for n in range(60):
        dtype, D, P = rng.choice([BF, HF, FP]), rng.choice([8, 40, 64, 72, 80, 96, 112, 128, 160, 192, 256]), \
            rng.choice([1, 3, 4, 8, 12, 16, 16, 32, 48, 64])
        Hkv, group = rng.choice([1, 2, 3]), rng.choice([1, 2, 4, 5, 8, 16, 40])
        T, B = rng.choice([0, 1, 2, 5, 8, 16, 33, 64]), rng.randint(1, 4)
        lens = [rng.choice([0, 1, rng.randint(0, 40), rng.randint(0, 300), rng.randint(0, 1000)]) for _ in range(B)]
        window = rng.choice([0, 0, 1, 7, 40, 130, 700]) or (0 if T else 50)
        sinks = rng.choice([0, 4, 20, 200]) if window else 0
        if sum(lens) * max(T, 1) * group * Hkv * D > 1e8:
            lens = [length % 30 for length in lens]
        say(f"{n}: {dtype} T{T} {group * Hkv}x{Hkv}x{D} P{P} {lens} window {window} sinks {sinks}")
        q, k, v, table, dl, masks = attention_case(dtype, B, T, group * Hkv, Hkv, D, P, lens, branch=rng.choice([1, 2, 5]),
                                                   seed=n, spare=rng.choice([1, 2, 40]))
        if masks and rng.random() < 0.3:
            masks = [[m if rng.random() < 0.8 else 0 for m in row] for row in masks]
        want, spread, size = attention_want(q, k, v, table, dl, masks, window, sinks, 1 / math.sqrt(D))
        b, t = rng.randrange(B), rng.randrange(max(T, 1))
        sees = visible(lens[b], masks[b] if masks else None, T, table.shape[1] * P, window, sinks)[t]
        used = torch.zeros(k.shape[0], P, dtype=torch.bool)
        for tok in np.nonzero(sees)[0]:
            used[int(table[b, tok // P]), tok % P] = True
        clean = attend(gpu, (q, k, v, table, dl, masks), window, sinks)
        attention_check(clean, want, spread, size, dtype, D, max(lens) + 64, "clean")
        k[~used] = rng.choice([math.nan, math.inf, 1.0, -3e4])
        v[~used] = rng.choice([math.nan, math.inf, -math.inf, 3e4])
        out = attend(gpu, (q, k, v, table, dl, masks), window, sinks)
        at = (b, t) if T else b
        attention_check(out[at], want[at], spread[at], size[at], dtype, D, max(lens) + 64, "poisoned")


def test_large_scores_stay_exact(gpu):
    """Scores of a few hundred: one token takes all of the weight."""
    say("large scores")
    for dtype in (BF, HF, FP):
        case = attention_case(dtype, 2, 5, 8, 2, 128, 16, [200, 64], k_scale=20.0)
        check_case(gpu, case, what=str(dtype))


def test_one_draft_is_decode(gpu):
    """A tree of one drafted token, and a window as long as the context, are gqa_decode."""
    say("T = 1 against gqa_decode")
    q, k, v, table, lens, _ = attention_case(BF, 4, 0, 8, 2, 128, 16, [1, 16, 200, 500])
    d = [x.to(gpu) for x in (q, k, v, table, lens)]
    want = attention_amd.gqa_decode(*d).float()
    window = attention_amd.gqa_decode_window(*d, window=500).float()
    one = torch.ones(4, 1, dtype=torch.int64, device=gpu)
    tree = attention_amd.gqa_decode_tree(d[0][:, None].contiguous(), *d[1:4], d[4] - 1, one)[:, 0].float()
    # Both round the same value: at most a step of bf16 apart where the sums fall on different sides.
    for got in (window, tree):
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-5).all()


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("T,window,sinks", [(16, 0, 0), (16, 24, 3), (40, 7, 1), (0, 70, 3)])
def test_hidden_tokens_cannot_reach_a_row(gpu, dtype, T, window, sinks):
    """NaN and Inf in everything that a query does not see: other branches, tokens past the drafted ones, tokens
    before the window (their page mates are seen), freed pages."""
    say(f"poison {dtype} T{T} window {window}")
    lens = [0, 70, 333]
    q, k, v, table, lens, masks = attention_case(dtype, 3, T, 8, 2, 128, 16, lens, branch=4, window=window, seed=5)
    from oracle.serving_oracle import visible
    P = 16
    clean, spread, size = attention_want(q, k, v, table, lens, masks, window, sinks, 0.1)
    bad = {n: x.clone() for n, x in (("k", k), ("v", v))}
    used = torch.zeros(k.shape[0], P, dtype=torch.bool)
    for b in range(3):
        sees = visible(int(lens[b]), masks[b] if masks else None, T, table.shape[1] * P, window, sinks)
        for tok in np.nonzero(sees.any(0))[0]:
            used[int(table[b, tok // P]), tok % P] = True
    bad["k"][~used] = float("nan")
    bad["v"][~used] = float("nan")
    out = attend(gpu, (q, bad["k"], bad["v"], table, lens, masks), window, sinks, scale=0.1)
    attention_check(out, clean, spread, size, dtype, 128, 400, "unseen by all")
    if not T:
        return
    # Seen by some: poison one drafted token after the other; the rows that do not see it keep their values.
    for j, poison in ((0, float("inf")), (3, float("nan")), (T - 1, float("-inf"))):
        bk, bv = bad["k"].clone(), bad["v"].clone()
        reach = np.zeros((3, T), dtype=bool)
        for b in range(3):
            tok = int(lens[b]) + j
            bk[int(table[b, tok // P]), tok % P] = poison
            bv[int(table[b, tok // P]), tok % P, :, 5] = poison
            reach[b] = visible(int(lens[b]), masks[b], T, table.shape[1] * P, window, sinks)[:, tok]
        for flags in (None, cabi.QD_FLAG_FORCE_GENERIC):
            out = attend(gpu, (q, bk, bv, table, lens, masks), window, sinks, flags=flags, scale=0.1).float().cpu()
            keep = torch.from_numpy(~reach)
            attention_check(out[keep].to(dtype), clean[~reach], spread[~reach], size[~reach], dtype, 128, 400,
                            f"without drafted token {j}")
            assert not torch.isfinite(out[~keep]).all(-1).any(), "a row that sees NaN must say so"


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("T,group,window,sinks", [(8, 16, 130, 0), (8, 16, 40, 30), (12, 16, 5, 3), (3, 64, 60, 2),
                                                  (5, 71, 33, 0), (4, 256, 100, 7), (2, 16, 1, 0)])
def test_hidden_tokens_where_workgroups_hold_one_query(gpu, dtype, T, group, window, sinks):
    """As above, with rows cut so that a workgroup serves heads of one query, whose window begins later than the
    first query's."""
    say(f"poison {dtype} T{T} group {group} window {window} sinks {sinks}")
    from oracle.serving_oracle import visible
    lens, P = [172, 8, 0, 300], 16
    q, k, v, table, lens, _ = attention_case(dtype, 4, T, 2 * group, 2, 72, P, lens, seed=T)
    masks = [[(2 << t) - 1 for t in range(T)],                         # a chain
             [(2 << t) - 1 if t else 0 for t in range(T)],             # whose first token is padding
             [1 | 1 << t for t in range(T)], [1 << t for t in range(T)]]
    clean, spread, size = attention_want(q, k, v, table, lens, masks, window, sinks, 0.1)
    for b in range(4):
        # One query at a time: everything that it does not see is poisoned.
        for t in range(T):
            seen = visible(int(lens[b]), masks[b], T, table.shape[1] * P, window, sinks)[t]
            used = torch.zeros(k.shape[0], P, dtype=torch.bool)
            for tok in np.nonzero(seen)[0]:
                used[int(table[b, tok // P]), tok % P] = True
            bk, bv = k.clone(), v.clone()
            bk[~used] = float("nan")
            bv[~used] = float("inf")
            out = attend(gpu, (q, bk, bv, table, lens, masks), window, sinks, scale=0.1)
            attention_check(out[b, t], clean[b, t], spread[b, t], size[b, t], dtype, 72, 400, f"sequence {b} query {t}")


def test_hidden_values_in_window_edge(gpu):
    """Infinite values (finite keys) in a token that only the earlier queries' windows hold."""
    say("window edge")
    q, k, v, table, lens, _ = attention_case(BF, 1, 8, 8, 2, 128, 16, [200], seed=3)
    masks = [[(1 << t + 1) - 1 for t in range(8)]]
    case = (q, k, v, table, lens, masks)
    clean, spread, size = attention_want(*case, 50, 2, 0.1)
    tok = 200 - 50 + 4                         # the window's first token of query 3; queries 4.. no longer see it
    v = v.clone()
    v[int(table[0, tok // 16]), tok % 16] = float("inf")
    out = attend(gpu, (q, k, v, table, lens, masks), 50, 2, scale=0.1).cpu()
    assert not torch.isfinite(out[0, :4]).any()
    attention_check(out[:, 4:], clean[:, 4:], spread[:, 4:], size[:, 4:], BF, 128, 64, "after the edge")


def test_freed_pages_are_never_read(gpu):
    """Table entries before the window are -1 or far outside, the pages poisoned: bitwise the same result."""
    say("freed pages")
    q, k, v, table, lens, _ = attention_case(BF, 3, 0, 8, 2, 128, 16, [700, 90, 2000])
    base = attend(gpu, (q, k, v, table, lens, None), 100, 4)
    t2, k2, v2 = table.clone(), k.clone(), v.clone()
    for b, n in enumerate(lens.tolist()):
        for page in list(range(1, max(1, (n - 100) // 16))) + list(range(-(-n // 16), table.shape[1])):
            k2[int(table[b, page])] = float("nan")
            v2[int(table[b, page])] = float("nan")
            t2[b, page] = -1 if page % 2 else 2 ** 31 - 1
    assert torch.equal(base, attend(gpu, (q, k2, v2, t2, lens, None), 100, 4))


def test_lengths_and_tables_out_of_range(gpu):
    """Lengths past the table are clamped to it (drafted tokens then lie outside and are not seen), negative ones
    are 0, page ids outside the pool are clamped."""
    say("lengths out of range")
    q, k, v, table, _, masks = attention_case(BF, 4, 6, 8, 2, 64, 16, [64] * 4, ragged=False, spare=0)
    cap = table.shape[1] * 16
    lens = torch.tensor([cap - 2, cap + 100, -5, 2 ** 31 - 1], dtype=torch.int32)
    check_case(gpu, (q, k, v, table, lens.clamp(max=cap), masks), what="at the end of the table")
    want = attend(gpu, (q, k, v, table, lens.clamp(0, cap), masks))
    assert torch.equal(want, attend(gpu, (q, k, v, table, lens, masks)))
    t2 = table.clone()
    t2[0, 1], t2[1, 0] = -7, 2 ** 31 - 1
    t3 = t2.clamp(0, k.shape[0] - 1)
    assert torch.equal(attend(gpu, (q, k, v, t3, lens, masks)), attend(gpu, (q, k, v, t2, lens, masks)))


def test_padded_rows_are_zero_and_bits_past_the_count_ignored(gpu):
    say("padding")
    q, k, v, table, lens, _ = attention_case(HF, 2, 5, 8, 2, 64, 16, [100, 7])
    masks = [[1, 3, 0, 9, 0], [0] * 5]
    out = check_case(gpu, (q, k, v, table, lens, masks), what="padded")
    assert (out[0, 2] == 0).all() and (out[1] == 0).all()
    high = [[m | (0x5A << 5) if m else 0 for m in row] for row in masks]
    assert torch.equal(out, attend(gpu, (q, k, v, table, lens, high)))
    assert (attend(gpu, (q, k, v, table, lens, [[1 << 9] * 5, [1 << 63] * 5])) == 0).all()


def test_tree_rows_do_not_depend_on_the_batch_around_them(gpu):
    say("batch independence")
    q, k, v, table, lens, masks = attention_case(BF, 3, 4, 8, 2, 128, 16, [300, 20, 800])
    whole = attend(gpu, (q, k, v, table, lens, masks)).float()
    for b in range(3):
        one = attend(gpu, (q[b:b + 1], k, v, table[b:b + 1].contiguous(), lens[b:b + 1], masks[b:b + 1])).float()
        # Contexts may be split elsewhere: a step of bf16 at most.
        assert ((one[0] - whole[b]).abs() <= 2.0 ** -7 * whole[b].abs() + 1e-4).all()


def test_repeats_are_bitwise_equal(gpu):
    say("repeats")
    case = attention_case(BF, 4, 16, 16, 2, 128, 16, [3000, 10, 700, 1500])
    first = attend(gpu, case)
    for _ in range(3):
        assert torch.equal(first, attend(gpu, case))


def test_unaligned_tensors(gpu):
    say("unaligned")
    q, k, v, table, lens, masks = attention_case(BF, 2, 3, 4, 2, 64, 16, [50, 7])
    want, spread, size = attention_want(q, k, v, table, lens, masks, 0, 0, 0.125)

    def shifted(x):
        big = torch.empty(x.numel() + 1, dtype=x.dtype, device=gpu)
        big[1:] = x.reshape(-1).to(gpu)
        return big[1:].view(x.shape)

    for which in range(3):
        args = [shifted(x) if i == which else x.to(gpu) for i, x in enumerate((q, k, v))]
        out = attention_amd.gqa_decode_tree(*args, table.to(gpu), lens.to(gpu), signed(masks).to(gpu))
        attention_check(out, want, spread, size, BF, 64, 60, f"tensor {which} off by one element")


def test_empty_batches(gpu):
    say("empty")
    k = torch.zeros(3, 16, 2, 64, dtype=BF, device=gpu)
    t, n = torch.zeros(0, 2, dtype=torch.int32, device=gpu), torch.zeros(0, dtype=torch.int32, device=gpu)
    q = torch.zeros(0, 4, 8, 64, dtype=BF, device=gpu)
    assert attention_amd.gqa_decode_tree(q, k, k, t, n, torch.zeros(0, 4, dtype=torch.int64, device=gpu)).shape == q.shape
    assert attention_amd.gqa_decode_window(q[:, 0], k, k, t, n, window=4).shape == (0, 8, 64)
    x = torch.zeros(0, 2, 64, dtype=BF, device=gpu)
    out = attention_amd.qk_norm_rope_write(q[:, 0], x, x, torch.zeros(4, 64, device=gpu), n, k, k.clone(), n.long())
    assert out.shape == (0, 8, 64)
    attention_amd.kv_compact([], t, n, torch.zeros(0, 4, dtype=torch.int32, device=gpu))
    attention_amd.kv_compact([k], t, n, torch.zeros(0, 4, dtype=torch.int32, device=gpu))
    attention_amd.kv_compact([k], torch.zeros(1, 2, dtype=torch.int32, device=gpu),
                             torch.zeros(1, dtype=torch.int32, device=gpu),
                             torch.zeros(1, 0, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()


def test_refusals_name_the_argument(gpu):
    say("refusals")
    q, k, v, table, lens, masks = (x.to(gpu) if isinstance(x, torch.Tensor) else x
                                   for x in attention_case(BF, 2, 3, 4, 2, 64, 16, [50, 7]))
    m = signed(masks).to(gpu)
    with pytest.raises(RuntimeError, match="tree_mask must be int64"):
        attention_amd.gqa_decode_tree(q, k, v, table, lens, m.int())
    with pytest.raises(RuntimeError, match="q must be contiguous"):
        attention_amd.gqa_decode_tree(q.transpose(1, 2), k, v, table, lens, m)
    with pytest.raises(RuntimeError, match="context_lens must be a CUDA tensor"):
        attention_amd.gqa_decode_tree(q, k, v, table, lens.cpu(), m)
    with pytest.raises(RuntimeError, match="sinks must be in"):
        attention_amd.gqa_decode_tree(q, k, v, table, lens, m, sinks=4)
    with pytest.raises(RuntimeError, match="window must be in"):
        attention_amd.gqa_decode_window(q[:, 0].contiguous(), k, v, table, lens, window=0)
    with pytest.raises(RuntimeError, match="the heads of a token must be contiguous"):
        attention_amd.qk_norm_rope_write(q[:, 0].transpose(1, 2), k[:2, 0], k[:2, 0], torch.zeros(4, 4, device=gpu), lens,
                                         k, v, lens.long())
    with pytest.raises(RuntimeError, match="caches must not overlap"):
        attention_amd.kv_compact([k, v, k], table, lens, lens[:, None].contiguous())
    with pytest.raises(RuntimeError, match="of one shape and dtype"):
        attention_amd.kv_compact([k, v.float()], table, lens, lens[:, None].contiguous())
    with pytest.raises(RuntimeError, match="of one shape and dtype"):
        attention_amd.kv_compact([k, v.cpu()], table, lens, lens[:, None].contiguous())


def test_attention_on_other_streams(gpu):
    """Calls in flight on two streams at once, each with its own workspace."""
    say("streams")
    cases = [attention_case(BF, 3, 8, 8, 2, 128, 16, [3000, 100, 1200], seed=s) for s in range(2)]
    wants = [attend(gpu, c) for c in cases]
    args = [([x.to(gpu) for x in c[:5]], signed(c[5]).to(gpu)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(attention_amd.gqa_decode_tree(*args[i][0], args[i][1]))
    torch.cuda.synchronize()
    for want, got in zip(wants, outs):
        assert all(torch.equal(want, o) for o in got)


def test_pool_past_four_gigabytes(gpu):
    """Pages at the end of a pool whose byte and element offsets pass 32 bits."""
    say("large pool")
    small_q, k, v, table, lens, masks = attention_case(BF, 2, 4, 4, 2, 128, 16, [100, 260], ragged=False)
    pages = (1 << 32) // (16 * 2 * 128) + 700          # more than 2^32 elements, 2^33 bytes
    far_k = torch.empty(pages, 16, 2, 128, dtype=BF, device=gpu)
    far_v = torch.empty(pages, 16, 2, 128, dtype=BF, device=gpu)
    at = pages - k.shape[0]
    far_k[at:], far_v[at:] = k.to(gpu), v.to(gpu)
    want = attend(gpu, (small_q, k, v, table, lens, masks))
    got = attention_amd.gqa_decode_tree(small_q.to(gpu), far_k, far_v, (table + at).to(gpu), lens.to(gpu),
                                        signed(masks).to(gpu))
    assert torch.equal(want, got)
    out = torch.empty_like(want)
    rc = cabi.gqa_decode_tree(small_q.to(gpu), far_k, far_v, (table + at).to(gpu), lens.to(gpu), signed(masks).to(gpu),
                              out, scale=1 / math.sqrt(128), flags=cabi.QD_FLAG_FORCE_GENERIC)
    assert rc == 0
    assert ((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-5).all()
    accepted = torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=gpu)
    attention_amd.kv_compact([far_k, far_v], (table + at).to(gpu), lens.to(gpu), accepted)
    for far, near in ((far_k, k), (far_v, v)):
        ref = oracle_compact(near.float().numpy(), table.numpy(), lens.numpy(), accepted.cpu().numpy())
        assert np.array_equal(far[at:].float().cpu().numpy(), ref)
    key = torch.randn(1, 2, 128, device=gpu).to(BF)
    attention_amd.qk_norm_rope_write(key, key, key, torch.zeros(1, 0, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu),
                                     far_k, far_v, torch.tensor([pages * 16 - 1], device=gpu))
    assert torch.equal(far_k[-1, -1], key[0]) and torch.equal(far_v[-1, -1], key[0])


# ---- Norm, rotation and write ----------------------------------------------------


WRITE_SHAPES = [
    # dtype, weights' dtype, N, Hq, Hkv, D, rotary, interleaved
    (BF, BF, 5, 8, 2, 128, 128, False),
    (BF, FP, 5, 8, 2, 128, 128, True),
    (HF, HF, 1, 8, 2, 64, 64, False),
    (HF, HF, 3, 4, 4, 80, 80, False),
    (HF, FP, 7, 3, 1, 96, 48, False),
    (BF, BF, 2, 71, 1, 72, 72, False),
    (BF, BF, 9, 5, 5, 112, 56, True),
    (BF, BF, 4, 16, 8, 256, 256, False),
    (BF, BF, 4, 16, 8, 192, 64, False),
    (HF, HF, 4, 2, 1, 160, 160, True),
    (FP, FP, 6, 8, 2, 128, 128, False),
    (FP, FP, 6, 8, 2, 256, 128, True),
    (FP, FP, 3, 2, 2, 72, 72, False),
    (BF, BF, 3, 2, 1, 17, 10, False),
    (FP, FP, 3, 2, 1, 33, 32, True),
    (HF, HF, 3, 2, 1, 100, 4, False),
    (BF, BF, 3, 2, 1, 64, 0, False),
    (BF, BF, 3, 2, 1, 1, 0, False),
    (BF, BF, 4, 2, 1, 64, 20, False),
    (BF, BF, 4, 2, 1, 64, 6, True),
    (BF, BF, 300, 32, 8, 128, 128, False),
]


def write_case(dtype, wdtype, N, Hq, Hkv, D, rot, seed=0, packed=True):
    gen = torch.Generator().manual_seed(seed)
    heads = Hq + 2 * Hkv
    qkv = (3 * torch.randn(N, heads, D, generator=gen)).to(dtype)
    positions = torch.randint(0, 500, (N,), generator=gen, dtype=torch.int32)
    angle = torch.arange(500, dtype=torch.float64)[:, None] * 0.7 ** torch.arange(rot // 2, dtype=torch.float64)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float()
    pool = -(-N // 4) + 3
    kc, vc = (torch.randn(pool, 4, Hkv, D, generator=gen).to(dtype) for _ in range(2))
    slots = torch.randperm(pool * 4, generator=gen)[:N]
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=gen)).to(wdtype) for _ in range(2))
    return qkv, cs, positions, kc, vc, slots, qw, kw


def write_check(got, want, magnitude, dtype, D, what):
    tol = HALF[dtype] * np.abs(want) + (D + 16) * U * magnitude + TINY[dtype]
    off = np.abs(f64(got) - want) / tol
    print(f"[case] {what}: {off.max():.3f} of the tolerance", flush=True)
    assert off.max() <= 1.0, what


def pair_sizes(x, weight, eps, rot, interleaved):
    """|a| + |b| of the pair that each element is turned in."""
    y = np.abs(x)
    if weight is not None:
        y = y / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.abs(weight)
    z = y.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        z[..., a] = z[..., b] = y[..., a] + y[..., b]
    return z


def run_write(gpu, case, Hq, Hkv, eps, interleaved, use_qw=True, use_kw=True):
    qkv, cs, positions, kc, vc, slots, qw, kw = case
    d = qkv.to(gpu)
    q, key, value = d.split([Hq, Hkv, Hkv], dim=1)
    dk, dv = kc.to(gpu), vc.to(gpu)
    out = attention_amd.qk_norm_rope_write(q, key, value, cs.to(gpu), positions.to(gpu), dk, dv, slots.to(gpu),
                                           q_weight=qw.to(gpu) if use_qw else None,
                                           k_weight=kw.to(gpu) if use_kw else None, eps=eps, interleaved=interleaved)
    torch.cuda.synchronize()
    assert out.is_contiguous() and torch.equal(d.cpu(), qkv)
    return out, dk, dv


def check_write(gpu, case, Hq, Hkv, eps, interleaved, use_qw=True, use_kw=True, what=""):
    qkv, cs, positions, kc, vc, slots, qw, kw = case
    dtype, D = qkv.dtype, qkv.shape[2]
    out, dk, dv = run_write(gpu, case, Hq, Hkv, eps, interleaved, use_qw, use_kw)
    x = f64(qkv)
    q, key, value = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    wq, wk = f64(qw) if use_qw else None, f64(kw) if use_kw else None
    want, wkc, wvc = oracle_write(q, key, value, f64(cs), positions.numpy(), f64(kc), f64(vc), slots.numpy(), wq, wk, eps,
                                  interleaved)
    rot = cs.shape[1]
    size = pair_sizes(q, wq, eps, rot, interleaved)
    write_check(out, want, size, dtype, D, f"{what} q")
    flat = f64(kc).reshape(-1, Hkv, D) * 0
    keep = (slots >= 0) & (slots < flat.shape[0]) & (positions >= 0) & (positions < cs.shape[0])
    flat[slots[keep].numpy()] = pair_sizes(key, wk, eps, rot, interleaved)[keep.numpy()]
    write_check(dk, wkc, flat.reshape(kc.shape), dtype, D, f"{what} k")
    assert np.array_equal(f64(dv), wvc)
    untouched = np.ones(flat.shape[0], dtype=bool)
    untouched[slots[keep].numpy()] = False
    assert np.array_equal(f64(dk).reshape(flat.shape)[untouched], f64(kc).reshape(flat.shape)[untouched])


@pytest.mark.parametrize("shape", WRITE_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-N{s[2]}-{s[3]}x{s[4]}x{s[5]}-r{s[6]}-{'i' if s[7] else 'h'}")
def test_write_matches_oracle(gpu, shape):
    dtype, wdtype, N, Hq, Hkv, D, rot, interleaved = shape
    say(f"write {shape}")
    case = write_case(dtype, wdtype, N, Hq, Hkv, D, rot, seed=N + D)
    check_write(gpu, case, Hq, Hkv, 1e-6, interleaved, what="both norms")
    check_write(gpu, case, Hq, Hkv, 0.5, interleaved, use_kw=False, what="query norm")
    check_write(gpu, case, Hq, Hkv, 1e-6, interleaved, use_qw=False, what="key norm")
    check_write(gpu, case, Hq, Hkv, 1e-6, interleaved, False, False, what="no norm")


def test_write_skips_what_lies_outside(gpu):
    say("write outside")
    for D in (128, 17):
        case = list(write_case(BF, BF, 8, 4, 2, D, 16))
        rows = case[3].shape[0] * 4
        case[2] = torch.tensor([0, 499, -1, 500, 7, 8, 2 ** 31 - 1, 9], dtype=torch.int32)
        case[5] = torch.tensor([0, rows - 1, 3, 4, -1, rows, 5, 1 << 40])
        check_write(gpu, tuple(case), 4, 2, 1e-6, False, what=f"D{D}")
        out, _, _ = run_write(gpu, tuple(case), 4, 2, 1e-6, False)
        assert (out[[2, 3, 6]] == 0).all()


def test_write_zero_rows_and_large_values(gpu):
    """A zero row stays zero under the norm; values near fp16's end do not overflow in the sum of squares."""
    say("write extremes")
    case = list(write_case(HF, FP, 4, 4, 2, 128, 128))
    case[0][0] = 0
    case[0][1] = 60000
    check_write(gpu, tuple(case), 4, 2, 1e-6, False, what="extremes")


def test_write_strided_contiguous_and_unaligned_agree(gpu):
    say("write strides")
    qkv, cs, positions, kc, vc, slots, qw, kw = write_case(BF, BF, 6, 8, 2, 128, 128)
    want, wk, wv = run_write(gpu, (qkv, cs, positions, kc, vc, slots, qw, kw), 8, 2, 1e-6, False)
    q, key, value = (x.contiguous().to(gpu) for x in qkv.split([8, 2, 2], dim=1))
    rest = dict(q_weight=qw.to(gpu), k_weight=kw.to(gpu))

    def call(q, key, value, k2, v2, **kw2):
        return attention_amd.qk_norm_rope_write(q, key, value, cs.to(gpu), positions.to(gpu), k2, v2, slots.to(gpu),
                                                **{**rest, **kw2})

    k2, v2 = kc.to(gpu), vc.to(gpu)
    assert torch.equal(want, call(q, key, value, k2, v2)) and torch.equal(wk, k2) and torch.equal(wv, v2)

    def shifted(x, by=1):
        big = torch.empty(x.numel() + by, dtype=x.dtype, device=gpu)
        big[by:] = x.reshape(-1)
        return big[by:].view(x.shape)

    for by in (1, 2):
        k2, v2 = shifted(kc.to(gpu), by), shifted(vc.to(gpu), by)
        got = call(shifted(q, by), shifted(key, by), shifted(value, by), k2, v2)
        # Another order of the sum of squares: a step of bf16 where a value falls on a border.
        assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs()).all()
        assert ((k2.float() - wk.float()).abs() <= 2.0 ** -7 * wk.float().abs()).all() and torch.equal(v2, wv)
    # One token's rows for all tokens (stride 0).
    k2, v2 = kc.to(gpu), vc.to(gpu)
    same = call(q[:1].expand(6, -1, -1), key[:1].expand(6, -1, -1), value[:1].expand(6, -1, -1), k2, v2)
    k3, v3 = kc.to(gpu), vc.to(gpu)
    full = call(*(x[:1].repeat(6, 1, 1) for x in (q, key, value)), k3, v3)
    assert torch.equal(same, full) and torch.equal(k2, k3) and torch.equal(v2, v3)


def test_write_caches_of_one_allocation(gpu):
    """Caches side by side in one tensor are written; one tensor for both is refused, before anything is written."""
    say("write caches")
    qkv, cs, positions, kc, vc, slots, qw, kw = write_case(BF, BF, 6, 8, 2, 128, 128)
    want, wk, wv = run_write(gpu, (qkv, cs, positions, kc, vc, slots, qw, kw), 8, 2, 1e-6, False)
    q, key, value = qkv.to(gpu).split([8, 2, 2], dim=1)
    rest = [x.to(gpu) for x in (cs, positions)]
    pool = torch.stack([vc, kc]).to(gpu)
    out = attention_amd.qk_norm_rope_write(q, key, value, *rest, pool[1], pool[0], slots.to(gpu), q_weight=qw.to(gpu),
                                           k_weight=kw.to(gpu), eps=1e-6)
    assert torch.equal(out, want) and torch.equal(pool[1], wk) and torch.equal(pool[0], wv)
    before = pool.clone()
    with pytest.raises(RuntimeError, match="k_cache and v_cache must not overlap"):
        attention_amd.qk_norm_rope_write(q, key, value, *rest, pool[0], pool[0], slots.to(gpu))
    torch.cuda.synchronize()
    assert torch.equal(pool, before)


# ---- Compaction ------------------------------------------------------------------


def compact_case(dtype, B, A, P, tail, lens, seed=0, caches=2):
    gen = torch.Generator().manual_seed(seed)
    width = max(-(-(n + A) // P) for n in lens) + 1
    N = B * width + 2
    table = torch.randperm(N, generator=gen)[:B * width].view(B, width).int().contiguous()
    pools = [torch.randn(N, P, *tail, generator=gen).to(dtype) for _ in range(caches)]
    return pools, table, torch.tensor(lens, dtype=torch.int32)


def check_compact(gpu, pools, table, lens, accepted):
    dev = [p.to(gpu) for p in pools]
    attention_amd.kv_compact(dev, table.to(gpu), lens.to(gpu), accepted.to(gpu))
    torch.cuda.synchronize()
    for d, p in zip(dev, pools):
        want = oracle_compact(p.float().numpy(), table.numpy(), lens.numpy(), accepted.numpy())
        assert np.array_equal(d.float().cpu().numpy(), want)


COMPACT_SHAPES = [
    # dtype, B, A, P, tail, lens, caches
    (BF, 3, 4, 16, (8, 128), [0, 15, 100], 2),
    (HF, 2, 16, 16, (2, 64), [7, 31], 2),
    (BF, 2, 17, 12, (2, 64), [7, 30], 4),
    (FP, 2, 64, 16, (4, 128), [5, 90], 2),
    (BF, 1, 64, 1, (8, 128), [33], 1),
    (BF, 2, 8, 64, (576,), [60, 10], 3),        # latent caches
    (HF, 2, 8, 7, (3, 17), [5, 20], 2),         # 102-byte rows
    (FP, 2, 8, 7, (1, 3), [5, 20], 2),
    (BF, 1, 5, 4, (1, 1), [3], 1),
    (BF, 5, 6, 16, (4, 64), [1, 2, 3, 4, 5], 130),
    (FP, 1, 3, 16, (128, 256), [14], 1),        # rows of many column blocks
]


@pytest.mark.parametrize("shape", COMPACT_SHAPES, ids=lambda s: f"{str(s[0])[6:]}-B{s[1]}-A{s[2]}-P{s[3]}-{'x'.join(map(str, s[4]))}-{s[6]}")
def test_compact_matches_oracle(gpu, shape):
    dtype, B, A, P, tail, lens, caches = shape
    say(f"compact {shape}")
    pools, table, lens = compact_case(dtype, B, A, P, tail, lens, caches=caches)
    gen = torch.Generator().manual_seed(1)
    path = torch.sort(torch.rand(B, A, generator=gen).argsort(1)[:, :-(-A // 2)], 1).values
    path = torch.cat([path, torch.full((B, A - path.shape[1]), -1)], 1).int().contiguous()
    check_compact(gpu, pools, table, lens, path)                                                # an accepted path
    check_compact(gpu, pools, table, lens, torch.rand(B, A, generator=gen).argsort(1).int())     # a permutation
    check_compact(gpu, pools, table, lens, torch.randint(-2, A, (B, A), generator=gen).int())    # repeats and gaps
    check_compact(gpu, pools, table, lens, torch.full((B, A), A - 1, dtype=torch.int32))         # one for all


def test_compact_skips_what_lies_outside(gpu):
    say("compact outside")
    pools, table, lens = compact_case(BF, 4, 8, 16, (2, 64), [40] * 4)
    cap = table.shape[1] * 16
    lens = torch.tensor([cap - 3, -1, 2 ** 31 - 1, 30], dtype=torch.int32)
    accepted = torch.tensor([[2, 1, 0, 5, 7, 6, 3, 4]] * 4, dtype=torch.int32)
    table[3, 2] = -1                                    # tokens 32..47
    check_compact(gpu, pools, table, lens, accepted)
    table[3, 2] = pools[0].shape[0]
    check_compact(gpu, pools, table, lens, accepted)
    accepted[0, 0] = 2 ** 31 - 1
    check_compact(gpu, pools, table, lens, accepted)


def test_compact_unaligned_caches(gpu):
    say("compact unaligned")
    pools, table, lens = compact_case(BF, 2, 6, 16, (2, 64), [10, 40])
    accepted = torch.tensor([[1, 3, 5, -1, -1, -1], [0, 2, 4, 5, -1, -1]], dtype=torch.int32)
    dev = []
    for p in pools:
        big = torch.empty(p.numel() + 1, dtype=p.dtype, device=gpu)
        big[1:] = p.reshape(-1).to(gpu)
        dev.append(big[1:].view(p.shape))
    attention_amd.kv_compact(dev, table.to(gpu), lens.to(gpu), accepted.to(gpu))
    for d, p in zip(dev, pools):
        want = oracle_compact(p.float().numpy(), table.numpy(), lens.numpy(), accepted.numpy())
        assert np.array_equal(d.float().cpu().numpy(), want)


# ---- The operators together -------------------------------------------------------


def speculative_step(q_in, key, value, cs, positions, caches, slots, table, lens, mask, accepted, weights, window, sinks):
    out = []
    for layer, (kc, vc) in enumerate(caches):
        q = attention_amd.qk_norm_rope_write(q_in[layer], key[layer], value[layer], cs, positions, kc, vc, slots,
                                             q_weight=weights[0], k_weight=weights[1])
        q = q.view(*mask.shape, *q.shape[1:])
        out.append(attention_amd.gqa_decode_tree(q, kc, vc, table, lens, mask, window=window, sinks=sinks))
    attention_amd.kv_compact([c for pair in caches for c in pair], table, lens, accepted)
    return out


def step_case(gpu, dtype=BF, layers=2, B=3, T=8, Hq=8, Hkv=2, D=128, P=16, lens=(70, 5, 300)):
    gen = torch.Generator().manual_seed(9)
    width = -(-(max(lens) + T + 1) // P)
    N = B * width
    table = torch.randperm(N, generator=gen).view(B, width).int()
    masks = tree_masks(gen, B, T, 3, False)
    at = torch.tensor([[n + j for j in range(T)] for n in lens])
    slots = (torch.gather(table.long(), 1, at // P) * P + at % P).reshape(-1)
    positions = torch.tensor([[n + bin(m).count("1") - 1 for m in row] for n, row in zip(lens, masks)], dtype=torch.int32)
    angle = torch.arange(400, dtype=torch.float64)[:, None] * 0.9 ** torch.arange(D // 2, dtype=torch.float64)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float()
    accepted = torch.full((B, T), -1, dtype=torch.int32)
    for b, row in enumerate(masks):
        best = max(row, key=lambda m: bin(m).count("1"))
        path = [j for j in range(T) if best >> j & 1]
        accepted[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
    x = [torch.randn(layers, B * T, Hq + 2 * Hkv, D, generator=gen).to(dtype)]
    caches = [tuple(torch.randn(N, P, Hkv, D, generator=gen).to(dtype) for _ in range(2)) for _ in range(layers)]
    weights = [(1 + 0.2 * torch.randn(D, generator=gen)).to(dtype) for _ in range(2)]
    return dict(qkv=x[0], cs=cs, positions=positions.reshape(-1), caches=caches, slots=slots, table=table.contiguous(),
                lens=torch.tensor(lens, dtype=torch.int32), masks=masks, accepted=accepted, weights=weights, Hq=Hq, Hkv=Hkv)


def on_gpu(gpu, c):
    d = {n: c[n].to(gpu) for n in ("qkv", "cs", "positions", "slots", "table", "lens", "accepted")}
    d["caches"] = [tuple(x.to(gpu) for x in pair) for pair in c["caches"]]
    d["weights"] = [w.to(gpu) for w in c["weights"]]
    d["mask"] = signed(c["masks"]).to(gpu)
    d["parts"] = d["qkv"].split([c["Hq"], c["Hkv"], c["Hkv"]], dim=2)
    return d


def run_step(d, window=None, sinks=0):
    q, key, value = d["parts"]
    return speculative_step(q, key, value, d["cs"], d["positions"], d["caches"], d["slots"], d["table"], d["lens"],
                            d["mask"], d["accepted"], d["weights"], window, sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 2)])
def test_a_step_of_drafting_matches_oracle(gpu, window, sinks):
    """Write, attend and compact two layers, then decode the next token over the compacted cache: the same as
    decoding the accepted path token by token."""
    say("step")
    c = step_case(gpu)
    d = on_gpu(gpu, c)
    outs = run_step(d, window, sinks)
    lens, table = c["lens"].numpy(), c["table"].numpy()
    for layer, (kc, vc) in enumerate(c["caches"]):
        x = f64(c["qkv"][layer])
        Hq, Hkv = c["Hq"], c["Hkv"]
        wq, wk = (f64(w) for w in c["weights"])
        q, k2, v2 = oracle_write(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], f64(c["cs"]), c["positions"].numpy(),
                                 f64(kc), f64(vc), c["slots"].numpy(), wq, wk, 1e-6, False)
        # Queries and keys are rounded to bf16 before they are multiplied.
        q, k2 = (torch.from_numpy(a).to(BF).double().numpy() for a in (q, k2))
        want, spread, size = oracle_tree(q.reshape(3, 8, Hq, -1), k2, v2, table, lens, c["masks"], window or 0, sinks,
                                         1 / math.sqrt(128))
        # An element of q or k whose float64 value lies within the write's error (about 150 u = 2^-17) of a border
        # of bf16 may round to the other side, a step of 2^-7: about one in 2^9.  Allowed: a sixteenth of a score's
        # size off by a step of each, which doubles in a weight.
        got = f64(outs[layer])
        rel = 2 * (132 * U + 2.0 ** -7 / 8) * size[..., None] + 2.0 ** -15
        assert (np.abs(got - want) <= HALF[BF] * np.abs(want) + rel * spread).all()
        for dev, near in zip(d["caches"][layer], (k2, v2)):
            after = oracle_compact(near, table, lens, c["accepted"].numpy())
            step = np.abs(f64(dev) - after) / np.maximum(np.abs(after), 1e-30)
            assert (step <= 2.0 ** -7).all()
    count = (d["accepted"] >= 0).sum(1).int()
    deepest = c["accepted"].max(1).values.long()
    after = d["lens"] + count
    for layer, (kc, vc) in enumerate(d["caches"]):
        q, _, _ = oracle_write(*(f64(p[layer]) for p in (d["parts"])), f64(c["cs"]), c["positions"].numpy(),
                               f64(kc) * 0, f64(vc) * 0, c["slots"].numpy(), *(f64(w) for w in c["weights"]), 1e-6, False)
        q = torch.from_numpy(q).to(BF).view(3, 8, c["Hq"], -1)[torch.arange(3), deepest].to(gpu)
        if window:
            next_out = attention_amd.gqa_decode_window(q, kc, vc, d["table"], after, window=window, sinks=sinks)
        else:
            next_out = attention_amd.gqa_decode(q, kc, vc, d["table"], after)
        drafted = outs[layer][torch.arange(3), deepest]
        # The same query over the same tokens, moved: equal but for the order of the sums and the border cases.
        assert ((next_out.float() - drafted.float()).abs() <= 2.0 ** -6 * drafted.float().abs() + 2e-2).all()


def test_a_step_captured_and_replayed(gpu):
    """Two captured graphs and eager calls in turn; every replay equals the eager result on the same inputs."""
    say("graph")
    c = step_case(gpu)
    fresh = on_gpu(gpu, c)
    want = [o.clone() for o in run_step(on_gpu(gpu, c))]
    after = on_gpu(gpu, c)
    run_step(after)
    graphs = []
    for _ in range(2):
        d = on_gpu(gpu, c)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run_step(d)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run_step(d)
        graphs.append((g, d, outs))
    for turn in range(4):
        for g, d, outs in graphs:
            for pair, clean in zip(d["caches"], fresh["caches"]):
                for x, y in zip(pair, clean):
                    x.copy_(y)
            torch.cuda.synchronize()
            g.replay()
            eager = run_step(on_gpu(gpu, c))
            torch.cuda.synchronize()
            for o, w, e in zip(outs, want, eager):
                assert torch.equal(o, w) and torch.equal(e, w), f"turn {turn}"
            for pair, done in zip(d["caches"], after["caches"]):
                assert all(torch.equal(x, y) for x, y in zip(pair, done))


def test_tree_decode_captured_with_split_contexts(gpu):
    """Split contexts use a workspace: two graphs of one pool replayed in turn, lengths changed between replays."""
    say("graph, split")
    q, k, v, table, lens, masks = attention_case(BF, 2, 4, 8, 1, 128, 16, [9000, 3000], ragged=False)
    d = [x.to(gpu) for x in (q, k, v, table, lens)]
    m = signed(masks).to(gpu)
    attention_amd.gqa_decode_tree(*d, m)
    torch.cuda.synchronize()
    graphs, pool = [], None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = attention_amd.gqa_decode_tree(*d, m)
        pool = g.pool()
        graphs.append((g, out))
    for n in ([9000, 3000], [10, 0], [5, 8000], [9000, 3000]):
        d[4].copy_(torch.tensor(n, dtype=torch.int32))
        eager = attention_amd.gqa_decode_tree(*d, m)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("T,P,width", [(0, 1 << 20, 2048), (2, 1 << 20, 2048), (1, (1 << 20) - 4, 2049)], ids=str)
def test_contexts_up_to_the_clamp(gpu, T, P, width):
    """Contexts that fill a table of 2^31 tokens and more: the last page's ids are listed, and nothing past the
    table is read.  Keys of all but a few tokens score 2^-184 of those; the few lie in the last page, some of them
    closer to the end than a page list is long."""
    say(f"clamp T{T} P{P}")
    D, capacity = 8, 2 ** 31 - 256
    gen = torch.Generator().manual_seed(3)
    few = [capacity - T - x for x in (1, 2, 17, 64, 300, 1030, 16000, 17000, 100000)]
    assert min(few) >= (width - 1) * P or P % 16
    table = torch.zeros(1, width, dtype=torch.int32)
    last = (capacity - 1) // P
    table[0, last] = 1
    few = [tok for tok in few if tok // P == last]
    assert len(few) > 5
    k = torch.full((2, P, 1, D), -16.0, dtype=BF)
    v = torch.full((2, P, 1, D), 9.0, dtype=BF)
    for tok in few:
        k[1, tok % P] = torch.rand(1, D, generator=gen).to(BF) / 4
        v[1, tok % P] = torch.randn(1, D, generator=gen).to(BF)
    q = torch.ones(*((1, T) if T else (1,)), 1, D, dtype=BF)
    masks = [[(2 << t) - 1 for t in range(T)]] if T else None
    lens = torch.tensor([capacity - T if T else 2 ** 31 - 1], dtype=torch.int32)
    window = 0 if T else 2 ** 31 - 1
    assert cabi.gqa_decode_tree_info(1, max(T, 1), 1, 1, D, P, width, int(T > 0), window, 0,
                                     cabi.DTYPE[BF])[0] == cabi.QD_TREE_MFMA_SPLIT
    got = f64(attend(gpu, (q, k, v, table, lens, masks), window, scale=1.0)).reshape(-1, D)
    at = [tok % P for tok in few]
    w = np.exp(f64(k)[1, at, 0].sum(1))
    w /= w.sum()
    want, spread = w @ f64(v)[1, at, 0], w @ np.abs(f64(v)[1, at, 0])
    # Scores up to 2; about 2^31 weights whose parts are at least 2^-133 add less than 2^-90.
    rel = 2 * (D + 4) * U * 2 + 8 * U + 2 * 64 * U + WEIGHT[BF]
    assert (np.abs(got - want) <= HALF[BF] * np.abs(want) + rel * spread + 2.0 ** -90).all()


@pytest.mark.parametrize("T,Hq", [(0, 2), (8, 8), (32, 8)], ids=lambda x: str(x))
def test_tokens_of_no_weight_do_not_add_up(gpu, T, Hq):
    """fp16: a first token of value 0 takes all of the weight, 2^58 times that of any of 65536 others, whose values
    are 1.  Their parts of a weight are at least 2^-24 (a part is never 0 where the weight is not), scaled by 2^14
    below a reference that the row's largest score exceeds by a factor of 2 at most: each adds up to 2^-38 to the
    output, and the rounding of a subnormal half a step."""
    say(f"no weight T{T} Hq{Hq}")
    B, n, D, P = 1030, 65536, 64, 16                     # more sequences than are split: one workgroup takes all
    gen = torch.Generator().manual_seed(T)
    table = torch.randint(1, 30, (B, n // P + 4), generator=gen, dtype=torch.int32)
    table[0, 0] = 0
    lens = torch.tensor([n] + [i % 20 for i in range(B - 1)], dtype=torch.int32)
    q = torch.ones(*((B, T) if T else (B,)), Hq, D, dtype=HF)
    k = torch.zeros(30, P, 1, D, dtype=HF)
    v = torch.ones(30, P, 1, D, dtype=HF)
    k[0, 0], v[0, 0] = 5.0, 0.0                          # a score of 64 x 5 / 8 = 40, 57.7 bits
    masks = [[(2 << t) - 1 for t in range(T)] for _ in range(B)] if T else None
    assert cabi.gqa_decode_tree_info(B, max(T, 1), Hq, 1, D, P, table.shape[1], int(T > 0), 0 if T else 1 << 20, 0,
                                     cabi.DTYPE[HF])[0] == cabi.QD_TREE_MFMA
    got = f64(attend(gpu, (q, k, v, table, lens, masks), 0 if T else 1 << 20))[0]
    want = (n + T) * math.exp(-40)
    print(f"[case] {got.max():.3g}", flush=True)
    assert (got >= 0).all() and got.max() <= want + (n + T) * 2.0 ** -38 + TINY[HF]
