"""Prompts, and a cache held in 8 bits, operator by operator, as measurable cases.

``prefill``  attention over whole prompts: causal, grouped heads, packed sequences of different lengths
``append``   writes keys and values (prompts or single tokens) to a paged 8-bit cache with a scale per page and head
``gather``   reads such a cache back as packed rows, for the next chunk of a prompt
``decode``   attention of one token per sequence over such a cache

A case is a dict of plain values.  Lengths follow from the case alone (so that its work is known); the seed gives the
order of the sequences, the page order and every tensor.

An 8-bit cache is returned as it is held, with its scales: scales are powers of two, so that every element is
determined, whatever computes it.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
SMALLEST_SCALE = 2.0 ** -100


def _prefill(name, dtype, batch, q_heads, kv_heads, head_dim, lo, hi, *, context=0, window=0, sinks=0):
    """``batch`` prompts of ``lo`` to ``hi`` tokens; ``context``: up to so many keys before each prompt's first."""
    return dict(name=name, op="prefill", dtype=dtype, batch=batch, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, len_lo=lo, len_hi=hi, context=context, window=window, sinks=sinks)


def _cache(name, op, dtype, cache, batch, kv_heads, head_dim, block_size, lo, hi, *, q_heads=0, tokens=0):
    """``lo`` to ``hi`` cached tokens per sequence; append: 1 to ``tokens`` written after them."""
    return dict(name=name, op=op, dtype=dtype, cache=cache, batch=batch, q_heads=q_heads or kv_heads,
                kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, len_lo=lo, len_hi=hi, tokens=tokens)


def listed():
    return [
        # One short prompt, as an interactive request brings it: the call's latency.
        _prefill("prefill-one-short", "bf16", 1, 32, 8, 128, 100, 100),
        # A batch of requests of mixed lengths, packed.
        _prefill("prefill-packed", "bf16", 16, 32, 8, 128, 65, 2000),
        # One long document.
        _prefill("prefill-long", "bf16", 1, 32, 8, 128, 12001, 12001),
        # Chunks of prompts whose earlier tokens are known, in a model with a window: small heads, fp16.
        _prefill("prefill-window-chunks", "fp16", 6, 16, 4, 64, 500, 1500, context=3500, window=1024, sinks=4),
        # A decoding step of a few and of many sequences: one token each.
        _cache("append-tokens-few", "append", "bf16", "e4m3", 8, 8, 128, 16, 50, 1000, tokens=1),
        _cache("append-tokens-many", "append", "fp16", "int8", 512, 4, 128, 32, 20, 700, tokens=1),
        # Prompts into the cache, some of them after tokens that are there already.
        _cache("append-prompts", "append", "bf16", "e4m3", 24, 8, 128, 64, 0, 300, tokens=6000),
        # A few short contexts, and long ones, read back for the next chunk.
        _cache("gather-short", "gather", "fp16", "int8", 4, 8, 64, 16, 100, 700),
        _cache("gather-long", "gather", "bf16", "e4m3", 16, 8, 128, 32, 1000, 9000),
        # Decoding: one sequence, an ordinary batch, a large batch of long contexts.
        _cache("decode-one", "decode", "bf16", "e4m3", 1, 8, 128, 16, 1500, 1500, q_heads=32),
        _cache("decode-batch", "decode", "bf16", "e4m3", 32, 8, 128, 16, 512, 4096, q_heads=32),
        _cache("decode-large", "decode", "fp16", "int8", 48, 8, 128, 64, 2000, 30000, q_heads=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prefill", "append", "gather", "decode"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    block = rng.choice([16, 16, 32, 48, 64, 128])
    if op == "prefill":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        hi = _log(rng, 1, 6000 if dtype != "fp32" else 2000)
        lo = rng.randint(1, hi)
        # At most the longest listed prompt's products.
        most = 128 * 32 * 12000 ** 2 * (0.5 if dtype != "fp32" else 0.02)
        per = head_dim * kv_heads * group * hi * hi
        batch = max(1, min(_log(rng, 1, 64), int(most / per)))
        context = rng.choice([0, 0, rng.randint(0, 3000)])
        window = rng.choice([0, 0, _log(rng, 16, 4000)])
        return {k: v for k, v in _prefill("", dtype, batch, kv_heads * group, kv_heads, head_dim, lo, hi,
                                          context=context if hi <= 4000 else 0, window=window,
                                          sinks=rng.choice([0, 4, 64]) if window else 0).items() if k != "name"}
    dtype, cache = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "int8"])
    row = kv_heads * head_dim
    if op == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, 6000)])
        batch = max(1, min(_log(rng, 1, 512), 24 * 6000 * 1024 // (row * tokens)))
        lo, hi = 0, _log(rng, 1, 800)
    else:
        tokens = 0
        hi = _log(rng, 1, 9000 if op == "gather" else 30000)
        lo = rng.randint(1 if op == "gather" else 0, hi)
        batch = max(1, min(_log(rng, 1, 256), (16 * 5000 if op == "gather" else 40 * 16000) * 1024 // (row * hi)))
    return {k: v for k, v in _cache("", op, dtype, cache, batch, kv_heads, head_dim, block, lo, hi,
                                    q_heads=kv_heads * group, tokens=tokens).items() if k != "name"}


# ----------------------------------------------------------------------------
# What a case's lengths are, and its work
# ----------------------------------------------------------------------------


def _lengths(case):
    """(tokens before, tokens of the call) per sequence."""
    rng = random.Random("-".join(str(case.get(k)) for k in ("op", "batch", "len_lo", "len_hi", "tokens", "context")))
    found = []
    for _ in range(case["batch"]):
        n = rng.randint(case["len_lo"], case["len_hi"])
        if case["op"] == "prefill":
            found.append((rng.randint(0, case["context"]), n))
        else:
            found.append((n, rng.randint(1, case["tokens"]) if case["tokens"] else 0))
    return found


def _seen(before, count, window, sinks):
    """Pairs of a query and a key that it sees."""
    if not window:
        return count * before + count * (count + 1) // 2
    total = 0
    for p in range(before, before + count):
        near = min(p + 1, window)
        total += near + min(sinks, p + 1 - near)
    return total


def work(case):
    lens, hkv, d = _lengths(case), case["kv_heads"], case["head_dim"]
    e = BYTES[case["dtype"]]
    if case["op"] == "prefill":
        queries, keys = sum(n for _, n in lens), sum(c + n for c, n in lens)
        pairs = sum(_seen(c, n, case["window"], case["sinks"]) for c, n in lens)
        return {"bytes": e * d * (2 * queries * case["q_heads"] + 2 * keys * hkv) + 8 * (case["batch"] + 1),
                "flops": 4 * d * case["q_heads"] * pairs}
    page, row = case["block_size"], hkv * d
    if case["op"] == "append":
        written = sum(n for _, n in lens)
        pages = sum((c + n - 1) // page - c // page + 1 for c, n in lens)
        return {"bytes": 2 * written * row * (e + 1) + pages * (8 * hkv + 4) + 8 * case["batch"],
                "flops": 4 * written * row}
    read, pages = sum(c for c, _ in lens), sum(-(-c // page) for c, _ in lens)
    meta = pages * (8 * hkv + 4) + 8 * case["batch"]
    if case["op"] == "gather":
        return {"bytes": 2 * read * row * (e + 1) + meta, "flops": 2 * read * row}
    return {"bytes": 2 * read * row + 2 * case["batch"] * case["q_heads"] * d * e + meta,
            "flops": 4 * read * case["q_heads"] * d}


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _starts(counts):
    total = [0]
    for n in counts:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, hq, hkv, d = DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    before, count = [c for c, _ in lens], [n for _, n in lens]
    state = {"op": case["op"]}
    if case["op"] == "prefill":
        queries, keys = sum(count), sum(before) + sum(count)
        if case["context"]:
            state["q"] = _randn(gen, queries, hq, d, dtype=dtype)
            state["key"], state["value"] = (_randn(gen, keys, hkv, d, dtype=dtype) for _ in range(2))
        else:  # queries, keys and values as one projection leaves them
            qkv = _randn(gen, queries, hq + 2 * hkv, d, dtype=dtype)
            state["q"], state["key"], state["value"] = qkv.split([hq, hkv, hkv], dim=1)
        state["cu"] = _starts(count)
        state["cu_k"] = _starts([c + n for c, n in lens]) if case["context"] else None
        state["most_q"], state["most_k"] = max(count), max(c + n for c, n in lens)
        state["window"], state["sinks"] = case["window"], case["sinks"]
        return state
    kind, page = CACHES[case["cache"]], case["block_size"]
    used = [-(-(c + n) // page) for c, n in lens]
    width, pages = max(1, max(used)), max(1, sum(used))
    live = torch.arange(width, device="cuda")[None, :] < torch.tensor(used, device="cuda")[:, None]
    place = live.reshape(-1).long().cumsum(0).sub_(1).clamp_(min=0).view_as(live)
    order = torch.randperm(pages, generator=gen, device="cuda")
    state["table"] = torch.where(live, order[place], -1).to(torch.int32).contiguous()
    state["lens"] = torch.tensor(before, dtype=torch.int32, device="cuda")
    state["kind"] = case["cache"]
    # Elements as a write leaves them: the largest of a page and head near the top of the range.
    for x in "kv":
        held = _randn(gen, pages, page, hkv, d, dtype=torch.bfloat16)
        if case["cache"] == "e4m3":
            state[x] = held.mul_(100.0).clamp_(-448, 448).to(kind)
        else:
            state[x] = held.mul_(30.0).round_().clamp_(-127, 127).to(kind)
        low = -8 if case["cache"] == "e4m3" else -6
        state[x + "_scales"] = torch.exp2(torch.randint(low, low + 3, (pages, hkv), generator=gen, device="cuda").float())
    if case["op"] == "append":
        total = sum(count)
        kv = _randn(gen, total, 2 * hkv, d, dtype=dtype)
        state["key"], state["value"] = kv.split([hkv, hkv], dim=1)
        state["cu"] = None if case["tokens"] == 1 else _starts(count)
    elif case["op"] == "gather":
        total = sum(before)
        state["cu"] = _starts(before)
        state["key"], state["value"] = (torch.zeros(total, hkv, d, device="cuda", dtype=dtype) for _ in range(2))
    else:
        state["q"] = _randn(gen, case["batch"], hq, d, dtype=dtype)
        state["most_k"] = max(1, max(before))
    return state


# ----------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------


def _softmax_product(score, sees, v):
    score = torch.where(sees, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(most > -math.inf, most, 0))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight / torch.where(total > 0, total, 1), v)


def _plain_prefill(s):
    """Packed sequences padded to the longest."""
    q, hkv = s["q"], s["key"].shape[1]
    tokens, hq, d = q.shape
    cu, cu_k = s["cu"].long(), (s["cu"] if s["cu_k"] is None else s["cu_k"]).long()
    nq, nk = cu.diff()[:, None], cu_k.diff()[:, None]
    i, j = torch.arange(s["most_q"], device=q.device)[None, :], torch.arange(s["most_k"], device=q.device)[None, :]
    there, key_there = i < nq, j < nk
    at = torch.where(there, cu[:-1, None] + i, 0)
    key_at = torch.where(key_there, cu_k[:-1, None] + j, 0)
    b, t, n = at.shape[0], at.shape[1], key_at.shape[1]
    x = q.float()[at].view(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    k = s["key"].float()[key_at].permute(0, 2, 3, 1).contiguous()
    v = s["value"].float()[key_at].transpose(1, 2).contiguous()
    place = (nk - nq + i)[:, :, None]
    sees = (j[:, None, :] <= place) & key_there[:, None, :]
    if s["window"]:
        sees = sees & ((j[:, None, :] > place - s["window"]) | (j[:, None, :] < s["sinks"]))
    score = (torch.matmul(x, k) * (1 / math.sqrt(d))).view(b, hkv, hq // hkv, t, n)
    out = _softmax_product(score, sees[:, None, None], v[:, :, None])
    out = out.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    return out[there].to(q.dtype)


def _power_scale(most, kind):
    """The smallest power of two that keeps ``most`` within the type."""
    part, power = torch.frexp(most)
    top, bits = (0.875, 9) if kind == "e4m3" else (127 / 128, 7)
    scale = torch.ldexp(torch.ones_like(most), torch.where(part > top, power + 1, power) - bits)
    return torch.where(most > 0, scale, SMALLEST_SCALE).clamp(min=SMALLEST_SCALE)


def _held(x, kind):
    return x.to(CACHES[kind]) if kind == "e4m3" else x.round().to(CACHES[kind])


def _plain_append(s):
    kind, table, page = s["kind"], s["table"].long(), s["k"].shape[1]
    first, tokens = s["lens"].long(), s["key"].shape[0]
    if s["cu"] is None:
        owner, nth = torch.arange(tokens, device=table.device), torch.zeros(tokens, device=table.device, dtype=torch.long)
    else:
        nth = torch.arange(tokens, device=table.device)
        owner = torch.searchsorted(s["cu"].long(), nth, right=True) - 1
        nth = nth - s["cu"].long()[owner]
    at = first[owner] + nth
    pages = table[owner, at // page]
    # The page that each sequence goes on with, if it has begun it.
    begun, slot = first % page, torch.arange(page, device=table.device)
    last = torch.gather(table, 1, (first // page)[:, None])[:, 0].clamp(min=0)
    for x, new in (("k", s["key"].float()), ("v", s["value"].float())):
        scales = s[x + "_scales"]
        most = torch.zeros_like(scales).index_reduce_(0, pages, new.abs().amax(-1), "amax")
        touched = torch.zeros(scales.shape[0], device=scales.device, dtype=torch.bool).index_fill_(0, pages, True)
        fresh = _power_scale(most, kind)
        old = scales[last]
        grown = torch.where((begun > 0)[:, None], torch.maximum(old, fresh[last]), fresh[last])
        kept = s[x].view(torch.uint8)[last].view(CACHES[kind]).float() * (old / grown)[:, None, :, None]
        scales.copy_(torch.where(touched[:, None], fresh, scales))
        scales[last] = grown
        rows = (slot[None, :] < begun[:, None]) & (old != grown).any(-1)[:, None]
        where, row = rows.nonzero(as_tuple=True)
        flat = s[x].view(torch.uint8).view(-1, *s[x].shape[2:])
        flat[last[where] * page + row] = _held(kept[where, row], kind).view(torch.uint8)
        flat[pages * page + at % page] = _held(new / scales[pages][:, :, None], kind).view(torch.uint8)


def _plain_rows(s, x, owner, at):
    """Values of tokens ``at`` of sequences ``owner`` in 32 bits."""
    page = s[x].shape[1]
    pages = s["table"].long()[owner, at // page].clamp(min=0)
    held = s[x].view(torch.uint8).view(-1, *s[x].shape[2:])[pages * page + at % page].view(CACHES[s["kind"]])
    return held.float() * s[x + "_scales"][pages][..., None]


def _plain_gather(s):
    tokens = s["key"].shape[0]
    nth = torch.arange(tokens, device=s["cu"].device)
    owner = torch.searchsorted(s["cu"].long(), nth, right=True) - 1
    at = nth - s["cu"].long()[owner]
    s["key"].copy_(_plain_rows(s, "k", owner, at))
    s["value"].copy_(_plain_rows(s, "v", owner, at))


def _plain_decode(s):
    q, hkv = s["q"], s["k"].shape[2]
    b, hq, d = q.shape
    j, owner = torch.arange(s["most_k"], device=q.device)[None, :], torch.arange(b, device=q.device)[:, None]
    sees = j < s["lens"].long()[:, None]
    at = torch.where(sees, j, 0)
    k = _plain_rows(s, "k", owner, at).permute(0, 2, 3, 1).contiguous()
    v = torch.where(sees[..., None, None], _plain_rows(s, "v", owner, at), 0).transpose(1, 2).contiguous()
    score = torch.matmul(q.float().view(b, hkv, hq // hkv, d), k) * (1 / math.sqrt(d))
    return _softmax_product(score, sees[:, None, None], v).reshape(b, hq, d).to(q.dtype)


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------


def run(state):
    s, op = state, state["op"]
    if own:
        import attention_amd
    if op == "prefill":
        if own:
            return attention_amd.gqa_prefill(s["q"], s["key"], s["value"], s["cu"], cu_seqlens_k=s["cu_k"],
                                             window=s["window"] or None, sinks=s["sinks"])
        return _plain_prefill(s)
    if op == "append":
        if own:
            attention_amd.kv_append_q8(s["key"], s["value"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["table"],
                                       s["lens"], s["cu"])
        else:
            _plain_append(s)
        return {"k": s["k"], "v": s["v"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if op == "gather":
        if own:
            attention_amd.kv_gather_q8(s["key"], s["value"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["table"],
                                       s["lens"], s["cu"])
        else:
            _plain_gather(s)
        return {"key": s["key"], "value": s["value"]}
    if own:
        return attention_amd.gqa_decode_q8(s["q"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["table"], s["lens"])
    return _plain_decode(s)


# ----------------------------------------------------------------------------
# The same in 64 bits
# ----------------------------------------------------------------------------


def _exact_heads(q, k, v, sees):
    """q [t, hq, d], k and v [n, hkv, d] in 64 bits; sees [t, n]."""
    t, hq, d = q.shape
    hkv, out = k.shape[1], torch.zeros_like(q)
    for h in range(hq):
        g = h // (hq // hkv)
        score = q[:, h] @ k[:, g].t().contiguous() / math.sqrt(d)
        out[:, h] = torch.softmax(score.masked_fill_(~sees, -math.inf), -1).nan_to_num_(0.0) @ v[:, g].contiguous()
    return out


def _exact_held(x, scale, kind):
    """x / scale on the type's grid, ties to even."""
    y = x / scale
    if kind == "int8":
        return torch.round(y)
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
    step = torch.exp2(torch.clamp(power, min=-6.0) - 3.0)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefill":
        if case["batch"] * case["q_heads"] > 20000:
            return None
        cu, cu_k = s["cu"].tolist(), (s["cu"] if s["cu_k"] is None else s["cu_k"]).tolist()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            q, k, v = s["q"][cu[b]:cu[b + 1]], s["key"][cu_k[b]:cu_k[b + 1]], s["value"][cu_k[b]:cu_k[b + 1]]
            far = torch.arange(len(q), device="cuda")[:, None] + len(k) - len(q) - torch.arange(len(k), device="cuda")
            sees = far >= 0
            if case["window"]:
                sees &= (far < case["window"]) | (torch.arange(len(k), device="cuda") < case["sinks"])
            out[cu[b]:cu[b + 1]] = _exact_heads(q.double(), k.double(), v.double(), sees)
        return out
    table, lens, page = s["table"].tolist(), s["lens"].tolist(), case["block_size"]
    if case["op"] == "append":
        if work(case)["bytes"] > 500 * case["block_size"] * case["kv_heads"] * case["head_dim"] * 100:
            return None
        found = {x: s[x].double() for x in "kv"} | {x + "_scales": s[x + "_scales"].double() for x in "kv"}
        cu = list(range(case["batch"] + 1)) if s["cu"] is None else s["cu"].tolist()
        top = LARGEST[case["cache"]]
        for x, rows in (("k", s["key"].double()), ("v", s["value"].double())):
            for b in range(case["batch"]):
                at, end = lens[b], lens[b] + cu[b + 1] - cu[b]
                while at < end:
                    stop = min(end, (at // page + 1) * page)
                    new = rows[cu[b] + at - lens[b]:cu[b] + stop - lens[b]]
                    p, a, z = table[b][at // page], at % page, at % page + stop - at
                    most = new.abs().amax((0, 2)) / top
                    scale = torch.exp2(torch.ceil(torch.log2(most.clamp(min=SMALLEST_SCALE))))
                    if a:
                        scale = torch.maximum(scale, found[x + "_scales"][p])
                        was = found[x][p, :a] * found[x + "_scales"][p][:, None]
                        found[x][p, :a] = _exact_held(was, scale[:, None], case["cache"])
                    found[x][p, a:z] = _exact_held(new, scale[:, None], case["cache"])
                    found[x + "_scales"][p] = scale
                    at = stop
        return found
    values = {x: s[x].double() * s[x + "_scales"].double()[:, None, :, None] for x in "kv"}
    out = torch.zeros_like(s["q"], dtype=torch.float64) if case["op"] == "decode" else {"key": [], "value": []}
    for b in range(case["batch"]):
        token = torch.arange(lens[b], device="cuda")
        k, v = (values[x][s["table"][b].long()[token // page], token % page] for x in "kv")
        if case["op"] == "gather":
            out["key"].append(k)
            out["value"].append(v)
        elif lens[b]:
            out[b] = _exact_heads(s["q"][b][None].double(), k, v, torch.ones(1, lens[b], dtype=torch.bool, device="cuda"))[0]
    return {x: torch.cat(y) for x, y in out.items()} if case["op"] == "gather" else out
