"""One decoding step with drafted tokens on a paged cache, operator by operator, as measurable cases.

``write``    norms and rotates queries and keys per head and writes keys and values to the cache
``window``   decode attention over the last tokens and a few first ones
``tree``     attention of a tree of drafted tokens over the cache
``compact``  moves the accepted drafted tokens' cache rows next to the context, in every layer's caches

A case is a dict of plain values.  Lengths and trees follow from the case alone (so that its work is known); the
seed gives the order of the sequences, the page order and every tensor.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
POSITIONS = 32768  # rows of the rotation table


def _write(name, dtype, batch, tokens, q_heads, kv_heads, head_dim, block_size, *, rotary=0, interleaved=False,
           norm=True):
    """``batch`` sequences of up to ``tokens`` tokens each; ``rotary`` 0: the whole head."""
    return dict(name=name, op="write", dtype=dtype, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, block_size=block_size, rotary=rotary or head_dim, interleaved=interleaved, norm=norm)


def _window(name, dtype, batch, q_heads, kv_heads, head_dim, block_size, lo, hi, window, sinks, *, k_scale=1.0):
    return dict(name=name, op="window", dtype=dtype, batch=batch, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, block_size=block_size, len_lo=lo, len_hi=hi, window=window, sinks=sinks,
                k_scale=k_scale)


def _tree(name, dtype, batch, tokens, q_heads, kv_heads, head_dim, block_size, lo, hi, *, branch=3, window=0, sinks=0,
          k_scale=1.0):
    """``branch`` 1: a chain of drafted tokens; else each one's parent is one of the ``branch`` before it."""
    return dict(name=name, op="tree", dtype=dtype, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, block_size=block_size, len_lo=lo, len_hi=hi, branch=branch, window=window,
                sinks=sinks, k_scale=k_scale)


def _compact(name, dtype, layers, batch, tokens, kv_heads, head_dim, block_size, lo, hi, *, branch=3):
    return dict(name=name, op="compact", dtype=dtype, layers=layers, batch=batch, tokens=tokens, kv_heads=kv_heads,
                head_dim=head_dim, block_size=block_size, len_lo=lo, len_hi=hi, branch=branch)


def listed():
    return [
        # The next token of a few sequences on a small model: launches and latency.
        _write("write-small", "fp16", 4, 1, 8, 2, 64, 16),
        # The drafted tokens of a mid-size batch.
        _write("write-draft", "bf16", 32, 16, 32, 8, 128, 16),
        # Prompts: the largest calls.
        _write("write-prompt", "bf16", 8, 2048, 32, 8, 128, 16),
        # A few short contexts on a small model.
        _window("window-small", "fp16", 4, 8, 2, 64, 16, 17, 512, 128, 4),
        # Chat contexts, of which each layer keeps about a thousand tokens.
        _window("window-serve", "bf16", 64, 32, 8, 128, 16, 512, 8192, 1024, 4),
        # Long documents with a wide window.
        _window("window-long", "bf16", 16, 64, 8, 128, 16, 32768, 131072, 32768, 64, k_scale=3.0),
        # A short chain of drafts, every head its own keys, a head_dim and pages that are no power of two.
        _tree("tree-chain", "fp16", 5, 7, 32, 32, 80, 12, 33, 700, branch=1),
        # Trees of 16 over chat contexts: the ordinary call.
        _tree("tree-serve", "bf16", 32, 16, 32, 8, 128, 16, 512, 4096),
        # The widest trees over long contexts: as much arithmetic as bandwidth.
        _tree("tree-wide", "bf16", 8, 64, 64, 8, 128, 64, 4096, 16384, branch=8, k_scale=2.0),
        # fp32 caches: numerics work and evaluation.
        _tree("tree-fp32", "fp32", 8, 8, 32, 8, 128, 16, 64, 1024),
        # One layer's caches.
        _compact("compact-small", "fp16", 1, 4, 8, 2, 64, 16, 17, 512),
        # Every layer of a model after its batch was verified.
        _compact("compact-step", "bf16", 36, 32, 16, 8, 128, 16, 16, 256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "window", "window", "tree", "tree", "tree", "compact"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    head_dim = rng.choice([64, 128, 128, 128, 256, 96, 80, 72, 112, 160, 192])
    block_size = rng.choice([16, 16, 16, 32, 64, 128, 8, 1, 12])
    kv_heads, group = rng.choice([(8, 4), (8, 4), (8, 5), (8, 8), (4, 7), (4, 8), (2, 4), (1, 8), (1, 32), (32, 1),
                                  (12, 1), (16, 2), (3, 3)])
    e = BYTES[dtype]
    if op == "write":
        tokens = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 64, 2048)])
        row = (group + 2) * kv_heads * head_dim * e
        batch = _log_int(rng, 1, max(1, min(512, 200_000_000 // (row * tokens))))
        rotary = rng.choice([head_dim, head_dim, head_dim, head_dim // 2])
        case = _write("", dtype, batch, tokens, group * kv_heads, kv_heads, head_dim, block_size, rotary=rotary,
                      interleaved=rng.choice([False, False, True]), norm=rng.choice([True, True, False]))
    elif op == "compact":
        tokens = _log_int(rng, 2, 64)
        layers = _log_int(rng, 1, 48)
        batch = _log_int(rng, 1, 48)
        row = kv_heads * head_dim * e
        hi = max(8, min(512, 6_000_000_000 // (2 * layers * batch * row) - tokens))
        batch = max(1, min(batch, 6_000_000_000 // (2 * layers * (hi + tokens) * row)))
        case = _compact("", dtype, layers, batch, tokens, kv_heads, head_dim, block_size, max(1, hi // 8), hi,
                        branch=rng.choice([2, 3, 6]))
    else:
        tokens = 1 if op == "window" else rng.choice([1, 2, 4, 7, 8, 16, 24, 33, 64])
        hi = _log_int(rng, 32, 65536)
        lo = rng.choice([1, max(1, hi // 8), max(1, hi // 2), hi])
        window = _log_int(rng, 16, 16384) if op == "window" or rng.random() < 0.3 else 0
        sinks = rng.choice([0, 4, 4, 64]) if window else 0
        # The pairs and bytes of the largest listed cases, several times less where a kernel of fp32 or of
        # padded heads takes longer per byte.
        tuned = head_dim in (64, 128) and dtype != "fp32"
        per_token = max(2 * kv_heads * head_dim * e, 4 * kv_heads * group * tokens * head_dim / 200)
        room = (400_000_000 if tuned else 100_000_000) / per_token
        seen = min(hi, window + sinks) if window else hi
        if seen > room:
            hi = lo = seen = max(1, int(room))
        batch = _log_int(rng, 1, max(1, min(256, int(room / seen), 2_000_000 // hi)))
        shape = (dtype, batch, group * kv_heads, kv_heads, head_dim, block_size, lo, hi)
        k_scale = rng.choice([1.0, 2.0, 3.0])
        if op == "window":
            case = _window("", *shape, window, sinks, k_scale=k_scale)
        else:
            case = _tree("", *shape[:2], tokens, *shape[2:], branch=rng.choice([1, 2, 3, 8]), window=window, sinks=sinks,
                         k_scale=k_scale)
    del case["name"]
    return case


# ----------------------------------------------------------------------------
# What follows from the case alone
# ----------------------------------------------------------------------------


def _rng(case):
    return random.Random("-".join(str(case.get(k)) for k in ("op", "batch", "tokens", "len_lo", "len_hi")))


def _lengths(case):
    rng = _rng(case)
    return [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def _trees(case):
    """Per sequence: the visible drafted tokens of each drafted token as bits (its ancestors and itself; 0 past the
    sequence's last drafted token), and the path of the deepest one, first to last."""
    rng, found = _rng(case), []
    for _ in range(case["batch"]):
        count = rng.randint((case["tokens"] + 1) // 2, case["tokens"])
        masks, paths = [], []
        for j in range(count):
            parent = j - rng.randint(1, case["branch"])
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << j)
            paths.append((paths[parent] if parent >= 0 else []) + [j])
        found.append((masks + [0] * (case["tokens"] - count), max(paths, key=len)))
    return found


def _spans(case, lens):
    """(sinks, first token of the rest, tokens seen by any query) per sequence, drafted ones included."""
    drafts = case["tokens"] if case["op"] == "tree" else 0
    spans = []
    for n in lens:
        first = max(0, n - case["window"] + (1 if drafts else 0)) if case["window"] else 0
        sinks = min(case["sinks"], first)
        spans.append((sinks, first, sinks + n + drafts - first))
    return spans


def work(case):
    e, b = BYTES[case["dtype"]], case["batch"]
    if case["op"] == "write":
        n = b * case["tokens"]
        row = (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * row * e + n * (4 * case["rotary"] + 16), "flops": 7 * n * row}
    if case["op"] == "compact":
        moved = sum(sum(i != j for i, j in enumerate(path)) for _, path in _trees(case))
        row = case["kv_heads"] * case["head_dim"] * e
        return {"bytes": 2 * moved * row * 2 * case["layers"] + 4 * b * (case["tokens"] + 2), "flops": 0}
    lens, page = _lengths(case), case["block_size"]
    spans = _spans(case, lens)
    row, heads = case["kv_heads"] * case["head_dim"] * e, case["q_heads"] * case["head_dim"]
    read = sum(n for _, _, n in spans)
    meta = 4 * b + 4 * sum(-(-n // page) for _, _, n in spans)
    if case["op"] == "window":
        return {"bytes": 2 * read * row + 2 * b * heads * e + meta, "flops": 4 * heads * read}
    pairs = sum(n - case["tokens"] + bin(m).count("1") for (_, _, n), (masks, _) in zip(spans, _trees(case))
                for m in masks if m)
    rows = b * case["tokens"]
    return {"bytes": 2 * read * row + 2 * rows * heads * e + 8 * rows + meta, "flops": 4 * heads * pairs}


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------


def _randn(gen, *shape, dtype, scale=1.0):
    x = torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _paged(gen, used, kept, width):
    """Block table [batch, width] of pages scattered over a pool of exactly the kept ones: ``used`` pages per
    sequence, of which the [a, b) of ``kept`` were freed again (-1)."""
    used = torch.tensor(used, device="cuda")[:, None]
    gone = torch.tensor(kept, device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    live = (col < used) & ~((col >= gone[:, :1]) & (col < gone[:, 1:]))
    total = int(live.sum())
    order = torch.randperm(total, generator=gen, device="cuda")
    place = live.reshape(-1).long().cumsum(0).sub_(1).clamp_(min=0).view_as(live)
    return torch.where(live, order[place], -1).to(torch.int32).contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, page = DTYPES[case["dtype"]], case["batch"], case["block_size"]
    hkv, d = case["kv_heads"], case["head_dim"]
    state = {"op": case["op"]}
    if case["op"] == "write":
        t, hq, rot = case["tokens"], case["q_heads"], case["rotary"]
        # Queries, keys and values as one projection leaves them.
        qkv = _randn(gen, b * t, hq + 2 * hkv, d, dtype=dtype)
        state["q"], state["key"], state["value"] = qkv.split([hq, hkv, hkv], dim=1)
        state["q_weight"] = (1 + 0.2 * _randn(gen, d, dtype=torch.float32)).to(dtype) if case["norm"] else None
        state["k_weight"] = (1 + 0.2 * _randn(gen, d, dtype=torch.float32)).to(dtype) if case["norm"] else None
        inverse = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] * inverse
        state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        first = torch.randint(0, POSITIONS - t + 1, (b,), generator=gen, device="cuda")
        at = first[:, None] + torch.arange(t, device="cuda")
        width = -(-t // page) + 1
        table = torch.randperm(b * width, generator=gen, device="cuda").view(b, width)
        place = (first % page)[:, None] + torch.arange(t, device="cuda")
        state["positions"] = at.reshape(-1).to(torch.int32).contiguous()
        state["slots"] = (torch.gather(table, 1, place // page) * page + place % page).reshape(-1).contiguous()
        state["k"] = _randn(gen, b * width, page, hkv, d, dtype=dtype)
        state["v"] = _randn(gen, b * width, page, hkv, d, dtype=dtype)
        state["interleaved"] = case["interleaved"]
        return state
    lens = _lengths(case)
    trees = _trees(case) if case["op"] != "window" else None
    order = list(range(b))
    random.Random(seed).shuffle(order)
    lens = [lens[i] for i in order]
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    drafts = case.get("tokens", 0)
    used = [-(-(n + drafts) // page) for n in lens]
    if case["op"] == "compact":
        state["table"], pages = _paged(gen, used, [(0, 0)] * b, max(used))
        # The caches of all layers, keys then values of each, in one allocation.
        state["pool"] = _randn(gen, 2 * case["layers"], pages, page, hkv, d, dtype=dtype)
        state["caches"] = list(state["pool"].unbind(0))
        paths = [trees[i][1] for i in order]
        state["accepted"] = torch.tensor([p + [-1] * (drafts - len(p)) for p in paths], dtype=torch.int32,
                                         device="cuda")
        return state
    # Pages whose tokens left the window were freed.
    spans = _spans(case, lens)
    state["table"], pages = _paged(gen, used, [(-(-s // page), f // page) if s < f else (0, 0) for s, f, _ in spans],
                                   max(used))
    state["spans"] = max(n for _, _, n in spans)
    state["window"], state["sinks"] = case["window"], case["sinks"]
    rows = (b, drafts) if drafts else (b,)
    state["q"] = _randn(gen, *rows, case["q_heads"], d, dtype=dtype)
    state["k"] = _randn(gen, pages, page, hkv, d, dtype=dtype, scale=case["k_scale"])
    state["v"] = _randn(gen, pages, page, hkv, d, dtype=dtype)
    if drafts:
        masks = [[m - (1 << 64) if m >> 63 else m for m in trees[i][0]] for i in order]
        state["mask"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
    return state


# ----------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------


def _plain_norm_rotate(x, weight, cos, sin, interleaved):
    """x [N, H, D] in 32 bits; cos, sin [N, 1, R/2]."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_write(s):
    rotation = s["cos_sin"][s["positions"].long()][:, None, :]
    cos, sin = rotation.chunk(2, -1)
    q = _plain_norm_rotate(s["q"].float(), s["q_weight"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    key = _plain_norm_rotate(s["key"].float(), s["k_weight"], cos, sin, s["interleaved"]).to(s["key"].dtype)
    s["k"].view(-1, *s["k"].shape[2:])[s["slots"]] = key
    s["v"].view(-1, *s["v"].shape[2:])[s["slots"]] = s["value"]
    return q


def _plain_attention(s):
    """Window and tree decode over the tokens that any query of a sequence sees, gathered and padded to the longest."""
    q = s["q"] if "mask" in s else s["q"][:, None]
    b, t, hq, d = q.shape
    page, hkv = s["k"].shape[1], s["k"].shape[2]
    drafts = t if "mask" in s else 0
    lens, far = s["lens"].long()[:, None], 1 << 40
    window = s["window"] or far
    first = (lens - window + (1 if drafts else 0)).clamp(min=0)
    sinks = first.clamp(max=s["sinks"])
    at = torch.arange(s["spans"], device=q.device)[None, :]
    token = torch.where(at < sinks, at, at - sinks + first)
    there = token < lens + drafts
    token = torch.where(there, token, 0)
    row = torch.gather(s["table"].long(), 1, token // page) * page + token % page
    row = row.clamp(min=0)
    k = s["k"].view(-1, hkv, d)[row].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"].view(-1, hkv, d)[row].float()
    v = torch.where(there[..., None, None], v, 0).transpose(1, 2).contiguous()
    if drafts:
        bits = (s["mask"][:, :, None] >> torch.arange(t, device=q.device)) & 1
        depth = bits.sum(-1) - 1
        draft = (token - lens).clamp(min=0, max=t - 1)
        is_draft = token >= lens
        place = torch.where(is_draft, lens + torch.gather(depth, 1, draft), token)
        asked = torch.gather(bits, 2, draft[:, None, :].expand(b, t, -1)) != 0
        mine = lens + depth
        sees = there[:, None] & (~is_draft[:, None] | asked) & (depth >= 0)[..., None]
        sees = sees & ((place[:, None] > mine[..., None] - window) | (place < s["sinks"])[:, None])
    else:
        sees = there[:, None]
    group = hq // hkv
    q = q.float().view(b, t, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, d)
    score = torch.matmul(q, k).view(b, hkv, t, group, -1) * (1 / math.sqrt(d))
    score = torch.where(sees[:, None, :, None], score, -math.inf)
    most = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(most > -math.inf, most, 0))
    total = weight.sum(-1, keepdim=True)
    weight = (weight / torch.where(total > 0, total, 1)).view(b, hkv, t * group, -1)
    out = torch.matmul(weight, v).view(b, hkv, t, group, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)
    return out.to(s["q"].dtype).view_as(s["q"])


def _plain_compact(s):
    pool, page, count = s["pool"], s["pool"].shape[2], s["accepted"].shape[1]
    rows = pool.view(pool.shape[0], -1, *pool.shape[3:])
    lens, to = s["lens"].long()[:, None], torch.arange(count, device=pool.device)[None, :]
    come = torch.where(s["accepted"] >= 0, s["accepted"].long(), to)
    table = s["table"].long()
    put = torch.gather(table, 1, (lens + to) // page) * page + (lens + to) % page
    take = torch.gather(table, 1, (lens + come) // page) * page + (lens + come) % page
    rows[:, put] = rows[:, take]


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------


def run(state):
    s, op = state, state["op"]
    if own:
        import attention_amd
    if op == "write":
        if own:
            q = attention_amd.qk_norm_rope_write(s["q"], s["key"], s["value"], s["cos_sin"], s["positions"], s["k"],
                                                 s["v"], s["slots"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                                 eps=EPS, interleaved=s["interleaved"])
        else:
            q = _plain_write(s)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "compact":
        if own:
            attention_amd.kv_compact(s["caches"], s["table"], s["lens"], s["accepted"])
        else:
            _plain_compact(s)
        return s["pool"]
    if not own:
        return _plain_attention(s)
    if op == "window":
        return attention_amd.gqa_decode_window(s["q"], s["k"], s["v"], s["table"], s["lens"], window=s["window"],
                                               sinks=s["sinks"])
    return attention_amd.gqa_decode_tree(s["q"], s["k"], s["v"], s["table"], s["lens"], s["mask"],
                                         window=s["window"] or None, sinks=s["sinks"])


# ----------------------------------------------------------------------------
# The same in 64 bits
# ----------------------------------------------------------------------------


def _exact_heads(x, weight, rotation, rotary, interleaved):
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * weight.double()
    z = y.clone()
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        c, s = rotation[:, None, i].double(), rotation[:, None, rotary // 2 + i].double()
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., a] * s + y[..., b] * c
    return z


def exact(case, seed):
    if case["op"] == "compact":
        return None  # rows are copied, no value is computed
    s = prepare(case, seed)
    if case["op"] == "write":
        rotation = s["cos_sin"].index_select(0, s["positions"])
        hkv, d = case["kv_heads"], case["head_dim"]
        k = s["k"].double().view(-1, hkv, d)
        k.index_copy_(0, s["slots"], _exact_heads(s["key"], s["k_weight"], rotation, case["rotary"], case["interleaved"]))
        return {"q": _exact_heads(s["q"], s["q_weight"], rotation, case["rotary"], case["interleaved"]),
                "k": k.view(s["k"].shape), "v": None}
    lens, table, page = s["lens"].tolist(), s["table"].long(), case["block_size"]
    hkv, d, group = case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    masks = s["mask"].tolist() if "mask" in s else [[0]] * case["batch"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rows = out if "mask" in s else out[:, None]
    asks = s["q"] if "mask" in s else s["q"][:, None]
    for i, n in enumerate(lens):
        count = len(masks[i]) if "mask" in s else 0
        # Absolute positions of context and drafted tokens, and which of them each query sees.
        deep = [bin(m % (1 << 64)).count("1") - 1 for m in masks[i]]
        place = torch.tensor(list(range(n)) + [n + deep[j] for j in range(count)], device="cuda")
        mine = torch.tensor([n + x for x in deep] if count else [n - 1], device="cuda")[:, None]
        near = (place > mine - case["window"]) | (place < case["sinks"]) if case["window"] else mine == mine
        asked = [[bool(m) and (j < n or bool(m >> j - n & 1)) for j in range(n - 1, n + count)] for m in masks[i]]
        asked = torch.tensor(asked, device="cuda") if count else mine == mine
        sees = near & torch.cat([asked[:, :1].expand(-1, n), asked[:, 1:]], 1)
        any_ = sees.any(0).nonzero()[:, 0]
        if not len(any_):
            continue
        sees = sees[:, any_]
        ids = table[i, any_ // page] * page + any_ % page
        k, v = (s[x].view(-1, hkv, d)[ids].double() for x in "kv")
        for h in range(hkv):
            q = asks[i].view(-1, hkv, group, d)[:, h].double().reshape(-1, d)
            score = (q @ k[:, h].t().contiguous() / math.sqrt(d)).masked_fill(~sees.repeat_interleave(group, 0), -math.inf)
            weight = torch.softmax(score, -1).nan_to_num(0.0)
            rows[i].view(-1, hkv, group, d)[:, h] = (weight @ v[:, h].contiguous()).view(-1, group, d)
    return out
