"""The serving operators on device buffers: their inputs, plain forms and calls.

Five operators of one decode step of a model with 4-bit weights, 8-bit
activations and an 8-bit paged key/value cache:

* tables:    block tables, slots and positions built on the GPU from request lengths;
* append:    new keys and values into the paged cache, one scale for each page and head;
* attention: queries over that cache, grouped heads, causal, with an optional window;
* norm:      residual addition and root-mean-square norm with an 8-bit output and scales;
* w4:        products of a 4-bit matrix with group scales and 8-bit vectors.

`own` false: the operators as elementary torch operations in 32 bits.
`own` true: the calls of the library (rkcuda).
"""
import math
import os
import random
import sys

import torch

own = False

HERE = os.path.dirname(os.path.abspath(__file__))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
K127 = 0.007874015718698502  # float32(1 / 127)
TINY = 2.0 ** -120           # a page or group whose scale is below this is stored as zeros
_lib = {}


def _rk():
    """The library's binding and device 0, opened once as a program does."""
    if not _lib:
        sys.path.insert(0, os.path.join(os.path.dirname(HERE), "rakkan-mesh_b200"))
        import rkcuda
        _lib["rk"], _lib["dev"] = rkcuda, rkcuda.Device(torch.cuda.current_device())
    return _lib["rk"], _lib["dev"]


# ---- cases -------------------------------------------------------------


def listed():
    return [
        # One sequence taking its next token: the call is all latency.
        {"name": "tables 1 request", "op": "tables", "n": 1, "block": 16, "ctx": 100, "new": 1},
        # A scheduler's step that mixes decoding sequences with prompts.
        {"name": "tables 1024 mixed", "op": "tables", "n": 1024, "block": 32, "ctx": 4096, "new": 96},
        # A decode step of 32 sequences: a token each, in pages begun earlier.
        {"name": "append 32 tokens", "op": "append", "seqs": 32, "new": 1, "block": 64, "kv_heads": 8, "head_size": 128, "type": "bf16"},
        # Prompts of 16 sequences at once, ragged.
        {"name": "append prompts", "op": "append", "seqs": 16, "new": 1024, "block": 64, "kv_heads": 8, "head_size": 128, "type": "bf16"},
        # A small model's single-token step in float32 early in its context.
        {"name": "attention 1x100 f32", "op": "attention", "n": 1, "ctx": 100, "ragged": False, "new": 1, "heads": 14, "kv_heads": 2, "head_size": 64, "block": 16, "window": 0, "type": "f32"},
        # Batched decode of 32 sequences of up to 4096 tokens.
        {"name": "attention 32x4096", "op": "attention", "n": 32, "ctx": 4096, "ragged": True, "new": 1, "heads": 32, "kv_heads": 8, "head_size": 128, "block": 64, "window": 0, "type": "bf16"},
        # One sequence with a very long context: few rows, a long axis.
        {"name": "attention 1x131072", "op": "attention", "n": 1, "ctx": 131072, "ragged": False, "new": 1, "heads": 64, "kv_heads": 8, "head_size": 128, "block": 64, "window": 0, "type": "bf16"},
        # Prompts taken in pieces of 64 tokens over earlier context.
        {"name": "attention 8x64 rows", "op": "attention", "n": 8, "ctx": 2048, "ragged": True, "new": 64, "heads": 32, "kv_heads": 8, "head_size": 128, "block": 32, "window": 0, "type": "f16"},
        # One token's norm before a product, float32 stream, the products' group of 32.
        {"name": "norm 1x4096 f32", "op": "norm", "rows": 1, "cols": 4096, "group": 32, "residual": True, "type": "f32"},
        # A prompt's rows, a scale for each 128 values.
        {"name": "norm 4096x5120", "op": "norm", "rows": 4096, "cols": 5120, "group": 128, "residual": True, "type": "bf16"},
        # The widest product of a layer for one token.
        {"name": "w4 28672x4096 x1", "op": "w4", "rows": 28672, "cols": 4096, "group": 128, "x_group": 128, "n": 1, "zeros": True, "scales": "f16", "type": "bf16"},
        # The down projection for 16 sequences, fine groups, float32 out.
        {"name": "w4 4096x14336 x16", "op": "w4", "rows": 4096, "cols": 14336, "group": 32, "x_group": 32, "n": 16, "zeros": False, "scales": "f32", "type": "f32"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "norm", "w4"])
    t = rng.choice(["f32", "f16", "bf16"])
    if op == "tables":
        return {"op": op, "n": _log(rng, 1, 1024), "block": rng.choice([16, 32, 64, 128]), "ctx": _log(rng, 1, 8192), "new": _log(rng, 1, 96)}
    if op == "append":
        new = _log(rng, 1, 1024)
        return {"op": op, "seqs": _log(rng, 1, max(1, min(256, 16384 // new))), "new": new, "block": rng.choice([16, 32, 64, 128]),
                "kv_heads": rng.randint(1, 8), "head_size": rng.choice([32, 48, 64, 80, 96, 128]), "type": t}
    if op == "attention":
        hs, group, kvh = rng.choice([32, 48, 64, 80, 96, 128, 256]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.randint(1, 8)
        new = _log(rng, 1, 64) if rng.random() < 0.5 else 1
        # at most 2^27 cached values a tensor, and the scores of a plain pass below 2^28
        top = min((1 << 27) // (kvh * hs), (1 << 28) // (kvh * group * new))
        n = _log(rng, 1, 64)
        ctx = max(new, _log(rng, 1, max(2, min(65536, top // n))))
        return {"op": op, "n": n, "ctx": ctx, "ragged": rng.random() < 0.7, "new": new, "heads": kvh * group, "kv_heads": kvh, "head_size": hs,
                "block": rng.choice([16, 32, 64, 128]), "window": _log(rng, 16, 4096) if rng.random() < 0.25 else 0, "type": t}
    if op == "norm":
        group = rng.choice([0, 32, 64, 128])
        cols = max(1, group) * _log(rng, 1, 8192 // max(1, group))
        return {"op": op, "rows": _log(rng, 1, min(8192, 20_000_000 // cols)), "cols": cols, "group": group, "residual": rng.random() < 0.8, "type": t}
    group, x_group = rng.choice([32, 64, 128]), rng.choice([32, 64, 128, 0])
    cols = max(group, x_group) * _log(rng, 2, 16384 // max(group, x_group))
    return {"op": "w4", "rows": _log(rng, 16, min(32768, 100_000_000 // cols)), "cols": cols, "group": group, "x_group": x_group, "n": _log(rng, 1, 16),
            "zeros": rng.random() < 0.5, "scales": rng.choice(["f32", "f16", "bf16"]), "type": t}


def _lens(case):
    """The lengths of a case's requests, the same for every seed: (context before, new tokens)."""
    rng = random.Random(case["op"] + str(sorted((k, v) for k, v in case.items() if isinstance(v, int) and k != "name")))
    if case["op"] == "tables":
        # three in four decode; the others bring a prompt, or a piece of one
        return [(rng.randint(0, case["ctx"]), 1 if rng.random() < 0.75 else rng.randint(0, case["new"])) for _ in range(case["n"])]
    if case["op"] == "append":
        return [(rng.randint(0, 2 * case["block"]), 1 if case["new"] == 1 else rng.randint(1, case["new"])) for _ in range(case["seqs"])]
    got = []
    for _ in range(case["n"]):
        new = case["new"]
        if case["ragged"] and new > 1:
            new = rng.randint(1, new)
        whole = rng.randint(max(new, case["ctx"] // 2), case["ctx"]) if case["ragged"] else case["ctx"]
        got.append((whole - new, new))
    return got


# ---- inputs ------------------------------------------------------------


def _ints(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _pages(lens, block, width, total, gen):
    """A table of `width` pages a request, its `pages(len)` first ones from a shuffled pool, -1 behind."""
    need = [-(-a // block) for a in lens]
    perm = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor([0] + need, device="cuda").cumsum(0)[:-1]
    at = torch.arange(width, device="cuda")[None]
    mine = at < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(mine, perm[(first[:, None] + at).clamp(max=total - 1)], table)
    return table, perm[sum(need):].contiguous()


def _cache(s, blocks, block, kv_heads, hs, gen):
    """A cache as earlier appends left it: values of about a normal's spread, scales around its largest / 127."""
    def values(shape):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["k"], s["v"] = values((blocks, kv_heads, block, hs)), values((blocks, kv_heads, hs, block))
    for name, base in (("k_scale", 0.03), ("v_scale", 0.02)):
        s[name] = base * torch.exp(0.3 * torch.randn((blocks, kv_heads), generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "tables":
        lens = _lens(case)
        block = case["block"]
        width = -(-(case["ctx"] + case["new"]) // block) + 1
        total = sum(-(-(a + b) // block) for a, b in lens) + 64
        s["ctx_lens"], s["new_lens"] = _ints([a for a, b in lens]), _ints([b for a, b in lens])
        s["table"], s["free"] = _pages([a for a, b in lens], block, width, total, gen)
        s["head"] = _ints([7])
        s["max_tokens"] = sum(b for a, b in lens) + 5  # a step's buffers are a little larger than its tokens
        if own:
            rk, dev = _rk()
            s["made"] = rk.PageTables(dev, case["n"], width, block, s["max_tokens"], table=s["table"])
    elif op == "append":
        lens = _lens(case)
        block, kvh, hs, t = case["block"], case["kv_heads"], case["head_size"], TYPES[case["type"]]
        tokens = sum(b for a, b in lens)
        width = max(-(-(a + b) // block) for a, b in lens)
        total = sum(-(-(a + b) // block) for a, b in lens) + 3
        table, _ = _pages([a + b for a, b in lens], block, width, total, gen)
        _cache(s, total, block, kvh, hs, gen)
        req = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor([b for a, b in lens])).cuda()
        first = torch.tensor([0] + [b for a, b in lens]).cumsum(0)[:-1].cuda()
        pos = torch.tensor([a for a, b in lens]).cuda()[req] + torch.arange(tokens, device="cuda") - first[req]
        s["slots"] = (table[req, pos // block] * block + pos % block).to(torch.int32)
        # new keys and values as they leave a fused projection: strided rows
        kv = torch.randn((tokens, 2, kvh, hs), generator=gen, device="cuda").to(t)
        s["k_new"], s["v_new"] = kv[:, 0], kv[:, 1]
        if own:
            rk, dev = _rk()
            s["cache"] = rk.PagedKV8(dev, s["k"], s["v"], s["k_scale"], s["v_scale"])
    elif op == "attention":
        lens = _lens(case)
        block, kvh, hs, t = case["block"], case["kv_heads"], case["head_size"], TYPES[case["type"]]
        whole = [a + b for a, b in lens]
        width = -(-max(whole) // block)
        total = sum(-(-a // block) for a in whole) + 3
        s["table"], _ = _pages(whole, block, width, total, gen)
        _cache(s, total, block, kvh, hs, gen)
        s["lens"] = _ints(whole)
        first = [0]
        for a, b in lens:
            first.append(first[-1] + b)
        s["q_start"] = None if case["new"] == 1 else _ints(first)
        s["q"] = (torch.randn((first[-1], case["heads"], hs), generator=gen, device="cuda") * 1.2).to(t)
        if own:
            rk, dev = _rk()
            s["cache"] = rk.PagedKV8(dev, s["k"], s["v"], s["k_scale"], s["v_scale"])
    elif op == "norm":
        t, shape = TYPES[case["type"]], (case["rows"], case["cols"])
        s["x"] = (torch.randn(shape, generator=gen, device="cuda") * 0.5).to(t)
        s["residual"] = (torch.randn(shape, generator=gen, device="cuda") * 3).to(t) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(case["cols"], generator=gen, device="cuda")).to(t)
        if own:
            s["rk"], s["dev"] = _rk()
    else:
        rows, cols, group = case["rows"], case["cols"], case["group"]
        xg = case["x_group"] or cols
        s["w"] = torch.randint(0, 256, (rows, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = (0.004 * torch.exp(0.3 * torch.randn((rows, cols // group), generator=gen, device="cuda"))).to(TYPES[case["scales"]])
        s["zeros"] = torch.randint(4, 12, (rows, cols // group), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["x"] = (torch.randn((case["n"], cols), generator=gen, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)
        s["x_scales"] = 0.02 * torch.exp(0.3 * torch.randn((case["n"], cols // xg), generator=gen, device="cuda"))
        if own:
            rk, dev = _rk()
            s["matrix"] = rk.W4Matrix(dev, s["w"].cpu(), s["scales"].cpu(), None if s["zeros"] is None else s["zeros"].cpu())
    return s


# ---- plain forms -------------------------------------------------------


def _plain_tables(s):
    B, T = s["case"]["block"], s["max_tokens"]
    ctx, new, table, head = s["ctx_lens"].long(), s["new_lens"].long(), s["table"], s["head"].long()
    n, width = table.shape
    ends = new.cumsum(0)
    fits = (ends <= T) & (ctx + new <= width * B)
    old, whole = (ctx + B - 1) // B, (ctx + new + B - 1) // B
    need = torch.where(fits, whole - old, 0)
    cum = need.cumsum(0)
    served = fits & ((need == 0) | (cum <= s["free"].numel() - head))
    q_start = torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=T)
    lens = torch.where(served, ctx + new, 0)
    before = head + cum - need  # the place in the free list of a request's first page
    at = torch.arange(width, device="cuda")[None]
    takes = served[:, None] & (at >= old[:, None]) & (at < whole[:, None])
    page = s["free"][(before[:, None] + at - old[:, None]).clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(takes, page, table))
    t = torch.arange(T, device="cuda")
    req = torch.searchsorted(q_start[1:].contiguous(), t, right=True).clamp(max=n - 1)
    inside = t < q_start[-1]
    pos = torch.where(inside, ctx[req] + t - q_start[req], 0)
    p = table[req, (pos // B).clamp(max=width - 1)].long()
    slots = torch.where(inside & served[req] & (p >= 0), p * B + pos % B, -1)
    taken = torch.where(served, cum, 0).max().reshape(1)
    info = torch.cat([q_start[-1:], taken, (~served).sum().reshape(1), head + taken])
    return {"table": table, "lens": lens.int(), "q_start": q_start.int(), "slots": slots.int(), "positions": pos.int(), "info": info.int()}


def _plain_store(x, slots, cache, scales, transposed):
    """New rows x [T, heads, hs] into int8 pages [blocks, heads, block, hs] under one scale a page and head."""
    pages = cache.transpose(2, 3) if transposed else cache  # a view: [blocks, heads, block, hs]
    blocks, heads, B, hs = pages.shape
    x = x.float()
    page, row = slots.long() // B, slots.long() % B
    peak = torch.zeros((blocks, heads), device="cuda").index_reduce_(0, page, x.abs().amax(2), "amax")
    first = torch.full((blocks,), B, device="cuda").index_reduce_(0, page, row, "amin")  # rows before it hold earlier tokens
    touched = first < B
    had = torch.where((first > 0)[:, None], scales, 0.0)
    scale = torch.maximum(had, peak * K127)
    scale = torch.where(scale < TINY, 0.0, scale)
    ratio = torch.where(scale > 0, had / scale, 0.0)
    again = (pages.float() * ratio[:, :, None, None]).round().to(torch.int8)
    earlier = touched[:, None, None, None] & (torch.arange(B, device="cuda")[None, :] < first[:, None])[:, None, :, None]
    pages.copy_(torch.where(earlier, again, pages))
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    pages[page, :, row] = (x * inverse[page][:, :, None]).round().clamp(-127, 127).to(torch.int8)
    scales.copy_(torch.where(touched[:, None], scale, scales))


def _plain_append(s):
    _plain_store(s["k_new"], s["slots"], s["k"], s["k_scale"], False)
    _plain_store(s["v_new"], s["slots"], s["v"], s["v_scale"], True)
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    case = s["case"]
    kvh, hs, B, new = case["kv_heads"], case["head_size"], case["block"], case["new"]
    G, (n, width), T = case["heads"] // case["kv_heads"], s["table"].shape, s["q"].shape[0]
    L = width * B
    at = s["table"].clamp(min=0).long()
    k = (s["k"][at].float() * s["k_scale"][at][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, kvh, L, hs)
    v = (s["v"][at].float() * s["v_scale"][at][..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, kvh, L, hs)
    first = torch.arange(n + 1, device="cuda") if s["q_start"] is None else s["q_start"].long()
    count = first[1:] - first[:-1]
    row = first[:-1, None] + torch.arange(new, device="cuda")
    q = s["q"].float()[row.clamp(max=T - 1)]  # [n, new, heads, hs]
    q = q.reshape(n, new, kvh, G, hs).permute(0, 2, 3, 1, 4).reshape(n, kvh, G * new, hs)
    score = (q @ k.transpose(2, 3)).reshape(n, kvh, G, new, L) / math.sqrt(hs)
    pos = (s["lens"].long() - count)[:, None] + torch.arange(new, device="cuda")  # [n, new]
    key = torch.arange(L, device="cuda")
    seen = (key <= pos[..., None]) & (key < s["lens"][:, None, None])
    if case["window"]:
        seen = seen & (key > pos[..., None] - case["window"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    o = (p.reshape(n, kvh, G * new, L) @ v).reshape(n, kvh, G, new, hs).permute(0, 3, 1, 2, 4).reshape(n, new, kvh * G, hs)
    t = torch.arange(T, device="cuda")
    req = torch.searchsorted(first[1:].contiguous(), t, right=True)
    return o[req, t - first[req]].to(s["q"].dtype)


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    rows, cols, group = case["rows"], case["cols"], case["group"] or case["cols"]
    h = s["x"].float() + s["residual"].float() if s["residual"] is not None else s["x"].float()
    # The integers do not depend on the row's norm, so they are taken before it: with y = h·w·r the
    # quotient y / (max|y| / 127) is h·w / (max|h·w| / 127).
    u = (h * s["weight"].float()).reshape(rows, cols // group, group)
    base = u.abs().amax(2) * K127
    base = torch.where(base < TINY, 0.0, base)
    inverse = torch.where(base > 0, 1.0 / base, 0.0)
    q = (u * inverse[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(rows, cols)
    r = torch.rsqrt(h.square().mean(1) + EPS)
    got = {"q": q, "scales": base * r[:, None]}
    if s["residual"] is not None:
        got["sum"] = h.to(t)
    return got


def _plain_w4(s):
    case = s["case"]
    rows, cols, group, xg = case["rows"], case["cols"], case["group"], case["x_group"] or case["cols"]
    w = s["w"].reshape(rows, cols // 32, 16)
    w = torch.cat([w & 15, w >> 4], 2).reshape(rows, cols // group, group).float()
    w = (w - (8.0 if s["zeros"] is None else s["zeros"].float()[..., None])) * s["scales"].float()[..., None]
    x = (s["x"].reshape(-1, cols // xg, xg).float() * s["x_scales"][..., None]).reshape(-1, cols)
    return (x @ w.reshape(rows, cols).T).to(TYPES[case["type"]])


# ---- one pass ----------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention, "norm": _plain_norm, "w4": _plain_w4}[op](s)
    case = s["case"]
    if op == "tables":
        t = s["made"]
        t.build(s["ctx_lens"], s["new_lens"], s["free"], s["head"])
        return {"table": t.table, "lens": t.lens, "q_start": t.q_start, "slots": t.slots, "positions": t.positions, "info": t.info}
    if op == "append":
        s["cache"].append(s["k_new"], s["v_new"], s["slots"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "attention":
        return s["cache"].attention(s["q"], s["table"], s["lens"], q_start=s["q_start"], window=case["window"])
    if op == "norm":
        q, scales, total = s["rk"].add_rmsnorm_q8(s["dev"], s["x"], s["weight"], EPS, group=case["group"], residual=s["residual"])
        return {"q": q, "scales": scales} if s["residual"] is None else {"q": q, "scales": scales, "sum": total}
    return s["matrix"].mulvec(s["x"], s["x_scales"], dtype=TYPES[case["type"]])


# ---- what a pass cannot do without -------------------------------------


def work(case):
    op = case["op"]
    if op == "tables":
        lens = _lens(case)
        tokens = sum(b for a, b in lens)
        pages = sum(-(-(a + b) // case["block"]) + (-a // case["block"]) for a, b in lens)
        # lengths in and out, row starts, slots and positions, the pages taken read and written
        return {"bytes": 4 * (4 * len(lens) + 1 + 2 * tokens + 2 * pages), "flops": 4 * tokens}
    if op == "append":
        tokens = sum(b for a, b in _lens(case))
        values = 2 * tokens * case["kv_heads"] * case["head_size"]
        return {"bytes": values * (SIZE[case["type"]] + 1) + 4 * tokens, "flops": 4 * values}
    if op == "attention":
        lens, wide = _lens(case), case["window"]
        cached = rows = pairs = pages = 0
        for a, b in lens:
            first = max(0, a + 1 - wide) if wide else 0
            cached += a + b - first
            pages += -(-(a + b) // case["block"]) - first // case["block"]
            rows += b
            pairs += sum(min(a + j + 1, wide) if wide else a + j + 1 for j in range(b))
        one = case["kv_heads"] * case["head_size"]
        return {"bytes": 2 * cached * one + 8 * pages * case["kv_heads"] + 4 * pages + 2 * rows * case["heads"] * case["head_size"] * SIZE[case["type"]],
                "flops": 4 * pairs * case["heads"] * case["head_size"]}
    if op == "norm":
        values = case["rows"] * case["cols"]
        group = case["group"] or case["cols"]
        return {"bytes": values * (SIZE[case["type"]] * (3 if case["residual"] else 1) + 1) + 4 * values // group + SIZE[case["type"]] * case["cols"],
                "flops": 6 * values}
    rows, cols, n = case["rows"], case["cols"], case["n"]
    groups = rows * (cols // case["group"])
    return {"bytes": rows * cols // 2 + groups * (SIZE[case["scales"]] + (1 if case["zeros"] else 0)) + n * cols + 4 * n * (cols // (case["x_group"] or cols))
            + n * rows * SIZE[case["type"]], "flops": 2 * rows * cols * n}


# ---- the definitions in 64 bits ----------------------------------------


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "tables":
        return None  # whole numbers: compared as they are
    if op == "append":
        return _exact_append(s)
    if op == "attention":
        return _exact_attention(s)
    if op == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        y = x / (x.pow(2).sum(1, keepdim=True) / case["cols"] + EPS).sqrt() * s["weight"].double()
        group = case["group"] or case["cols"]
        got = {"q": None, "scales": torch.stack([c.abs().max(1).values / 127 for c in y.split(group, 1)], 1)}
        return got if s["residual"] is None else {**got, "sum": x}
    out = torch.empty((case["n"], case["rows"]), dtype=torch.float64, device="cuda")
    xs = s["x_scales"].double().repeat_interleave(case["x_group"] or case["cols"], 1) * s["x"].double()
    for r in range(0, case["rows"], 2048):  # a byte's low half is column j of its block of 32, the high half column j + 16
        b = s["w"][r:r + 2048].long().view(-1, case["cols"] // 32, 16)
        q = torch.stack([b % 16, b // 16], 2).view(b.shape[0], case["cols"]).double()
        z = 8 if s["zeros"] is None else s["zeros"][r:r + 2048].double().repeat_interleave(case["group"], 1)
        out[:, r:r + 2048] = xs @ ((q - z) * s["scales"][r:r + 2048].double().repeat_interleave(case["group"], 1)).t()
    return out


def _exact_append(s):
    """The scales of the pages: each new row's largest magnitude against its page's."""
    B, got = s["case"]["block"], {"k": None, "v": None}
    slots = s["slots"].cpu().tolist()
    for name in ("k", "v"):
        peak = (s[name + "_new"].double().abs().max(2).values / 127).cpu()
        scale, begun = s[name + "_scale"].double().cpu(), {}
        for t, slot in enumerate(slots):
            p = slot // B
            if p not in begun:
                begun[p] = True
                if slot % B == 0:
                    scale[p] = 0
            scale[p] = torch.maximum(scale[p], peak[t])
        got[name + "_scale"] = scale
    return got


def _exact_attention(s):
    case = s["case"]
    B, G, hs = case["block"], case["heads"] // case["kv_heads"], case["head_size"]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (before, new) in enumerate(_lens(case)):
        have = before + new
        pages = s["table"][i, :-(-have // B)].long()
        for h in range(case["kv_heads"]):
            k = (s["k"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, hs)[:have]
            v = (s["v"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, hs)[:have]
            for j0 in range(0, new, 16):
                j1 = min(new, j0 + 16)
                q = s["q"][at + j0:at + j1, h * G:(h + 1) * G].double()
                a = torch.einsum("jgd,ld->jgl", q, k) / hs ** 0.5
                where = torch.arange(have, device="cuda")[None] - torch.arange(before + j0, before + j1, device="cuda")[:, None]
                hidden = where > 0
                if case["window"]:
                    hidden = hidden | (where <= -case["window"])
                a = a.masked_fill(hidden[:, None], -math.inf).softmax(-1)
                out[at + j0:at + j1, h * G:(h + 1) * G] = torch.einsum("jgl,ld->jgd", a, v)
        at += new
    return out
