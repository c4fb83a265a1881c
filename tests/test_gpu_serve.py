"""The serving operators on the GPU against their definitions: integers and
scales against a plain restatement value by value, floating outputs against
64 bits within bounds derived from the arithmetic (u below is float32's half
step, 2^-24)."""
import math

import numpy as np
import pytest

import rkcuda as rk

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def dtype(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def ints(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- page tables -------------------------------------------------------


def tables_plain(ctx, new, free, head, table, block, max_tokens):
    """rk_page_tables, a request after the other."""
    n, width = table.shape
    table, avail = table.copy(), len(free) - head if 0 <= head <= len(free) else 0
    lens, start, slots, pos = [], [], [-1] * max_tokens, [0] * max_tokens
    end = cum = taken = refused = 0
    for i in range(n):
        c, m = max(0, ctx[i]), max(0, new[i])
        start.append(min(end, max_tokens))
        fits = end + m <= max_tokens and c + m <= width * block
        need = -(-(c + m) // block) + (-c // block) if fits else 0
        cum += need
        ok = fits and (need == 0 or cum <= avail)
        if ok:
            for j in range(need):
                table[i, -(-c // block) + j] = free[head + cum - need + j]
            taken = max(taken, cum) if need else taken
        refused += not ok
        lens.append(c + m if ok else 0)
        for j in range(max(0, min(m, max_tokens - end))):
            pos[end + j] = min(c + j, 2 ** 31 - 1)
            if ok and table[i, (c + j) // block] >= 0:
                slots[end + j] = table[i, (c + j) // block] * block + (c + j) % block
        end += m
    rows = min(end, max_tokens)
    return table, lens, start + [rows], slots, pos, [rows, taken, refused, head + taken]


def run_tables(torch, dev, ctx, new, free, head, width, block, max_tokens, first_page=1000):
    """Builds once on the GPU and compares everything; existing pages are numbered from first_page."""
    n = len(ctx)
    table = np.full((n, max(width, 0)), -7, np.int32)
    at = first_page
    for i in range(n):
        for j in range(min(width, -(-max(0, ctx[i]) // block))):
            table[i, j] = at
            at += 1
    want = tables_plain(ctx, new, free, head, table, block, max_tokens)
    t = rk.PageTables(dev, n, width, block, max_tokens, table=torch.from_numpy(table.copy()).cuda())
    args = ints(torch, ctx), ints(torch, new), ints(torch, free), None if head == 0 else ints(torch, [head])
    for _ in range(2):  # the same again: nothing is kept between calls
        t.build(*args)
        got = [x.cpu().numpy() for x in (t.table, t.lens, t.q_start, t.slots, t.positions, t.info)]
        for g, w, what in zip(got, want, ("table", "lens", "q_start", "slots", "positions", "info")):
            np.testing.assert_array_equal(g, np.array(w, np.int32).reshape(g.shape), err_msg=what)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 31, 513])
def test_tables_random(torch, dev, n, block):
    rng = np.random.default_rng(n * 1000 + block)
    ctx = rng.integers(0, 5 * block, n).tolist()
    new = [int(rng.choice([0, 1, 1, 1, rng.integers(0, 3 * block)])) for _ in range(n)]
    free = rng.permutation(n * 10)[: n * 5 + 3].tolist()
    run_tables(torch, dev, ctx, new, free, 2, 9, block, sum(new) + 3)


@pytest.mark.parametrize("case", [
    ([16, 32], [1, 1], 1, 4, 8),        # the second finds no page
    ([15, 16, 15], [1, 1, 1], 0, 4, 8), # only the one that needs a page is refused
    ([0, 0, 0], [5, 9, 2], 9, 4, 13),   # the second passes the rows, and the third with it
    ([60, 3], [5, 5], 9, 4, 99),        # the first passes the table's width
    ([60, 3], [4, 5], 9, 4, 9),         # ... and just not
    ([-3, 0], [-2, 0], 3, 4, 4),        # below zero is zero
    ([5, 7], [0, 0], 0, 1, 0),          # no rows at all
    ([2 ** 31 - 1, 1], [2 ** 31 - 1, 2 ** 31 - 1], 3, 4, 6),  # sums past 32 bits
], ids=str)
def test_tables_refuse_requests(torch, dev, case):
    ctx, new, n_free, width, rows = case
    run_tables(torch, dev, ctx, new, list(range(n_free)), 0, width, 16, rows)


@pytest.mark.parametrize("head", [-1, 5, 6])
def test_tables_free_head_outside_the_list(torch, dev, head):
    run_tables(torch, dev, [0, 3], [1, 1], [4, 5, 6, 7, 8], head, 2, 16, 4)


def test_tables_of_no_requests_and_of_the_most(torch, dev):
    run_tables(torch, dev, [], [], [1, 2], 1, 3, 16, 5)
    n = rk.MAX_REQUESTS
    ctx, new = [(7 * i) % 50 for i in range(n)], [i % 3 for i in range(n)]
    run_tables(torch, dev, ctx, new, list(range(n)), 0, 4, 16, sum(new))


# ---- append ------------------------------------------------------------


def q127(x, inv):
    with np.errstate(invalid="ignore", over="ignore"):
        p = (x * inv).astype(np.float32)
    return np.where(np.isnan(p), 0, np.rint(np.clip(np.nan_to_num(p, nan=0.0, posinf=127, neginf=-127), -127, 127))).astype(np.int8)


def append_plain(pages, scales, x, slots, block):
    """rk_kv8_append of one tensor; pages [blocks][heads][block][hs], float32 arithmetic a run at a time."""
    k127, tiny = np.float32(1.0 / 127), np.float32(2.0 ** -120)
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= pages.shape[0] * block:
            t += 1
            continue
        p, first, e = slots[t] // block, slots[t] % block, t
        while e < len(slots) and slots[e] >= 0 and slots[e] // block == p:
            e += 1
        for h in range(pages.shape[1]):
            run = x[t:e, h].astype(np.float32)
            a = np.abs(run)
            m = np.float32(a[np.isfinite(a)].max(initial=0))
            had = scales[p, h] if first else np.float32(0)
            s = max(had, np.float32(m * k127))
            s = np.float32(0) if s < tiny else s
            inv = np.float32(1) / s if s else np.float32(0)
            if had != s:
                pages[p, h, :first] = q127(pages[p, h, :first].astype(np.float32), np.float32(had / s) if s else np.float32(0))
            for j in range(t, e):
                pages[p, h, slots[j] % block] = q127(run[j - t], inv)
            scales[p, h] = s
        t = e


def cache(torch, dev, rng, blocks, heads, block, hs):
    k = rng.integers(-127, 128, (blocks, heads, block, hs)).astype(np.int8)
    v = rng.integers(-127, 128, (blocks, heads, hs, block)).astype(np.int8)
    ks, vs = (np.exp(rng.normal(-3.5, 0.5, (blocks, heads))).astype(np.float32) for _ in range(2))
    return rk.PagedKV8(dev, *(torch.from_numpy(a.copy()).cuda() for a in (k, v, ks, vs))), [k, v, ks, vs]


def check_append(torch, dev, rng, kv, host, x, slots, t="f32"):
    k, v, ks, vs = host
    kn, vn = (torch.from_numpy(a).cuda().to(dtype(torch, t)) for a in x)
    kv.append(kn, vn, ints(torch, slots))
    vt = np.ascontiguousarray(v.transpose(0, 1, 3, 2))
    append_plain(k, ks, kn.float().cpu().numpy(), slots, kv.block)
    append_plain(vt, vs, vn.float().cpu().numpy(), slots, kv.block)
    v[:] = vt.transpose(0, 1, 3, 2)
    for got, want, what in ((kv.k, k, "k"), (kv.v, v, "v"), (kv.k_scale, ks, "k_scale"), (kv.v_scale, vs, "v_scale")):
        np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=what)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block,hs,heads", [(16, 64, 2), (16, 48, 1), (32, 80, 3), (64, 128, 2), (128, 16, 1), (64, 256, 1),
                                            (128, 112, 2)])
def test_append_runs(torch, dev, block, hs, heads, t):
    """Runs of one row to several pages, begun inside a page and at its start."""
    rng = np.random.default_rng(block + hs)
    kv, host = cache(torch, dev, rng, 16, heads, block, hs)
    page, slots = iter(rng.permutation(16)), []
    for first, rows in ((0, 1), (block - 1, 1), (3, block - 3), (5, 2), (0, 2 * block + 1), (block // 2, block)):
        p = next(page)
        for j in range(rows):
            if j and (first + j) % block == 0:
                p = next(page)
            slots.append(int(p) * block + (first + j) % block)
        slots.append(-1)
    n = len(slots)
    x = [rng.normal(0, 1, (n, heads, hs)).astype(np.float32) for _ in range(2)]
    check_append(torch, dev, rng, kv, host, x, slots, t)
    # again, larger by a few steps: every earlier row of a begun page is scaled down
    check_append(torch, dev, rng, kv, host, [9 * a for a in x], slots, t)


def test_append_token_by_token(torch, dev):
    rng = np.random.default_rng(5)
    kv, host = cache(torch, dev, rng, 3, 2, 16, 32)
    for j in range(40):
        x = [(rng.normal(0, 1 + j / 8, (1, 2, 32))).astype(np.float32) for _ in range(2)]
        check_append(torch, dev, rng, kv, host, x, [(2 - j // 16) * 16 + j % 16])


def test_append_special_values(torch, dev):
    """NaN is stored as 0, infinities at the page's end of the range; pages of zeros and of values too small for a scale."""
    rng = np.random.default_rng(6)
    kv, host = cache(torch, dev, rng, 6, 1, 16, 16)
    x = [rng.normal(0, 1, (6, 1, 16)).astype(np.float32) for _ in range(2)]
    for a in x:
        a[0, 0, :3] = np.nan, np.inf, -np.inf
        a[1] = 0
        a[2] = 1e-36
        a[3] = np.inf
        a[4] = np.nan
        a[5, 0, 0] = 3e38
    check_append(torch, dev, rng, kv, host, x, [0, 16, 32, 48 + 5, 64, 80])
    check_append(torch, dev, rng, kv, host, [a[::-1].copy() for a in x], [1, 17, 33, 48 + 6, 65, 81])


def test_append_many_rows_and_strides(torch, dev):
    """Enough rows that a CTA looks through several; keys and values as slices of a fused projection."""
    rng = np.random.default_rng(7)
    heads, hs, block, rows = 8, 32, 64, 64 * 50 + 17
    kv, host = cache(torch, dev, rng, 52, heads, block, hs)
    fused = torch.from_numpy(rng.normal(0, 1, (rows, 5 * heads * hs)).astype(np.float32)).cuda()
    kn = fused[:, 2 * heads * hs:3 * heads * hs].unflatten(1, (heads, hs))
    vn = fused[:, 4 * heads * hs:].unflatten(1, (heads, hs))
    perm = rng.permutation(52)
    slots = [int(perm[(j + 5) // block]) * block + (j + 5) % block for j in range(rows)]
    kv.append(kn, vn, ints(torch, slots))
    k, v, ks, vs = host
    vt = np.ascontiguousarray(v.transpose(0, 1, 3, 2))
    append_plain(k, ks, kn.cpu().numpy(), slots, block)
    append_plain(vt, vs, vn.cpu().numpy(), slots, block)
    np.testing.assert_array_equal(kv.k.cpu().numpy(), k)
    np.testing.assert_array_equal(kv.v.cpu().numpy(), vt.transpose(0, 1, 3, 2))
    np.testing.assert_array_equal(kv.k_scale.cpu().numpy(), ks)
    np.testing.assert_array_equal(kv.v_scale.cpu().numpy(), vs)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_append_slots_with_gaps_and_repeats(torch, dev, t):
    """Runs that skip offsets, and a slot given twice: the later row stays."""
    rng = np.random.default_rng(17)
    kv, host = cache(torch, dev, rng, 4, 2, 32, 48)
    slots = [1, 4, 5, 31, 32 + 7, 32 + 7, 32 + 8, 64, 64, 96 + 3, 96 + 30]
    x = [rng.normal(0, 2, (len(slots), 2, 48)).astype(np.float32) for _ in range(2)]
    check_append(torch, dev, rng, kv, host, x, slots, t)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("first", [0, 1, 2, 3, 13])
def test_append_unaligned_rows(torch, dev, first, t):
    """Keys and values that begin off a 16-byte boundary, runs at every offset of a word of four tokens."""
    rng = np.random.default_rng(18 + first)
    kv, host = cache(torch, dev, rng, 3, 2, 16, 32)
    slots = [(16 * (j // 16) + j % 16) for j in range(first, first + 22)]
    wide = torch.from_numpy(rng.normal(0, 1, (22, 2 * 64 + 3)).astype(np.float32)).cuda().to(dtype(torch, t))
    kn, vn = wide[:, 1:65].unflatten(1, (2, 32)), wide[:, 66:130].unflatten(1, (2, 32))
    kv.append(kn, vn, ints(torch, slots))
    k, v, ks, vs = host
    vt = np.ascontiguousarray(v.transpose(0, 1, 3, 2))
    append_plain(k, ks, kn.float().cpu().numpy(), slots, 16)
    append_plain(vt, vs, vn.float().cpu().numpy(), slots, 16)
    np.testing.assert_array_equal(kv.k.cpu().numpy(), k)
    np.testing.assert_array_equal(kv.v.cpu().numpy(), vt.transpose(0, 1, 3, 2))


def test_append_leaves_out_slots_behind_the_cache(torch, dev):
    rng = np.random.default_rng(8)
    kv, host = cache(torch, dev, rng, 2, 2, 16, 16)
    x = [rng.normal(0, 1, (4, 2, 16)).astype(np.float32) for _ in range(2)]
    rk.device_check(dev)
    check_append(torch, dev, rng, kv, host, x, [3, 32, 2 ** 31 - 1, 16])
    with pytest.raises(rk.RkError) as e:
        rk.device_check(dev)
    assert e.value.code == rk.RK_ERR_ARGS
    rk.device_check(dev)


# ---- attention ---------------------------------------------------------


def attention_exact(torch, kv, q, table, lens, starts, scale, window):
    """The definition in 64 bits, with each output's bound. A row of queries is
    held as integers of its largest magnitude: 127 * 257 steps for 16-bit types
    (half a step is 2^-16 of the largest), 127 * 65793 for float32 (2^-24, and
    2^-24 for the product before the rounding), and the products are summed and
    joined in float32, so a score is off by at most
      ds = scale * sum_d |q_d k_d| * (hs + 4) u + scale * max|q| * sum_d |k_d| * (2^-16 or 2^-23 + 2^-22),
    and in powers of two |s| * 4u more; a weight by 2 ds + 2^-20 relative; the
    sums over n tokens by n u of the sum of magnitudes. Also returned: that sum,
    sum_t p_t |v_t|, and n 2^-38 of the largest value: weights enter as float16
    with the largest near 2^14, so one is off by 2^-11 of itself (16-bit types,
    one term) or 2^-39 of the largest."""
    B, hs, heads = kv.block, kv.head_size, q.shape[1]
    G = heads // kv.kv_heads
    k, v = kv.k.double() * kv.k_scale.double()[..., None, None], kv.v.double() * kv.v_scale.double()[..., None, None]
    k, v = k, v.transpose(2, 3)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound, mass, tiny = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    for i, have in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        pages = table[i][:-(-max(have, 0) // B)].long()
        ok = ((pages >= 0) & (pages < kv.blocks)).repeat_interleave(B)[:max(have, 0)]
        pages = pages.clamp(0, kv.blocks - 1)
        for t in range(a, b):
            pos = have - (b - t)
            lo, hi = max(0, pos + 1 - window) if window else 0, min(pos + 1, len(ok))
            if hi <= lo or not bool(ok[lo:hi].any()):
                continue
            keep = torch.nonzero(ok[lo:hi]).flatten() + lo
            for h in range(kv.kv_heads):
                kk = k[pages, h].reshape(-1, hs)[keep]
                vv = v[pages, h].reshape(-1, hs)[keep]
                qq = q[t, h * G:(h + 1) * G].double()
                s = qq @ kk.T * scale
                p = torch.softmax(s, -1)
                out[t, h * G:(h + 1) * G] = p @ vv
                ds = scale * (qq.abs() @ kk.abs().T) * (hs + 4) * U + s.abs() * 4 * U \
                    + scale * qq.abs().amax(1, keepdim=True) * kk.abs().sum(1)[None] * ((2.0 ** -23 if q.dtype == torch.float32 else 2.0 ** -16) + 2.0 ** -22)
                rel = 2 * ds.amax(1, keepdim=True) + 2.0 ** -20 + 2 * len(keep) * U
                bound[t, h * G:(h + 1) * G] = rel * (p @ vv.abs())
                mass[t, h * G:(h + 1) * G] = p @ vv.abs()
                tiny[t, h * G:(h + 1) * G] = len(keep) * 2.0 ** -38 * vv.abs().max()
    return out, bound, mass, tiny


def attention_bound(t, want, bound, mass, tiny):
    """How far an output of type t may be off: the above, the weights' rounding, and its own."""
    return bound + (0 if t == "f32" else 2.0 ** -11) * mass + tiny + HALF[t] * (want.abs() + bound + mass * 2.0 ** -10) \
        + {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[t]


def attention_case(torch, dev, seed, heads, kvh, hs, block, lens, new, t, window=0, scale=0.0, spare=0, spread=1.0, strided=False):
    """One call against the definition; new None: a query row each, without q_start."""
    rng = np.random.default_rng(seed)
    need = [-(-max(x, 0) // block) for x in lens]
    width = max(need + [0]) + 1
    kv, _ = cache(torch, dev, rng, sum(need) + 2, kvh, block, hs)
    perm, at = rng.permutation(sum(need) + 2), 0
    table = np.full((len(lens), width), 2 ** 30, np.int32)  # never followed behind a length
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(new if new is not None else [1] * len(lens))]).astype(int).tolist()
    rows = starts[-1] + spare
    x = torch.from_numpy((rng.normal(0, spread, (rows, heads, hs)))).cuda().to(dtype(torch, t))
    if strided:
        wide = torch.zeros((rows, heads * hs + 48), dtype=x.dtype, device="cuda")
        q = wide[:, 16:16 + heads * hs].unflatten(1, (heads, hs))
        q.copy_(x)
        out = torch.full((rows, 3, heads, hs), 77.0, dtype=x.dtype, device="cuda")[:, 1]
    else:
        q, out = x, torch.full(x.shape, 77.0, dtype=x.dtype, device="cuda")
    table = torch.from_numpy(table).cuda()
    got = kv.attention(q, table, ints(torch, lens), q_start=None if new is None else ints(torch, starts), scale=scale,
                       window=window, out=out)
    assert got is out
    rk.device_check(dev)
    want, *more = attention_exact(torch, kv, q, table, lens, starts, scale or 1 / math.sqrt(hs), window)
    assert bool((got[starts[-1]:].float() == 77.0).all()), "rows behind the last request were written"
    n = starts[-1]
    most = attention_bound(t, want, *more)[:n]
    off = (got[:n].double() - want[:n]).abs()
    assert bool(torch.isfinite(got[:n].float()).all())
    worst = (off / most).max().item() if n else 0
    assert worst <= 1, worst


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs", [16, 32, 48, 64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_one_token(torch, dev, t, hs, block):
    attention_case(torch, dev, hs + block, 6, 2, hs, block, [1, 15, 16, 17, 0, 33, 100, 259, block, block + 1], None, t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (5, 1), (7, 7), (14, 2), (8, 1), (9, 1), (32, 2), (17, 1), (48, 1)])
def test_attention_head_layouts(torch, dev, t, heads, kvh):
    attention_case(torch, dev, heads, heads, kvh, 64, 32, [77, 1, 300], None, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lens", [([3, 0, 1, 17, 64], [3, 50, 1, 60, 200]), ([1], [1]), ([130], [130]), ([33, 40], [33, 777])],
                         ids=str)
def test_attention_several_rows(torch, dev, t, new, lens):
    attention_case(torch, dev, len(new), 8, 2, 64, 16, lens, new, t, spare=3)
    attention_case(torch, dev, len(new), 6, 1, 128, 64, lens, new, t, spare=1, strided=True)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
@pytest.mark.parametrize("block", [16, 64])
def test_attention_window(torch, dev, window, block):
    attention_case(torch, dev, window, 4, 2, 64, block, [1, 40, 300, 0], None, "f32", window=window)
    attention_case(torch, dev, window, 4, 2, 64, block, [30, 40, 300], [30, 2, 64], "bf16", window=window)


@pytest.mark.parametrize("new", [None, [20, 7]], ids=str)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_rows_off_boundaries(torch, dev, t, new):
    """Rows of q and out one value off any boundary, an odd stride apart: the same bits."""
    rng = np.random.default_rng(14)
    kv, _ = cache(torch, dev, rng, 60, 2, 32, 80)
    starts = None if new is None else ints(torch, [0, 20, 27])
    rows = 2 if new is None else 27
    q = torch.from_numpy(rng.normal(0, 1, (rows, 6, 80))).cuda().to(dtype(torch, t))
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(2, 30)
    lens = ints(torch, [900, 33])
    want = kv.attention(q, table, lens, q_start=starts)
    wide = torch.full((2, rows, 483), 77.0, dtype=q.dtype, device="cuda")
    q2, out = (wide[i, :, 1:481].unflatten(1, (6, 80)) for i in range(2))
    q2.copy_(q)
    kv.attention(q2, table, lens, q_start=starts, out=out)
    assert bool(torch.equal(out, want))
    assert bool((wide[1, :, 0] == 77).all()) and bool((wide[1, :, 481:] == 77).all())


def test_attention_rows_without_a_token(torch, dev):
    """Lengths of zero and below, and queries in front of the first token, give zeros."""
    attention_case(torch, dev, 1, 4, 2, 32, 16, [0, 5, -4, 0], [2, 9, 3, 0], "f32")
    attention_case(torch, dev, 1, 4, 2, 32, 16, [0, 0], None, "bf16")


def test_attention_long(torch, dev):
    attention_case(torch, dev, 2, 8, 2, 64, 32, [20011], None, "f32")
    attention_case(torch, dev, 3, 4, 1, 128, 64, [9000, 3, 7001], None, "bf16")
    attention_case(torch, dev, 4, 4, 1, 128, 16, [6000, 33], [20, 7], "f16")


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_peaked_and_flat(torch, dev, t):
    """Scores from flat to one that takes all, and a given scale."""
    attention_case(torch, dev, 5, 4, 2, 64, 32, [500, 70], None, t, spread=30.0)
    attention_case(torch, dev, 6, 4, 2, 64, 32, [500, 70], None, t, spread=1e-4)
    attention_case(torch, dev, 7, 4, 2, 64, 32, [500, 70], None, t, scale=0.01)


def test_attention_scales_far_apart(torch, dev):
    """Pages whose value scales differ by many powers of two, one of them zero: the small ones count where their scores do."""
    rng = np.random.default_rng(9)
    kv, _ = cache(torch, dev, rng, 8, 1, 16, 32)
    kv.v_scale.copy_(torch.tensor([1e-6, 1e6, 1.0, 0.0, 1e-20, 1e20, 1e3, 1.0], device="cuda")[:, None])
    q = torch.from_numpy(rng.normal(0, 3, (4, 2, 32)).astype(np.float32)).cuda()
    table = torch.tensor([[0, 1], [2, 3], [4, 4], [6, 0]], dtype=torch.int32, device="cuda")
    lens = [32, 30, 32, 17]
    got = kv.attention(q, table, ints(torch, lens))
    want, *more = attention_exact(torch, kv, q, table, lens, [0, 1, 2, 3, 4], 1 / math.sqrt(32), 0)
    assert bool(((got.double() - want).abs() <= attention_bound("f32", want, *more)).all())


def test_attention_bad_pages_are_left_out(torch, dev):
    rng = np.random.default_rng(10)
    kv, _ = cache(torch, dev, rng, 4, 2, 16, 64)
    q = torch.from_numpy(rng.normal(0, 1, (3, 4, 64)).astype(np.float32)).cuda()
    table = torch.tensor([[0, -1, 1], [4, 2, 2 ** 31 - 1], [-5, 99, 7]], dtype=torch.int32, device="cuda")
    lens = [40, 48, 33]
    rk.device_check(dev)
    got = kv.attention(q, table, ints(torch, lens))
    with pytest.raises(rk.RkError):
        rk.device_check(dev)
    want, *more = attention_exact(torch, kv, q, table, lens, [0, 1, 2, 3], 1 / 8, 0)
    assert bool(((got.double() - want).abs() <= attention_bound("f32", want, *more)).all())
    assert bool((got[2] == 0).all())


def test_attention_lengths_past_the_table(torch, dev):
    """A length past the table's width ends at the table."""
    rng = np.random.default_rng(11)
    kv, _ = cache(torch, dev, rng, 4, 1, 16, 32)
    q = torch.from_numpy(rng.normal(0, 1, (2, 1, 32)).astype(np.float32)).cuda()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    got = kv.attention(q, table, ints(torch, [1000, 2 ** 31 - 1]))
    want = kv.attention(q, table, ints(torch, [32, 32]))
    assert bool(torch.equal(got, want))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_queries_that_are_not_finite(torch, dev, t):
    """A query with a NaN or an infinity gives NaN, and no other row or head does."""
    rng = np.random.default_rng(12)
    kv, _ = cache(torch, dev, rng, 8, 2, 16, 64)
    q = torch.from_numpy(rng.normal(0, 1, (5, 6, 64))).cuda().to(dtype(torch, t))
    clean = q.clone()
    q[1, 2, 5], q[3, 0, 63], q[4, 5, 0] = math.nan, math.inf, -math.inf
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    got = kv.attention(q, table, ints(torch, [100]), q_start=ints(torch, [0, 5]))
    want = kv.attention(clean, table, ints(torch, [100]), q_start=ints(torch, [0, 5]))
    bad = torch.zeros((5, 6), dtype=torch.bool, device="cuda")
    bad[1, 2] = bad[3, 0] = bad[4, 5] = True
    assert bool(got[bad].isnan().all())
    assert bool(torch.equal(got[~bad], want[~bad]))


def test_attention_large_and_small_queries(torch, dev):
    """float32 and bfloat16 queries outside float16's range."""
    for spread, scale in ((1e30, 1e-30), (1e-30, 1e30), (1e5, 1e-5)):
        for t in ("f32", "bf16"):
            attention_case(torch, dev, 13, 4, 2, 64, 16, [100, 7], None, t, spread=spread, scale=scale)


def test_attention_many_requests(torch, dev):
    rng = np.random.default_rng(14)
    attention_case(torch, dev, 14, 4, 2, 32, 16, rng.integers(0, 90, 300).tolist(), None, "bf16")
    attention_case(torch, dev, 15, 2, 1, 64, 32, rng.integers(20, 300, 70).tolist(), rng.integers(0, 20, 70).tolist(), "f32")


def test_attention_offsets_past_32_bits(torch, dev):
    """Pages whose bytes lie behind 2^31 and 2^32 of a cache of 4.3 GB a tensor."""
    kv = rk.PagedKV8.new(dev, (1 << 32) // (8 * 64 * 128) + 40, 8, 64, 128)
    rng = np.random.default_rng(16)
    pages = [kv.blocks - 1, kv.blocks - 30, kv.blocks // 2 + 3]
    rows = 64 * 3
    x = [torch.from_numpy(rng.normal(0, 1, (rows, 8, 128)).astype(np.float32)).cuda() for _ in range(2)]
    slots = [pages[j // 64] * 64 + j % 64 for j in range(rows)]
    kv.append(x[0], x[1], ints(torch, slots))
    q = torch.from_numpy(rng.normal(0, 1, (1, 16, 128)).astype(np.float32)).cuda()
    got = kv.attention(q, ints(torch, [pages]), ints(torch, [rows]))
    small = rk.PagedKV8.new(dev, 3, 8, 64, 128)
    small.append(x[0], x[1], ints(torch, list(range(rows))))
    want = small.attention(q, ints(torch, [[0, 1, 2]]), ints(torch, [rows]))
    assert bool(torch.equal(got, want)) and bool((got != 0).any())
    for j, p in enumerate(pages):
        assert bool(torch.equal(kv.v[p], small.v[j])) and bool(torch.equal(kv.k_scale[p], small.k_scale[j]))


def test_attention_workspace_is_checked(torch, dev):
    """Wide tables need the workspace, whole and aligned; those of 512 tokens none."""
    import ctypes as C
    kv = rk.PagedKV8.new(dev, 2, 1, 16, 32)
    need = rk.lib().rk_kv8_attention_workspace(dev.h, kv.at, 2)
    assert need > 0
    q, lens = torch.zeros((1, 2, 32), device="cuda"), ints(torch, [3])

    def call(width, ws, size):
        table = torch.zeros((1, width), dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()  # the call runs on the device's own stream
        return rk.lib().rk_kv8_attention(dev.h, kv.at, 0, 1, 2, 1, q.data_ptr(), 64, None, lens.data_ptr(), table.data_ptr(), width,
                                         C.c_float(0), 0, q.data_ptr(), 64, ws, size, None)
    for ws, size in ((None, need), (q.data_ptr(), need - 1), (q.data_ptr() + 4, need)):
        assert call(33, ws, size) == rk.RK_ERR_ARGS
    assert call(32, None, 0) == rk.RK_OK
    rk.device_check(dev)
    torch.cuda.synchronize()


# ---- norm --------------------------------------------------------------


def check_norm(torch, dev, x, w, eps, group, residual=None, sum_out=None):
    """The integers and h value by value; the scales within the error of a sum of cols squares (cols u / 2 after the root) and a few roundings."""
    xf, cols = x.float(), x.shape[1]
    rf = None if residual is None else residual.float()
    h = xf if rf is None else xf + rf
    q, scales, total = rk.add_rmsnorm_q8(dev, x, w, eps, group=group, residual=residual, sum_out=sum_out)
    g = group or cols
    u = (h * w.float()).reshape(-1, cols // g, g)
    base = u.abs().amax(2) * torch.tensor(np.float32(1 / 127), device="cuda")
    base = torch.where(base < 2.0 ** -120, torch.zeros_like(base), base)
    inv = torch.where(base > 0, torch.ones_like(base) / base, torch.zeros_like(base))
    want = (u * inv[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(x.shape)
    assert bool(torch.equal(q, want))
    r = 1 / ((h.double() ** 2).mean(1) + eps).sqrt()
    ws = base.double() * r[:, None]
    assert bool(((scales.double() - ws).abs() <= ws * (cols / 2 + 8) * U + 2.0 ** -149).all())
    if total is None:
        assert residual is None and sum_out is None
    else:
        assert bool(torch.equal(total, h.to(x.dtype)))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape,group", [((1, 32), 32), ((3, 96), 32), ((5, 288), 0), ((2, 1), 0), ((4, 77), 0), ((7, 77), 11),
                                         ((3, 4096), 32), ((2, 5120), 128), ((33, 896), 64), ((1, 30000), 0), ((2, 65536), 64),
                                         ((300, 640), 32), ((3, 4096), 4096), ((1, 262144), 128), ((2, 1000), 8), ((2, 520), 4)],
                         ids=str)
def test_norm(torch, dev, t, shape, group):
    gen = torch.Generator(device="cuda").manual_seed(shape[0] + shape[1])
    x = torch.randn(shape, generator=gen, device="cuda").to(dtype(torch, t))
    w = (1 + 0.2 * torch.randn(shape[1], generator=gen, device="cuda")).to(x.dtype)
    res = (3 * torch.randn(shape, generator=gen, device="cuda")).to(x.dtype)
    check_norm(torch, dev, x, w, 1e-5, group)
    check_norm(torch, dev, x, w, 1e-6, group, res)
    out = torch.empty_like(x)
    check_norm(torch, dev, x, w, 0.0, group, None, out)
    # rows a stride apart, of an odd offset; the sum written over the residual
    wide = torch.randn((shape[0], 2 * shape[1] + 5), generator=gen, device="cuda").to(x.dtype)
    want = (wide[:, 1:1 + shape[1]].float() + res.float()).to(x.dtype)
    q, s, total = rk.add_rmsnorm_q8(dev, wide[:, 1:1 + shape[1]], w, 1e-5, group=group, residual=res.clone())
    inplace = res.clone()
    q2, s2, total2 = rk.add_rmsnorm_q8(dev, wide[:, 1:1 + shape[1]], w, 1e-5, group=group, residual=inplace, sum_out=inplace)
    assert bool(torch.equal(q, q2)) and bool(torch.equal(s, s2)) and bool(torch.equal(inplace, want)) and bool(torch.equal(total, want))
    assert total2 is inplace


def test_norm_special_rows(torch, dev):
    """Rows of zeros, of tiny and of huge values, with a NaN, with an infinity."""
    x = torch.randn((6, 64), device="cuda")
    x[0], x[1], x[2] = 0, 1e-38, x[2] * 1e15
    w = torch.ones(64, device="cuda")
    check_norm(torch, dev, x[:4].contiguous(), w, 1e-5, 32)
    x[4, 3], x[5, 40] = math.nan, math.inf
    q, s, _ = rk.add_rmsnorm_q8(dev, x, w, 1e-5, group=32)
    assert bool(s[4].isnan().all()) and q[4, 3] == 0
    assert s[5, 0] == 0 and bool(s[5, 1].isnan()) and bool((q[5, 32:] == 0).all())
    assert bool((s[0] == 0).all()) and bool((q[0] == 0).all())
    check_norm(torch, dev, x[3:4].contiguous(), w, 1e-5, 32)


# ---- 4-bit products ----------------------------------------------------


def w4_case(torch, dev, rows, cols, group, xg, n, zeros, st, t, extra=0):
    gen = torch.Generator(device="cuda").manual_seed(rows + cols + n)
    w = torch.randint(0, 256, (rows, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = (0.01 * torch.exp(torch.randn((rows, cols // group), generator=gen, device="cuda"))).to(dtype(torch, st))
    z = torch.randint(0, 16, s.shape, generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    x = torch.randint(-127, 128, (n, cols), generator=gen, device="cuda", dtype=torch.int8)
    xs = 0.02 * torch.exp(torch.randn((n, cols // xg), generator=gen, device="cuda"))
    used = dev.used()
    m = rk.W4Matrix(dev, w, s, z)
    assert m.bytes() > 0 and dev.used() == used + m.bytes()
    out = torch.full((n + 1, rows + extra), 5.0, dtype=dtype(torch, t), device="cuda")
    got = m.mulvec(x, xs, out=out[:n, :rows])
    b = w.reshape(rows, cols // 32, 16).long()
    W = torch.cat([b & 15, b >> 4], 2).reshape(rows, cols // group, group).double()
    W = ((W - (8 if z is None else z.double()[..., None])) * s.double()[..., None]).reshape(rows, cols)
    X = (x.reshape(n, cols // xg, xg).double() * xs.double()[..., None]).reshape(n, cols)
    want, mass = X @ W.T, X.abs() @ W.abs().T
    # each run of columns: the integer's and the scales' roundings, and the sum over the runs
    runs = cols // min(group, xg) + 8
    off = (got.double() - want).abs()
    tiny = 2.0 ** -25 if t == "f16" else 0
    assert bool((off <= mass * runs * U + HALF[t] * (want.abs() + mass * runs * U) + tiny).all()), (off / mass).max()
    assert bool((out[n] == 5.0).all()) and bool((out[:n, rows:] == 5.0).all())
    again = m.mulvec(x, xs, dtype=dtype(torch, t))
    assert bool(torch.equal(again, got))
    m.free()
    assert dev.used() == used


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,cols,group,xg,n", [(1, 32, 32, 32, 1), (16, 64, 32, 64, 2), (17, 96, 32, 96, 3), (100, 896, 128, 32, 1),
                                                  (33, 4096, 128, 128, 8), (64, 288, 96, 32, 9), (257, 1024, 1024, 1024, 16),
                                                  (48, 640, 64, 160, 17), (130, 2048, 32, 32, 5), (5, 14336, 64, 128, 1),
                                                  (2000, 512, 128, 512, 40), (31, 160, 160, 32, 33)], ids=str)
def test_w4(torch, dev, rows, cols, group, xg, n, zeros, t):
    w4_case(torch, dev, rows, cols, group, xg, n, zeros, {"f32": "f16", "f16": "bf16", "bf16": "f32"}[t], t, extra=3)


def test_w4_wide(torch, dev):
    w4_case(torch, dev, 20, rk.MAX_COLS, 128, 128, 2, True, "f16", "f32")
    w4_case(torch, dev, 20, rk.MAX_COLS, rk.MAX_COLS, rk.MAX_COLS, 1, True, "f32", "f32")


def test_w4_extreme_integers(torch, dev):
    """The largest sums: every product 15 * 127 over the widest row."""
    cols = rk.MAX_COLS
    w = torch.full((1, cols // 2), 0xff, dtype=torch.uint8)
    m = rk.W4Matrix(dev, w, torch.ones((1, 1)), torch.zeros((1, 1), dtype=torch.uint8))
    x = torch.full((1, cols), -127, dtype=torch.int8, device="cuda")
    assert m.mulvec(x, torch.ones((1, 1), device="cuda")).item() == float(np.float32(-127 * 15 * cols))
    m.free()


# ---- together ----------------------------------------------------------


class Step:
    """A layer's decode step as a program would write it: norm, fused projection,
    pages, append, attention, output projection and the next norm."""

    def __init__(self, torch, dev, t, dim=256, heads=4, kvh=2, hs=64, block=16, n=3, rows=8, seed=3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.dev, self.heads, self.kvh, self.hs, self.n, self.block = torch, dev, heads, kvh, hs, n, block

        def w4(r, c):
            w = torch.randint(0, 256, (r, c // 2), generator=gen, device="cuda", dtype=torch.uint8)
            return rk.W4Matrix(dev, w, torch.full((r, c // 64), 0.01).half(), torch.full((r, c // 64), 7, dtype=torch.uint8))
        self.qkv, self.wo = w4((heads + 2 * kvh) * hs, dim), w4(dim, heads * hs)
        self.w = torch.ones(dim, device="cuda", dtype=t)
        self.wa = torch.ones(heads * hs, device="cuda", dtype=t)
        self.x = torch.randn((rows, dim), generator=gen, device="cuda").to(t)
        self.res = torch.randn((rows, dim), generator=gen, device="cuda").to(t)
        self.kv = rk.PagedKV8.new(dev, 40, kvh, block, hs)
        self.pages = rk.PageTables(dev, n, 12, block, rows)
        self.ctx, self.new = ints(torch, [0] * n), ints(torch, [0] * n)
        self.free, self.head = ints(torch, list(range(39, -1, -1))), ints(torch, [0])

    def run(self):
        q, s, h = rk.add_rmsnorm_q8(self.dev, self.x, self.w, 1e-5, group=32, residual=self.res)
        qkv = self.qkv.mulvec(q, s, dtype=self.x.dtype).unflatten(1, (self.heads + 2 * self.kvh, self.hs))
        self.pages.build(self.ctx, self.new, self.free, self.head)
        self.kv.append(qkv[:, self.heads:self.heads + self.kvh], qkv[:, self.heads + self.kvh:], self.pages.slots)
        out = self.torch.zeros((self.x.shape[0], self.heads, self.hs), device="cuda", dtype=self.x.dtype)
        self.kv.attention(qkv[:, :self.heads], self.pages.table, self.pages.lens, q_start=self.pages.q_start, out=out)
        a, sa, _ = rk.add_rmsnorm_q8(self.dev, out.flatten(1), self.wa, 1e-5, group=64)
        return self.wo.mulvec(a, sa, dtype=self.x.dtype), h, qkv, out

    def advance(self):
        self.ctx.copy_(self.pages.lens)
        self.head.copy_(self.pages.info[3:4])

    def free_all(self):
        self.qkv.free()
        self.wo.free()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_decode_step_together(torch, dev, t):
    """Prompts, then single tokens, in padded steps of 8 rows, run eagerly and as one captured graph: the same bits, and the
    attention of each step is its definition's over what the cache holds."""
    eager, graphed = (Step(torch, dev, dtype(torch, t)) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.run()
    torch.cuda.current_stream().wait_stream(side)
    graphed.kv.k.zero_(), graphed.kv.v.zero_(), graphed.kv.k_scale.zero_(), graphed.kv.v_scale.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = graphed.run()
    total = [0, 0, 0]
    for new in ([5, 0, 3], [1, 1, 1], [1, 7, 0], [0, 0, 0], [1, 1, 1], [6, 1, 1], [1, 1, 1]):
        for s in (eager, graphed):
            s.new.copy_(ints(torch, new))
        got = eager.run()
        graph.replay()
        for a, b in zip(got, kept):
            assert bool(torch.equal(a, b))
        total = [a + b for a, b in zip(total, new)]
        assert eager.pages.lens.tolist() == total and eager.pages.info.tolist()[2] == 0
        rows = sum(new)
        starts = [0, new[0], new[0] + new[1], rows]
        want, *more = attention_exact(torch, eager.kv, got[2][:, :4], eager.pages.table, total, starts, 1 / 8, 0)
        assert bool(((got[3].double() - want).abs() <= attention_bound(t, want, *more))[:rows].all())
        assert bool((got[3][rows:] == 0).all())
        for s in (eager, graphed):
            s.advance()
    rk.device_check(dev)
    eager.free_all()
    graphed.free_all()


def test_two_streams_at_once(torch, dev):
    """Two calls on streams of their own give what each gives alone."""
    rng = np.random.default_rng(20)
    kv, _ = cache(torch, dev, rng, 300, 2, 32, 64)
    table = torch.arange(300, dtype=torch.int32, device="cuda")[None].contiguous()
    qs = [torch.from_numpy(rng.normal(0, 1, (1, 8, 64)).astype(np.float32)).cuda() for _ in range(2)]
    lens = [ints(torch, [9600]), ints(torch, [4000])]
    want = [kv.attention(q, table, n) for q, n in zip(qs, lens)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for st, q, n in zip(streams, qs, lens):
            with torch.cuda.stream(st):
                got.append(kv.attention(q, table, n))
        torch.cuda.synchronize()
        assert all(bool(torch.equal(g, w)) for g, w in zip(got, want))


def test_binding_refuses_tensors(torch, dev):
    kv = rk.PagedKV8.new(dev, 2, 2, 16, 32)
    q = torch.zeros((1, 4, 32), device="cuda")
    table, lens = ints(torch, [[0]]), ints(torch, [1])
    x8 = torch.zeros((1, 64), dtype=torch.int8, device="cuda")
    m = rk.W4Matrix(dev, torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 2)))
    for call in (lambda: kv.attention(q.cpu(), table, lens), lambda: kv.attention(q.double(), table, lens),
                 lambda: kv.attention(q[:, :3], table, lens), lambda: kv.attention(q[..., :16], table, lens),
                 lambda: kv.attention(q, table.long(), lens), lambda: kv.attention(q, table, lens[:0]),
                 lambda: kv.attention(q.transpose(1, 2).contiguous().transpose(1, 2), table, lens),
                 lambda: kv.attention(q, table, lens, window=-1), lambda: kv.attention(q, table, lens, out=q.half()),
                 lambda: kv.append(q, q, lens), lambda: kv.append(q[:, :2], q[:, :2].half(), lens),
                 lambda: kv.append(q[:, :2], q[:, :2], lens.long()), lambda: kv.append(q[:, :2], q[:, 2:], torch.zeros(2, dtype=torch.int32)),
                 lambda: rk.PagedKV8(dev, kv.k, kv.k, kv.k_scale, kv.v_scale),
                 lambda: rk.PagedKV8(dev, kv.k, kv.v, kv.k_scale.double(), kv.v_scale),
                 lambda: rk.add_rmsnorm_q8(dev, q[0], q[0], 1e-5), lambda: rk.add_rmsnorm_q8(dev, q[0], q[0, 0].half(), 1e-5),
                 lambda: rk.add_rmsnorm_q8(dev, q[0], q[0, 0], 1e-5, group=5), lambda: rk.add_rmsnorm_q8(dev, q[0], q[0, 0], 1e-5, group=-1),
                 lambda: rk.add_rmsnorm_q8(dev, q[0], q[0, 0], 1e-5, residual=q[0, :2]),
                 lambda: m.mulvec(x8[:, :32], torch.ones((1, 1), device="cuda")), lambda: m.mulvec(x8, torch.ones((1, 3), device="cuda")),
                 lambda: m.mulvec(x8, torch.ones((1, 4), device="cuda")), lambda: m.mulvec(x8, torch.ones((1, 2))),
                 lambda: m.mulvec(x8, torch.ones((1, 2), device="cuda"), dtype=torch.float64),
                 lambda: rk.W4Matrix(dev, torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 3))),
                 lambda: rk.W4Matrix(dev, torch.zeros((4, 32), dtype=torch.int8), torch.ones((4, 2))),
                 lambda: rk.PageTables(dev, 1, 1, 16, 4, table=lens),
                 lambda: rk.PageTables(dev, 1, 1, 16, 4).build(lens, lens.long(), lens),
                 lambda: rk.PageTables(dev, 1, 1, 17, 4).build(lens, lens, lens)):
        with pytest.raises(rk.RkError) as e:
            call()
        assert e.value.code == rk.RK_ERR_ARGS
    m.free()
    rk.device_check(dev)


# ---- calls beside the ordinary ones ------------------------------------


@pytest.mark.parametrize("new,spare", [([1, 1, 1], 0), ([1, 1, 1], 253), ([1, 1, 1, 64], 0), ([2, 40], 0)], ids=str)
def test_attention_precision_goes_by_type_alone(torch, dev, new, spare):
    """float16 queries enter with 24 bits and their weights with 22 whatever else the call holds: alone, in a buffer far
    larger than its rows, beside a prompt. So the float32 bound holds with float16's own rounding on top. (The value
    scales lie half a step beside a float16, where a weight held in one float16 is off by 2^-12.)"""
    rng = np.random.default_rng(30)
    kv, _ = cache(torch, dev, rng, 40, 2, 16, 64)
    kv.v_scale.fill_(1 + 0.98 * 2.0 ** -11)
    lens = [90, 33, 100, 150][:len(new)]
    starts = np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
    q = torch.from_numpy(rng.normal(0, 1, (starts[-1] + spare, 4, 64))).cuda().half()
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)[:len(new)].contiguous()
    got = kv.attention(q, table, ints(torch, lens), q_start=ints(torch, starts))[:starts[-1]]
    want, *more = (x[:starts[-1]] for x in attention_exact(torch, kv, q.float(), table, lens, starts, 1 / 8, 0))
    most = attention_bound("f32", want, *more)
    off, allowed = (got.double() - want).abs(), most + HALF["f16"] * (want.abs() + most) + 2.0 ** -25
    assert bool((off <= allowed).all()), (off / allowed).max().item()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_attention_does_not_depend_on_pages_it_does_not_hold(torch, dev, t):
    """Pages of no request, page 0 among them, may hold anything: the last 16 tokens of a tile of 32 may have no page."""
    rng = np.random.default_rng(33)
    kv, _ = cache(torch, dev, rng, 12, 2, 16, 32)
    q = torch.from_numpy(rng.normal(0, 1, (3, 4, 32))).cuda().to(dtype(torch, t))
    table = torch.tensor([[3, 0, 0], [4, 5, 6], [7, -1, -1]], dtype=torch.int32, device="cuda")
    args = table, ints(torch, [10, 48, 16])
    want = kv.attention(q, *args)
    for scale in (math.nan, math.inf):
        for x in (kv.k_scale, kv.v_scale):
            x[:3] = scale
            x[8:] = scale
        assert bool(torch.equal(kv.attention(q, *args), want))
    rk.device_check(dev)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("window", [1, 16, 20, 100])
def test_attention_pages_in_front_of_the_window(torch, dev, t, block, window):
    """Pages that lie wholly in front of every row's window may have left the table: nothing looks them up."""
    rng = np.random.default_rng(34)
    lens, new = [300, 141, 47, 16, 33, 128], [1, 3, 1, 1, 2, 1]
    need = [-(-n // block) for n in lens]
    kv, _ = cache(torch, dev, rng, sum(need), 2, block, 32)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
    q = torch.from_numpy(rng.normal(0, 1, (starts[-1], 4, 32))).cuda().to(dtype(torch, t))
    whole, at = np.full((len(lens), max(need)), -1, np.int32), 0
    for i, n in enumerate(need):
        whole[i, :n] = range(at, at + n)
        at += n
    gone = whole.copy()
    for i, n in enumerate(lens):
        first = max(0, n - new[i] + 1 - window)  # the first row's first visible token
        gone[i, :first // block] = -1
    rk.device_check(dev)
    want, got = (kv.attention(q, torch.from_numpy(x).cuda(), ints(torch, lens), q_start=ints(torch, starts), window=window)
                 for x in (whole, gone))
    rk.device_check(dev)
    assert bool(torch.equal(got, want))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [None, [20, 7]], ids=str)
def test_attention_scales_below_zero(torch, dev, t, new):
    """A page's integers times its scale, whatever the scale's sign."""
    rng = np.random.default_rng(31)
    kv, _ = cache(torch, dev, rng, 12, 2, 16, 64)
    kv.k_scale[::3].neg_()
    kv.v_scale[::2].neg_()
    lens, starts = [90, 80], [0, 1, 2] if new is None else [0, 20, 27]
    q = torch.from_numpy(rng.normal(0, 1, (starts[-1], 4, 64))).cuda().to(dtype(torch, t))
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    got = kv.attention(q, table, ints(torch, lens), q_start=None if new is None else ints(torch, starts))
    want, *more = attention_exact(torch, kv, q, table, lens, starts, 1 / 8, 0)
    assert bool(((got.double() - want).abs() <= attention_bound(t, want, *more)).all())


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_attention_scales_that_are_not_finite(torch, dev, t, scale, which):
    """Rows that see a token of such a page give NaN; the others give what they give without it."""
    rng = np.random.default_rng(32)
    kv, _ = cache(torch, dev, rng, 12, 1, 16, 32)
    q = torch.from_numpy(rng.normal(0, 1, (30, 2, 32))).cuda().to(dtype(torch, t))
    table = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32, device="cuda")
    args = table, ints(torch, [40, 64]), ints(torch, [0, 20, 30])
    want = kv.attention(q, *args)
    getattr(kv, which)[1] = scale  # tokens 16 .. 31 of the first request, whose rows are at 20 .. 39
    getattr(kv, which)[8:] = scale
    getattr(kv, which)[3] = scale  # behind the first request's end
    got = kv.attention(q, *args)
    assert bool(got[:20].isnan().all())
    assert bool(torch.equal(got[20:], want[20:]))
    kv.k_scale[1] = kv.v_scale[1] = 0.01
    getattr(kv, which)[1] = scale
    rows = ints(torch, [0, 20, 20])
    lens = ints(torch, [25, 0])  # rows at 5 .. 24: those up to 15 do not see page 1
    got = kv.attention(q, table, lens, q_start=rows)
    getattr(kv, which)[1] = 0.01
    want = kv.attention(q, table, lens, q_start=rows)
    assert bool(got[11:20].isnan().all())
    assert bool(torch.equal(got[:11], want[:11]))


def test_norm_products_past_float32(torch, dev):
    """h and weight finite, their product infinite: the group's factor is zero, and so are its integers."""
    for t, cols, group in (("f32", 64, 32), ("f32", 64, 0), ("f32", 77, 11), ("f32", 66, 2), ("bf16", 256, 64)):
        x = torch.randn((3, cols), device="cuda")
        w = torch.ones(cols, device="cuda")
        x[1, 3], w[3], w[5] = 1e10, 1e30, 1e-3
        x[1, 5] = -2.0
        x, w = x.to(dtype(torch, t)), w.to(dtype(torch, t))
        check_norm(torch, dev, x[::2].contiguous(), w, 1e-5, group)
        q, s, _ = rk.add_rmsnorm_q8(dev, x, w, 1e-5, group=group)
        g = group or cols
        first, end = 3 // g * g, 3 // g * g + g  # the group of column 3
        assert bool((q[1, first:end] == 0).all()) and s[1, 3 // g] == math.inf
        if group:
            check_norm(torch, dev, x[:, end:].contiguous(), w[end:].contiguous(), 1e-5, group)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("had,ratio", [(-2.0, -1.0), (-0.001, None), (math.nan, 0.0), (math.inf, 1.0)])
def test_append_to_pages_of_any_scale(torch, dev, t, had, ratio):
    """A page's scale counts by its magnitude, as zero if it is NaN; what the page held is rounded to the new one with its sign."""
    rng = np.random.default_rng(35)
    kv, host = cache(torch, dev, rng, 2, 2, 16, 32)
    kv.k_scale.fill_(had)
    kv.v_scale.fill_(had)
    x = torch.from_numpy(rng.normal(0, 1, (3, 2, 32))).cuda().to(dtype(torch, t))
    kv.append(x, x, ints(torch, [5, 6, 7]))
    m = x.float().abs().amax((0, 2)).cpu().numpy() * np.float32(1 / 127)
    s = np.maximum(m, np.float32(0 if math.isnan(had) else abs(had)))
    for scale in (kv.k_scale, kv.v_scale):
        np.testing.assert_array_equal(scale[0].cpu().numpy(), s)
        assert bool((scale[1].isnan() if math.isnan(had) else scale[1] == had).all())
    r = np.float32(had) / s if ratio is None else np.full_like(s, ratio)
    for got, before in ((kv.k, host[0]), (kv.v.transpose(2, 3), host[1].transpose(0, 1, 3, 2))):
        np.testing.assert_array_equal(got[0, :, :5].cpu().numpy(), np.rint(before[0, :, :5].astype(np.float32) * r[:, None, None]).astype(np.int8))
        inv = np.where(np.isinf(s), np.float32(0), np.float32(1) / s)
        np.testing.assert_array_equal(got[0, :, 5:8].cpu().numpy(), np.rint(x.float().cpu().numpy().transpose(1, 0, 2) * inv[:, None, None]).astype(np.int8))
        np.testing.assert_array_equal(got[0, :, 8:].cpu().numpy(), before[0, :, 8:])
        np.testing.assert_array_equal(got[1].cpu().numpy(), before[1])


def test_errors_of_these_operators_are_reported_by_the_check_alone(torch, dev):
    """A bad slot or page fails no other call on the device, and is not lost to one."""
    rng = np.random.default_rng(36)
    kv, _ = cache(torch, dev, rng, 2, 1, 16, 16)
    q = torch.zeros((1, 1, 16), device="cuda")
    m = rk.Matrix(dev, 4, 32, rk.FMT_F32, np.ones((4, 32), np.float32))
    rk.device_check(dev)
    for bad in (lambda: kv.append(q, q, ints(torch, [99])), lambda: kv.attention(q, ints(torch, [[7]]), ints(torch, [3]))):
        bad()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(m.mulvec(np.ones(32, np.float32)), np.full(4, 32, np.float32))
        with pytest.raises(rk.RkError) as e:
            rk.device_check(dev)
        assert e.value.code == rk.RK_ERR_ARGS
        rk.device_check(dev)
    m.free()


def test_requests_that_wait_for_a_page(torch, dev):
    """Three sequences share pages for two: a refused request keeps its context (ctx takes lens where lens is not zero), is
    given the same token again, and attends to all it holds once another sequence has ended."""
    n, block, width, kvh, hs = 3, 16, 3, 1, 16
    rng = np.random.default_rng(37)
    kv = rk.PagedKV8.new(dev, 5, kvh, block, hs)
    pages = rk.PageTables(dev, n, width, block, 64)
    ctx, free, head = ints(torch, [0] * n), ints(torch, [0, 1, 2, 3, 4]), ints(torch, [0])
    held = [[] for _ in range(n)]  # the keys of each sequence

    def step(new):
        pages.build(ctx, ints(torch, new), free, head)
        starts, lens = pages.q_start.tolist(), pages.lens.tolist()
        x = torch.from_numpy(rng.normal(0, 1, (64, kvh, hs)).astype(np.float32)).cuda()
        kv.append(x, x, pages.slots)
        for i in range(n):
            if lens[i]:
                held[i] += list(x[starts[i]:starts[i + 1]])
        out = torch.zeros((64, 2, hs), device="cuda")
        q = torch.zeros_like(out)  # even weights: the mean of the values
        kv.attention(q, pages.table, pages.lens, q_start=pages.q_start, out=out)
        for i in range(n):
            for j in range(new[i]):
                got = out[starts[i] + j, 0]
                if not lens[i]:
                    assert bool((got == 0).all())
                    continue
                seen = torch.stack(held[i])[:len(held[i]) - new[i] + j + 1, 0]
                # each value rounded to its page's scale, at most once more a growth of it
                assert bool(((got - seen.mean(0)).abs() <= 4 * 0.5 * 5 / 127).all())
        ctx.copy_(torch.where(pages.lens > 0, pages.lens, ctx))
        head.copy_(pages.info[3:4])
        return lens

    assert step([30, 16, 14]) == [30, 16, 14]          # 2 + 1 + 1 pages
    assert step([1, 1, 1]) == [31, 17, 15]             # the last page goes to the second
    assert step([1, 1, 1]) == [32, 18, 16]
    assert step([1, 1, 1]) == [0, 19, 0]               # no page for the first and the third
    assert ctx.tolist() == [32, 19, 16] and pages.info.tolist()[2] == 2
    assert step([1, 1, 1]) == [0, 20, 0]
    assert ctx.tolist() == [32, 20, 16]
    ended = pages.table[1, :2].clone()                  # the second ends: its pages are free again
    free, ctx[1], held[1] = ended, 0, []
    head.zero_()
    assert step([1, 0, 1]) == [33, 0, 17]
    assert pages.table[0].tolist()[2] == ended[0] and pages.table[2].tolist()[1] == ended[1]
    rk.device_check(dev)


def test_tables_of_buffers_side_by_side(torch, dev):
    """All of a call's buffers, and those between two steps, in one piece of memory."""
    n, width, rows, block = 3, 4, 9, 16
    ctx, new, free = [30, 0, 16], [3, 5, 1], [40, 41, 42, 43]
    sizes = [n, n, len(free), 1, n * width, n, n + 1, rows, rows, 4]
    at = np.concatenate([[0], np.cumsum(sizes)])
    arena = torch.full((int(at[-1]) + 1,), -9, dtype=torch.int32, device="cuda")
    arena[:at[4]] = ints(torch, ctx + new + free + [1])
    table = np.full((n, width), -9, np.int32)
    table[0, :2], table[2, :1] = (7, 8), 9
    arena[at[4]:at[5]] = torch.from_numpy(table).cuda().flatten()
    p = [arena[int(a):].data_ptr() for a in at[:-1]]
    torch.cuda.synchronize()  # the call runs on the device's own stream
    assert rk.lib().rk_page_tables(dev.h, n, block, p[0], p[1], p[2], p[3], len(free), p[4], width, p[5], p[6], p[7], p[8], rows,
                                   p[9], None) == rk.RK_OK
    rk.device_check(dev)
    assert rk.lib().rk_device_check(dev.h, None) == rk.RK_OK
    want = tables_plain(ctx, new, free, 1, table, block, rows)
    for i, w in enumerate(want):
        np.testing.assert_array_equal(arena[at[4 + i]:at[5 + i]].cpu().numpy(), np.array(w, np.int32).flatten())
    assert arena[-1].item() == -9


def test_attention_from_threads_of_one_stream(torch, dev):
    """Two threads that call on the same stream, whose calls share the stream's workspace."""
    import threading
    rng = np.random.default_rng(38)
    kv, _ = cache(torch, dev, rng, 300, 2, 32, 64)
    table = torch.arange(300, dtype=torch.int32, device="cuda")[None].contiguous()
    qs = [torch.from_numpy(rng.normal(0, 1, (k, 8, 64)).astype(np.float32)).cuda() for k in (1, 40)]
    lens, starts = [ints(torch, [9600]), ints(torch, [4000])], [ints(torch, [0, 1]), ints(torch, [0, 40])]
    want = [kv.attention(q, table, n, q_start=s) for q, n, s in zip(qs, lens, starts)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        for _ in range(200):
            got[i].append(kv.attention(qs[i], table, lens[i], q_start=starts[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 200 and all(bool(torch.equal(g, want[i])) for g in got[i])


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("shape,group", [((5000, 640), 32), ((3001, 1000), 8), ((3001, 1001), 7), ((4001, 77), 0), ((2001, 5120), 128)],
                         ids=str)
def test_norm_many_rows(torch, dev, t, shape, group):
    """More rows than the CTAs that the SMs hold, so that each takes several, and the sum in place."""
    gen = torch.Generator(device="cuda").manual_seed(39)
    x = torch.randn(shape, generator=gen, device="cuda").to(dtype(torch, t))
    w = (1 + 0.2 * torch.randn(shape[1], generator=gen, device="cuda")).to(x.dtype)
    res = (3 * torch.randn(shape, generator=gen, device="cuda")).to(x.dtype)
    check_norm(torch, dev, x, w, 1e-5, group, res)
    want = rk.add_rmsnorm_q8(dev, x, w, 1e-5, group=group, residual=res)
    for k in range(2):  # the sum over x, over the residual
        a, b = x.clone(), res.clone()
        got = rk.add_rmsnorm_q8(dev, a, w, 1e-5, group=group, residual=b, sum_out=b if k else a)
        assert all(bool(torch.equal(g, v)) for g, v in zip(got, want))


@pytest.mark.parametrize("rows,cols,group,xg,n,zeros,st", [
    (80000, 256, 128, 64, 1, True, "f16"), (80000, 256, 32, 32, 11, False, "bf16"),        # teams take several tiles
    (120007, 128, 64, 128, 8, True, "f32"), (90000, 96, 32, 96, 16, True, "f16"),
    (48, 14336, 32, 32, 9, False, "f16"), (48, 14336, 32, 32, 16, True, "f32"),            # vectors that do not fit
    (40, 14368, 32, 32, 16, True, "f16"), (40, 14368, 32, 14368, 9, False, "f32"),
    (40, 14400, 64, 64, 15, True, "bf16"), (5000, 8224, 32, 32, 40, True, "f16"),
    (3000, 14336, 128, 128, 16, True, "f16"), (40000, 4128, 32, 32, 16, True, "f32"),
    (9000, 14336, 32, 32, 16, True, "f32"), (9000, 14368, 32, 32, 9, False, "f16")], ids=str)
def test_w4_many_tiles_and_wide_rows(torch, dev, rows, cols, group, xg, n, zeros, st):
    w4_case(torch, dev, rows, cols, group, xg, n, zeros, st, "f32", extra=1)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs", [16, 32, 48, 64, 80, 96, 112, 128, 256])
def test_attention_pieces_of_every_head_size(torch, dev, t, hs):
    """Enough rows a request for two row tiles a warp, at short tables and over a joined long one."""
    attention_case(torch, dev, hs, 6, 2, hs, 16, [3, 60, 300], [3, 20, 64], t, spare=2)
    attention_case(torch, dev, hs + 1, 4, 1, hs, 64, [40, 2500], [7, 33], t, window=700)
