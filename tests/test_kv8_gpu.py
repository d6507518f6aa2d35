"""GPU tests of the paged 8-bit cache: block tables and slot maps, the quantising append (both bit for bit) and the attention
over it, against the plain 64-bit forms of kv8_ref. Bounds are derived there, per element."""
import numpy as np
import pytest
import torch

import dgx_attn as A
import kv8_ref as R

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


# ---------------------------------------------------------------- plan
def ref_plan(ctx, add, page, table, free, count, rows):
    """(status, table, cu, slots, left)"""
    B, cols = table.shape
    have, want = -(-ctx // page), -(-(ctx + add) // page)
    status = (1 if (want - have).sum() > count else 0) | (2 if (want > cols).any() else 0) | (4 if add.sum() > rows else 0)
    slots, cu = np.full(rows, -1), np.zeros(B + 1, int)
    if status:
        return status, table, cu, slots, count
    table, top, r = table.copy(), count, 0
    for b in range(B):
        for c in range(have[b], want[b]):
            top -= 1
            table[b, c] = free[top]
        for i in range(add[b]):
            p = ctx[b] + i
            slots[r] = table[b, p // page] * page + p % page
            r += 1
        cu[b + 1] = r
    return 0, table, cu, slots, top


def run_plan(ctx, add, page, table, free, count, rows, in_place=False):
    t = i32(table)
    cnt, left = i32([count]), i32([-7])
    if in_place:
        left = cnt
    cu, slots, status = i32(np.full(len(ctx) + 1, -9)), i32(np.full(rows, -9)), i32([-9])
    A.kv8_plan(i32(ctx), i32(add), page, t, i32(free), cnt, left, cu, slots, status)
    return int(status[0]), t.cpu().numpy(), cu.cpu().numpy(), slots.cpu().numpy(), int(left[0])


def plan_case(rng, B, hi, top, page, extra):
    ctx, add = rng.integers(0, hi + 1, B), rng.integers(0, top + 1, B)
    have, want = -(-ctx // page), -(-(ctx + add) // page)
    P = int(want.sum()) + extra
    ids = rng.permutation(P)
    table = np.full((B, int(want.max()) + 2), -1)
    for b in range(B):
        table[b, :have[b]], ids = ids[:have[b]], ids[have[b]:]
    return ctx, add, table, ids


@pytest.mark.parametrize("B,hi,top,page,spare,in_place", [
    (1, 0, 1, 16, 0, False), (1, 0, 0, 64, 0, True), (3, 40, 5, 16, 1, False), (64, 300, 1, 32, 3, True), (65, 100, 70, 64, 0, False),
    (300, 1000, 3, 64, 9, True), (1024, 64, 2, 16, 0, False), (1025, 64, 2, 16, 0, True), (2600, 50, 3, 32, 5, False),
    (40, 200, 900, 16, 2, False), (40, 200, 900, 16, 2, True), (1500, 30, 40, 16, 0, False)])
def test_plan(B, hi, top, page, spare, in_place):
    rng = np.random.default_rng(B * 7 + page)
    ctx, add, table, free = plan_case(rng, B, hi, top, page, 4)
    rows = int(add.sum()) + spare
    got = run_plan(ctx, add, page, table, free, len(free), rows, in_place)
    want = ref_plan(ctx, add, page, table, free, len(free), rows)
    for g, w, what in zip(got, want, ("status", "table", "cu", "slots", "left")):
        assert np.array_equal(g, w), what


@pytest.mark.parametrize("why,status", [("pages", 1), ("cols", 2), ("rows", 4), ("negative", 8), ("count", 8)])
@pytest.mark.parametrize("big", [False, True])
def test_plan_takes_all_or_nothing(why, status, big):
    rng = np.random.default_rng(5)
    ctx, add, table, free = plan_case(rng, 50, 100, 600 if big else 9, 16, 0)
    rows, count = int(add.sum()), len(free)
    if why == "pages":
        count -= 1
    elif why == "cols":
        table = table[:, :-3]
    elif why == "rows":
        rows -= 1
    elif why == "negative":
        add[17] = -1
    else:
        count += 1
    st, t, cu, slots, left = run_plan(ctx, add, 16, table, free, count, rows)
    assert st & status and (st == status or why in ("negative", "cols")), st
    assert np.array_equal(t, table) and not cu.any() and (slots == -1).all() and left == count


def test_plan_lengths_near_2_31():
    """Sums and positions past 32 bits are told, not wrapped."""
    table = np.full((3, 4), -1)
    for ctx, add in (([2 ** 31 - 1, 5, 5], [2 ** 31 - 1, 1, 1]), ([5, 5, 5], [2 ** 31 - 1] * 3), ([2 ** 31 - 1, 1, 1], [0, 1, 1])):
        st, t, cu, slots, left = run_plan(np.array(ctx), np.array(add), 64, table, np.arange(9), 9, 40)
        assert st & 2 and np.array_equal(t, table) and not cu.any() and (slots == -1).all() and left == 9


# ---------------------------------------------------------------- append
def test_plan_of_more_rows_than_32_bit_scans_hold():
    """Room for more than 2^20 rows: the wide scans, over more requests than a tile's 1024."""
    rng = np.random.default_rng(8)
    B, page, rows = 1500, 64, (1 << 20) + 777
    ctx, add = rng.integers(0, 300, B), rng.integers(0, 900, B)
    need = int((-(-(ctx + add) // page) - -(-ctx // page)).sum())
    free = rng.permutation(need + 3)
    table = np.full((B, 20), -7)
    have = -(-ctx // page)
    for b in range(B):
        table[b, :have[b]] = 500 + b
    for in_place in (False, True):
        got = run_plan(ctx, add, page, table, free, len(free), rows, in_place)
        for g, w in zip(got, ref_plan(ctx, add, page, table, free, len(free), rows)):
            assert np.array_equal(g, w)


def values(rng, rows, NKV, HD, dtype, sd=1.0):
    """Rows as the source type stores them: (tensor on the GPU, float64)."""
    t = torch.from_numpy(rng.standard_normal((rows, NKV, HD)) * sd).to(R.DTYPES[dtype])
    return t.cuda(), t.double().numpy()


def same_cache(cache, K, V, Ks, Vs, what=""):
    assert np.array_equal(cache.Ks.cpu().numpy(), Ks) and np.array_equal(cache.Vs.cpu().numpy(), Vs), f"{what}: scales"
    for t, want, name in ((cache.K, K, "K"), (cache.V, V, "V")):
        bad = np.argwhere(R.codes(t) != want)
        assert len(bad) == 0, f"{what}: {len(bad)} {name} codes differ, first at {bad[0].tolist()}: {R.codes(t)[tuple(bad[0])]:#x} for {want[tuple(bad[0])]:#x}"


@pytest.mark.parametrize("page,NKV,HD", [(16, 1, 128), (16, 3, 256), (32, 2, 512), (64, 4, 128), (64, 2, 256), (64, 1, 512)])
@pytest.mark.parametrize("dtype", ["fp32", "f16", "bf16"])
def test_append_runs_of_every_kind(page, NKV, HD, dtype):
    """Whole pages, runs that begin or end inside one, single tokens, skipped rows; then again behind them with larger values
    (the scales grow, the held codes are rounded again), then smaller ones (they stay)."""
    rng = np.random.default_rng(page * HD + NKV)
    P = 11
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    # request lengths 0 | page - 1 | 5 | page + 3 | 0; new tokens per call
    ctx = np.array([0, page - 1, 5, page + 3, 0])
    table = R.tables(rng, ctx + 3 * (page // 4) + 2 * page + 20, page, 60, 8) % P
    table = rng.permutation(P)[:10].reshape(5, 2)
    for step, (adds, sd) in enumerate((((2 * page, 1, 3, 1, 1), 1.0), ((0, page, 7, page // 4, page - 2), 9.0), ((0, 0, 1, 2, 1), 0.01))):
        slots = []
        for b in range(5):
            for i in range(adds[b]):
                p = int(ctx[b]) + i
                slots.append(int(table[b, p // page]) * page + p % page if p < 2 * page else -1)
            slots += [-1] if b % 2 else [P * page + 3]
            ctx[b] += adds[b]
        slots = np.array(slots)
        kt, k = values(rng, len(slots), NKV, HD, dtype, sd)
        vt, v = values(rng, len(slots), NKV, HD, dtype, sd * 0.3)
        R.append(K, V, Ks, Vs, k, v, slots)
        A.kv8_append(kt, vt, cache, i32(slots))
        torch.cuda.synchronize()
        same_cache(cache, K, V, Ks, Vs, f"step {step}")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_append_rounds_to_nearest_even_at_every_code(dtype):
    """Midpoints between all codes and their neighbours in fp32, subnormals, and magnitudes at the edges of a scale."""
    page, NKV, HD = 16, 1, 256
    mids = (R.POSITIVE[:-1] + R.POSITIVE[1:]) / 2
    x = np.concatenate([mids, np.nextafter(mids.astype(np.float32), np.float32(1e9)).astype(np.float64),
                        np.nextafter(mids.astype(np.float32), np.float32(0)).astype(np.float64), R.POSITIVE, [2.0 ** -10, 2.0 ** -30]])
    x = np.resize(np.concatenate([x, -x]), 15 * HD).reshape(15, 1, HD)
    edge = np.zeros((1, 1, HD))
    for top in (448.0, np.nextafter(np.float32(448), np.float32(0)), np.nextafter(np.float32(448), np.float32(500)), 256.0, 449.0):
        for sc in (1.0, 2.0 ** -20, 2.0 ** 30, 2.0 ** -45, 2.0 ** 41):
            edge[0, 0, 7] = -float(top)
            kk = torch.from_numpy(np.concatenate([x, edge]) * sc).to(R.DTYPES[dtype])
            k = kk.double().numpy()
            if not np.isfinite(k).all():
                continue
            K, V, Ks, Vs = R.make_cache(np.random.default_rng(1), 1, page, NKV, HD)
            cache = R.to_cache(A, K, V, Ks, Vs)
            slots = np.arange(16)
            R.append(K, V, Ks, Vs, k, k, slots)
            A.kv8_append(kk.cuda(), kk.cuda(), cache, i32(slots))
            same_cache(cache, K, V, Ks, Vs, f"top {top} scale {sc}")


@pytest.mark.parametrize("dtype", ["fp32", "f16", "bf16"])
def test_append_values_that_are_not_finite(dtype):
    rng = np.random.default_rng(3)
    page, NKV, HD, P = 32, 2, 128, 4
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    kt, _ = values(rng, 40, NKV, HD, dtype)
    vt, _ = values(rng, 40, NKV, HD, dtype)
    kt[3, 0, 17], kt[9, 1, 0], vt[3, 1, 5], vt[20, 0, 127], vt[33, 1, 64] = float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")
    kt[5] = float("nan")
    slots = np.arange(40) + 2 * page - 9        # 9 tokens into page 1, 31 into page 2
    R.append(K, V, Ks, Vs, kt.double().cpu().numpy(), vt.double().cpu().numpy(), slots)
    A.kv8_append(kt, vt, cache, i32(slots))
    same_cache(cache, K, V, Ks, Vs)
    grow, _ = values(rng, 1, NKV, HD, dtype, 50.0)   # and held NaN codes stay NaN when the scale grows
    R.append(K, V, Ks, Vs, grow.double().cpu().numpy(), grow.double().cpu().numpy(), np.array([2 * page + 31]))
    A.kv8_append(grow, grow, cache, i32([2 * page + 31]))
    same_cache(cache, K, V, Ks, Vs, "grown")


def test_append_strided_rows_of_a_fused_projection_and_many_rows():
    """K and V as column blocks of one [rows, (NQ + 2 NKV) HD] projection; enough rows for the windowed form."""
    rng = np.random.default_rng(8)
    page, NKV, HD, NQ = 16, 8, 128, 16
    lens = [700, 1, 513, 64, 900]
    rows, P = sum(lens), sum(-(-n // page) for n in lens)
    table = R.tables(rng, lens, page, P)
    slots = np.concatenate([[table[b, j // page] * page + j % page for j in range(n)] for b, n in enumerate(lens)])
    assert rows * NKV > 16384
    qkv = torch.from_numpy(rng.standard_normal((rows, (NQ + 2 * NKV) * HD))).to(torch.bfloat16).cuda()
    k = qkv[:, NQ * HD:(NQ + NKV) * HD].unflatten(1, (NKV, HD))
    v = qkv[:, (NQ + NKV) * HD:].unflatten(1, (NKV, HD))
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    R.append(K, V, Ks, Vs, k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
    A.kv8_append(k, v, cache, i32(slots))
    same_cache(cache, K, V, Ks, Vs)


@pytest.mark.parametrize("B,NKV,top", [(700, 8, 1), (900, 8, 3), (900, 16, 5), (9000, 4, 1)])
def test_append_of_many_short_runs(B, NKV, top):
    """Windows of 4 and 16 rows that hold many runs each: requests of a few tokens, some behind others of their page."""
    rng = np.random.default_rng(B)
    page, HD = 16, 128
    have, add = rng.integers(0, page - top, B), rng.integers(1, top + 1, B)
    K, V, Ks, Vs = R.make_cache(rng, B, page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    slots = np.concatenate([p * page + h + np.arange(n) for p, h, n in zip(rng.permutation(B), have, add)])
    slots = np.insert(slots, rng.integers(0, len(slots), len(slots) // 10), -1)
    assert len(slots) * NKV > 4096
    kt, k = values(rng, len(slots), NKV, HD, "bf16", 3.0)
    vt, v = values(rng, len(slots), NKV, HD, "bf16", 0.1)
    A.kv8_append(kt, vt, cache, i32(slots))
    R.append(K, V, Ks, Vs, k, v, slots)
    same_cache(cache, K, V, Ks, Vs)


@pytest.mark.parametrize("page", [16, 64])
def test_append_with_skipped_rows_between_a_pages_rows(page):
    """Rows of one page with up to 32 skipped ones between them (drafts that were not accepted), in windows of 1, 4 and 16 rows:
    one run, so the scale is the least that holds all of them and every code is rounded once."""
    rng = np.random.default_rng(page)
    for NKV, runs in ((1, 6), (2, 60), (16, 150)):
        HD, slots = 128, []
        for pid in rng.permutation(runs):
            off = int(rng.integers(0, page))
            n = int(rng.integers(1, page - off + 1))
            rows = np.full(n + int(rng.integers(0, 33)), -1)
            at = np.sort(rng.choice(len(rows) - 2, n - 2, replace=False) + 1) if n > 2 else np.array([], int)
            at = np.concatenate([[0], at, [len(rows) - 1]])[:n] if n > 1 else np.array([0])
            rows[at] = pid * page + off + np.arange(n)
            rows[rows < 0] = rng.choice([-1, runs * page, 1 << 30], (rows < 0).sum())
            slots += list(rows) + [-5] * int(rng.integers(0, 70) if rng.random() < 0.2 else 0)
        K, V, Ks, Vs = R.make_cache(rng, runs, page, NKV, HD)
        cache = R.to_cache(A, K, V, Ks, Vs)
        kt, k = values(rng, len(slots), NKV, HD, "f16", 2.0)
        scale = torch.from_numpy(2.0 ** rng.integers(-3, 4, len(slots))).to(kt).view(-1, 1, 1)
        kt = kt * scale
        A.kv8_append(kt, kt, cache, i32(slots))
        k = kt.double().cpu().numpy()
        R.append(K, V, Ks, Vs, k, k, slots)
        same_cache(cache, K, V, Ks, Vs, f"{NKV} heads, {len(slots)} rows")


# ---------------------------------------------------------------- attention
HEADS = {"q6": (24, 4, 256), "g2": (4, 2, 256), "g16": (16, 1, 512), "s4": (8, 2, 128), "g1": (2, 2, 128), "g5": (5, 1, 512), "g3": (6, 2, 128),
         "g20": (20, 1, 256), "g96": (96, 1, 128), "g130": (130, 1, 256)}


def attn_case(seed, heads, page, io, ctx, add, window=0, tree=False, chunk=0, out=None, spread=2, uniform=False, scale=0.0, hurt=None,
              max_pos=None, T=None):
    """One call against the 64-bit form, with NaN codes in every token that is nobody's."""
    NQ, NKV, HD = HEADS[heads]
    rng = np.random.default_rng(seed)
    ctx, add = np.array(ctx), np.array(add)
    lens = np.where(add > 0, ctx + add, np.maximum(ctx, 0))
    P = int(sum(-(-int(max(n, 0)) // page) for n in lens)) + 2
    table = R.tables(rng, np.maximum(lens, 0), page, P, int(-(-max(lens.max(), 1) // page)) + 1)
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD, spread)
    R.blank_tail(K, V, table, np.maximum(lens, 0), page)
    if hurt:
        hurt(K, V, Ks, Vs, table)
    cu = np.concatenate([[0], np.cumsum(add)])
    rows = int(cu[-1]) if uniform else int(cu[-1]) + 3
    dt = R.DTYPES[io]
    Qt = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).to(dt)
    anc = None
    if tree:
        anc = np.array([rng.integers(0, 1 << 32) if (r % 5 == 4) else int(rng.integers(0, 1 << 32)) | (1 << max(0, r - int(cu[np.searchsorted(cu, r, "right") - 1]) if r < cu[-1] else 0))
                        for r in range(rows)], np.uint64) & np.uint64(0xFFFFFFFF)
    O = torch.full((rows, NQ, HD), 77.0, dtype=R.DTYPES[out] if out else dt, device="cuda")
    lse = torch.full((rows, NQ), 77.0, device="cuda")
    cache = R.to_cache(A, K, V, Ks, Vs)
    T = int(add.max()) if T is None else T
    mp = int(max((ctx + add).max() - 1, 0)) if max_pos is None else max_pos
    tb = np.full((len(ctx), max(table.shape[1], mp // page + 1) + 1), -1)
    tb[:, :table.shape[1]] = table
    dev_anc = None if anc is None else torch.from_numpy(anc.astype(np.uint32).view(np.int32)).cuda()
    A.attn_kv8(Qt.cuda(), cache, i32(tb), i32(ctx), O, T, mp, cu=None if uniform else i32(cu), anc=dev_anc, chunk=chunk, window=window,
               lse=lse, scale=scale)
    torch.cuda.synchronize()
    assert bool((O[int(cu[-1]):] == 77).all()) and bool((lse[int(cu[-1]):] == 77).all()), "rows behind the last request were written"
    ref = R.attention(Qt.double().numpy(), K, V, Ks, Vs, table, ctx, cu, scale=scale, window=window, anc=anc)
    R.check(O, lse, ref, f"{heads} page {page} {io}")
    return O, lse


@pytest.mark.parametrize("heads", ["q6", "g2", "g16", "s4", "g1", "g5"])
@pytest.mark.parametrize("page,io", [(16, "f16"), (32, "bf16"), (64, "f16"), (64, "bf16")])
def test_single_tokens(heads, page, io):
    attn_case(1, heads, page, io, [0, 1, 14, 15, 16, 62, 63, 64, 200, 255, 256, 700], [1] * 12)


@pytest.mark.parametrize("heads,window", [("q6", 1), ("g2", 16), ("s4", 100), ("g16", 64), ("g2", 1000), ("g1", 65)])
def test_single_tokens_in_a_window(heads, window):
    attn_case(2, heads, 16, "bf16", [0, 63, 64, 130, 400, 901], [1] * 6, window=window, uniform=True)


@pytest.mark.parametrize("chunk", [64, 128, 192, 256, 512, 1024])
@pytest.mark.parametrize("heads", ["q6", "g16"])
def test_chunks(chunk, heads):
    attn_case(3, heads, 32, "f16", [0, 300, 63, 1025, 640], [1] * 5, chunk=chunk)


@pytest.mark.parametrize("heads,add", [("q6", [8] * 4), ("q6", [2, 1, 0, 5]), ("g2", [32, 7, 1, 16]), ("g2", [8, 8, 1, 3]), ("s4", [16, 1, 0, 9]),
                                       ("g16", [4, 2, 0, 3]), ("g16", [8, 1, 1, 5]), ("g5", [7, 3, 1, 2]), ("g3", [21, 20, 4, 0]), ("g20", [3, 1, 2, 3])])
@pytest.mark.parametrize("tree", [False, True])
def test_short_runs_and_trees(heads, add, tree):
    attn_case(4, heads, 64 if heads == "q6" else 16, "f16" if tree else "bf16", [0, 70, 33, 500], add, tree=tree, chunk=128)
    attn_case(5, heads, 32, "bf16", [63, 1, 0, 257], add, tree=tree, window=0 if tree else 50)


@pytest.mark.parametrize("heads,io,page,add", [("q6", "f16", 64, [77]), ("g2", "bf16", 64, [130, 33, 1, 64]), ("g2", "f16", 16, [300]), ("s4", "f16", 32, [65, 17, 200]),
                                               ("g16", "bf16", 64, [40, 9]), ("g5", "f16", 16, [90]), ("g1", "bf16", 16, [257, 128, 0, 5]), ("g3", "f16", 64, [150, 1])])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_prompts(heads, io, page, add, window):
    rng = np.random.default_rng(len(add))
    attn_case(6, heads, page, io, rng.integers(0, 150, len(add)), add, window=window)
    if window == 0:
        attn_case(7, heads, page, io, [0] * len(add), add)
        attn_case(8, heads, page, io, [190] * len(add), add, chunk=64, out="fp32")


# Sizes from which a call takes each tile (see kv8_choose): (heads, page, ctx, add, window), checked against the rule.
FORMS = {
    "128 rows, HD 256": ("q6", 64, [0, 30, 500], [800, 1111, 1500], 0),
    "128 rows, HD 256, window": ("g2x8", 16, [40], [4001], 300),
    "128 rows, HD 128": ("s4", 32, [5, 0, 64] * 9, [1200, 400, 333] * 9, 0),
    "64 rows, HD 256": ("g2x8", 64, [7], [1800], 0),
    "64 rows, HD 128, window": ("s4", 16, [100, 0], [3100, 3500], 500),
    "64 rows, HD 512": ("g16", 64, [3, 0, 77], [600, 601, 512], 0),
    "split, 64-row groups": ("q6", 64, [3000, 2500], [64, 33], 0),
    "split, 32-row groups, HD 512": ("g16", 16, [3000, 1], [100, 65], 0),
    "32-row groups, unsplit": ("g2x8", 32, [900], [1000], 0),
    "16-row groups, unsplit": ("q6", 16, [0, 100, 3], [150, 20, 1], 0),
}


@pytest.mark.parametrize("form", FORMS)
def test_every_form_of_prompts(form):
    """Rows of the last tiles, of tile and request borders and some between, of larger calls: each against its 64-bit value."""
    heads, page, ctx, add, window = FORMS[form]
    NQ, NKV, HD = dict(HEADS, g2x8=(16, 8, 256))[heads]
    rng = np.random.default_rng(len(form))
    ctx, add = np.array(ctx), np.array(add)
    lens = ctx + add
    P = int((-(-lens // page)).sum()) + 1
    table = R.tables(rng, lens, page, P)
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    R.blank_tail(K, V, table, lens, page)
    cu = np.concatenate([[0], np.cumsum(add)])
    rows = int(cu[-1])
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).to(torch.bfloat16)
    O, lse = torch.full((rows + 1, NQ, HD), 77.0, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, NQ, device="cuda")
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(table), i32(ctx), O[:rows], int(add.max()), int(lens.max()) - 1, cu=i32(cu),
               window=window, lse=lse)
    torch.cuda.synchronize()
    assert bool((O[rows] == 77).all()) and not bool((O[:rows] == 77).all(-1).any()) and bool(torch.isfinite(O.float()).all())
    G = NQ // NKV
    edges = {t * 64 // G + d for t in range(0, rows * G // 64 + 1, max(1, rows * G // 64 // 6)) for d in (-1, 0)}
    some = sorted({int(r) for b in range(len(add)) for r in (cu[b], cu[b + 1] - 1)} | {int(r) for r in rng.integers(0, rows, 12)} |
                  {r for r in edges if 0 <= r < rows})
    seq = np.searchsorted(cu, some, side="right") - 1
    for r, b in zip(some, seq):
        one = R.attention(Q[r:r + 1].double().numpy(), K, V, Ks, Vs, table[b:b + 1], [int(ctx[b] + r - cu[b])], np.array([0, 1]), window=window)
        R.check(O[r:r + 1], lse[r:r + 1], one, f"{form}, row {r}")


@pytest.mark.parametrize("heads,add", [("g96", [1, 1]), ("g130", [1, 0, 1]), ("g96", [5, 3]), ("g130", [7, 32]), ("g96", [150, 110]), ("g130", [3, 190])])
def test_more_heads_than_a_tiles_rows(heads, add):
    """Groups of 96 and 130 q-heads: a token's rows lie in several tiles, in every form."""
    ctx = [130, 7, 61][:len(add)]
    attn_case(26, heads, 16, "f16", ctx, add)
    attn_case(27, heads, 64, "bf16", ctx, add, window=70)
    if max(add) <= 32:
        attn_case(28, heads, 32, "bf16", ctx, add, tree=True, chunk=64)


def test_prompts_of_many_requests():
    """More requests than lanes, some empty, in every form: the order of tiles and items."""
    rng = np.random.default_rng(9)
    attn_case(9, "s4", 16, "f16", rng.integers(0, 90, 70), rng.integers(0, 4, 70))
    attn_case(10, "g2", 64, "bf16", [0, 30] * 9, [129, 200] * 9)
    add = rng.integers(0, 60, 130)
    add[3] = 80
    attn_case(11, "g1", 16, "bf16", rng.integers(0, 90, 130), add, window=70)
    attn_case(12, "s4", 16, "f16", [5, 0, 64] * 11, [90, 33, 64] * 11, window=70)


@pytest.mark.parametrize("heads,B,T", [("q6", 8, 8), ("s4", 30, 5), ("g16", 9, 4)])
def test_merge_of_many_rows(heads, B, T):
    """Enough rows for the merge by waves; requests without keys in some splits, and without rows."""
    rng = np.random.default_rng(B)
    ctx, add = rng.integers(0, 400, B), rng.integers(0, T + 1, B)
    add[0] = T
    assert B * T * HEADS[heads][0] * max(1, HEADS[heads][2] // 256) >= 1024  # a unit is a row and head of up to 256 dims
    attn_case(13, heads, 32, "f16", ctx, add, chunk=64)
    attn_case(14, heads, 16, "bf16", ctx, add, chunk=128, window=90, out="fp32")
    attn_case(15, heads, 16, "bf16", ctx, add, chunk=64, tree=True)


@pytest.mark.parametrize("io,out", [("f16", "f16"), ("f16", "bf16"), ("f16", "fp32"), ("bf16", "f16"), ("bf16", "fp32")])
@pytest.mark.parametrize("add", [[1, 1], [70, 90]])
def test_types_and_a_scale_of_the_callers(io, out, add):
    attn_case(11, "s4", 32, io, [100, 3], add, out=out, scale=0.31)


@pytest.mark.parametrize("add", [[1, 1, 1], [6, 3, 1], [80, 70, 1]])
def test_scales_far_apart(add):
    """Pages whose scales differ by 2^30: the small ones' values are as exact as the large ones'."""
    def hurt(K, V, Ks, Vs, table):
        Vs[:] = (2.0 ** (np.arange(Vs.size).reshape(Vs.shape) % 3 * 15.0 - 25.0)).astype(np.float32)
        Ks[::2] = 2.0 ** -9
    attn_case(12, "s4", 16, "f16", [140, 90, 31], add, hurt=hurt, out="fp32")


@pytest.mark.parametrize("add", [[1, 1, 1], [5, 2, 1], [90, 70, 3]])
@pytest.mark.parametrize("heads", ["g2", "s4"])
def test_nan_tokens_reach_the_rows_that_attend_them_and_no_other(add, heads):
    """K codes NaN in token 60 of request 0, in the last token of request 1 and in token 0 of request 2 (behind the window of
    every row but the first ones)."""
    def hurt(K, V, Ks, Vs, table):
        last = 40 + add[1] - 1
        K[table[0, 60 // 32], :, 60 % 32] = 0x7F
        K[table[1, last // 32], 0, last % 32] = 0xFF
        K[table[2, 0], 1, 0] = 0x7F
    O, lse = attn_case(13, heads, 32, "f16", [58, 40, 3], add, window=40, hurt=hurt)


@pytest.mark.parametrize("add", [[1, 1, 1], [4, 4, 2], [100, 66, 1]])
def test_pages_outside_the_pool_are_not_attended(add):
    """Entries -1 and >= pages: a gap, every page of a request (O = 0, lse = -inf), pages behind the window."""
    def hurt(K, V, Ks, Vs, table):
        table[0, 1] = -1
        table[0, 3] = K.shape[0]
        table[1, :] = 1 << 30
        table[2, :2] = -5
    attn_case(14, "s4", 16, "bf16", [100, 50, 200], add, hurt=hurt)
    attn_case(15, "g2", 16, "bf16", [100, 50, 200], add, hurt=hurt, window=64)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 0.0, -1.0])
@pytest.mark.parametrize("add", [[1, 1, 1], [4, 4, 2], [100, 66, 1], [900, 1200, 1100]])
def test_scales_of_pages_without_tokens_may_be_anything(add, scale):
    """Scales that nobody has written, in pages that no row attends: those of nobody, page 0 in place of entries outside the
    pool, and stale table entries behind the requests' last pages."""
    def hurt(K, V, Ks, Vs, table):
        spare = np.setdiff1d(np.arange(K.shape[0]), table)
        if not (spare == 0).any():                                   # page 0 becomes a spare one
            for x in (K, V, Ks, Vs):
                x[spare[0]] = x[0]
            table[table == 0] = spare[0]
            spare[0] = 0
        Ks[spare], Vs[spare] = scale, scale
        K[spare], V[spare] = 0x7F, 0x7F
        for b, n in enumerate(lens):
            table[b, -(-n // 16):] = spare[-1]
        table[0, 1] = -1
        table[2, :3] = K.shape[0] + 7
    ctx = [100, 50, 200]
    lens = [c + a for c, a in zip(ctx, add)]
    attn_case(23, "s4", 16, "bf16", ctx, add, hurt=hurt)
    attn_case(24, "g2", 16, "f16", ctx, add, hurt=hurt)


@pytest.mark.parametrize("ctx,add", [([-3, 5, -1], [1, 1, 1]), ([-3, 5, -1], [6, 2, 1]), ([-9, 5], [90, 70])])
def test_rows_without_keys(ctx, add):
    """Positions below zero attend nothing and are written as such; requests without rows are not touched."""
    attn_case(16, "g2", 16, "f16", ctx, add)
    attn_case(17, "g2", 16, "f16", ctx, add, chunk=64, max_pos=200)


def test_trees_that_hide_every_token():
    """Ancestor masks of zero over an empty cache: no key is left."""
    NQ, NKV, HD = HEADS["s4"]
    rng = np.random.default_rng(1)
    K, V, Ks, Vs = R.make_cache(rng, 2, 16, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    Q = torch.randn(4, NQ, HD, device="cuda").half()
    O, lse = torch.ones_like(Q), torch.zeros(4, NQ, device="cuda")
    A.attn_kv8(Q, cache, i32([[0], [1]]), i32([0, 0]), O, 2, 1, anc=i32([0, 2, 1, 0]), lse=lse)
    assert bool((O[[0, 3]] == 0).all()) and bool(torch.isneginf(lse[[0, 3]]).all()) and bool(torch.isfinite(lse[[1, 2]]).all())
    table = np.array([[0], [1]])
    R.check(O, lse, R.attention(Q.double().cpu().numpy(), K, V, Ks, Vs, table, [0, 0], np.array([0, 2, 4]), anc=[0, 2, 1, 0]))


def test_infinite_queries_stay_in_their_rows():
    NQ, NKV, HD = HEADS["g2"]
    rng = np.random.default_rng(2)
    for T in (3, 60):
        K, V, Ks, Vs = R.make_cache(rng, 8, 32, NKV, HD)
        cache = R.to_cache(A, K, V, Ks, Vs)
        Q = torch.randn(T, NQ, HD, device="cuda").half()
        P = Q.clone()
        P[1, 2, 5] = float("inf")
        P[T - 1, 0] = float("nan")
        out = []
        for q in (Q, P):
            O = torch.empty_like(q)
            A.attn_kv8(q, cache, i32([[3, 1, 0, 5, 7, 2]]), i32([100]), O, T, 100 + T - 1)
            out.append(O)
        same = torch.ones(T, NQ, dtype=torch.bool, device="cuda")
        same[1, 2] = same[T - 1, 0] = False
        assert torch.equal(out[0][same], out[1][same]) and bool(torch.isnan(out[1][T - 1, 0]).all())


def test_a_rows_bits_do_not_depend_on_its_batch():
    """The same request alone and among others, at the same T, max_pos and chunk."""
    NQ, NKV, HD = HEADS["q6"]
    rng = np.random.default_rng(4)
    K, V, Ks, Vs = R.make_cache(rng, 120, 16, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    ctx, T = [400, 17, 600, 250], 5
    table = R.tables(rng, [n + T for n in ctx], 16, 120, 40)
    Q = torch.randn(4 * T, NQ, HD, device="cuda").to(torch.bfloat16)
    for chunk in (64, 256):
        O = torch.empty_like(Q)
        A.attn_kv8(Q, cache, i32(table), i32(ctx), O, T, 620, chunk=chunk)
        for b in range(4):
            one = torch.empty_like(Q[:T])
            A.attn_kv8(Q[b * T:(b + 1) * T].contiguous(), cache, i32(table[b:b + 1]), i32(ctx[b:b + 1]), one, T, 620, chunk=chunk)
            assert torch.equal(one, O[b * T:(b + 1) * T]), (chunk, b)


def test_cache_past_4_gib():
    """A pool whose last pages lie beyond 2^32 bytes."""
    NKV, HD, page = 4, 512, 64
    P = (1 << 32) // (NKV * HD * page) + 40
    K = torch.zeros(P, NKV, page, HD, dtype=torch.uint8, device="cuda")
    V = torch.zeros(P, NKV, HD, page, dtype=torch.uint8, device="cuda")
    Ks, Vs = torch.ones(P, NKV, device="cuda"), torch.ones(P, NKV, device="cuda")
    cache = A.KV8Cache(K.view(torch.float8_e4m3fn), V.view(torch.float8_e4m3fn), Ks, Vs)
    rng = np.random.default_rng(6)
    for T, NQ in ((150, 4), (66, 8)):
        ids = P - 1 - rng.permutation(30)[:3]
        slots = np.concatenate([ids[j // page] * page + [j % page] for j in range(T)])
        kt, k = values(rng, T, NKV, HD, "bf16")
        vt, v = values(rng, T, NKV, HD, "bf16")
        A.kv8_append(kt, vt, cache, i32(slots))
        sub = torch.from_numpy(ids).cuda()
        k8, v8, s8, t8 = (np.zeros((3, NKV, page, HD), np.uint8), np.zeros((3, NKV, HD, page), np.uint8), np.ones((3, NKV), np.float32), np.ones((3, NKV), np.float32))
        if T == 150:
            R.append(k8, v8, s8, t8, k, v, np.arange(T))
            assert np.array_equal(K[sub].cpu().numpy(), k8) and np.array_equal(V[sub].cpu().numpy(), v8)
        else:
            k8, v8, s8, t8 = K[sub].cpu().numpy(), V[sub].cpu().numpy(), Ks[sub].cpu().numpy(), Vs[sub].cpu().numpy()
        for rows in (T, 1):
            Q = torch.randn(rows, NQ, HD, device="cuda").to(torch.bfloat16)
            O = torch.empty_like(Q)
            A.attn_kv8(Q, cache, i32(ids[None]), i32([T - rows]), O, rows, T - 1)
            ref = R.attention(Q.double().cpu().numpy(), k8, v8, s8, t8, np.array([[0, 1, 2]]), [T - rows], np.array([0, rows]))
            R.check(O, None, ref, f"T {T} rows {rows}")


# ---------------------------------------------------------------- together
def test_a_serving_run_of_the_three_together():
    """Prompts, then single tokens, then a draft: tables, append and attention of each step from the lengths alone, and pages
    given back and taken again."""
    NQ, NKV, HD = HEADS["g2"]
    page, B, P = 16, 3, 40
    rng = np.random.default_rng(9)
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    cache.K.view(torch.uint8).fill_(0x7F)
    cache.V.view(torch.uint8).fill_(0x7F)
    K[:], V[:] = 0x7F, 0x7F
    table, tb = i32(np.full((B, 12), -1)), np.full((B, 12), -1)
    free, count = i32(rng.permutation(P)), i32([P])
    status = i32([0])
    ctx = np.zeros(B, int)
    ctx_d = i32(ctx)
    for adds in ([70, 5, 0], [1, 1, 33], [1, 1, 1], [1, 1, 1], [4, 4, 4]):
        adds = np.array(adds)
        rows = int(adds.sum()) + 2
        cu, slots = i32(np.zeros(B + 1)), i32(np.zeros(rows))
        want = ref_plan(ctx, adds, page, tb, free.cpu().numpy(), int(count[0]), rows)
        A.kv8_plan(ctx_d, i32(adds), page, table, free, count, count, cu, slots, status)
        kt, k = values(rng, rows, NKV, HD, "bf16")
        vt, v = values(rng, rows, NKV, HD, "bf16")
        A.kv8_append(kt, vt, cache, slots)
        Q = torch.randn(rows, NQ, HD, device="cuda").half()
        O = torch.full_like(Q, 3.0)
        mp = int((ctx + adds).max()) - 1
        A.attn_kv8(Q, cache, table, ctx_d, O, int(adds.max()), mp, cu=cu)
        tb = want[1]
        assert int(status[0]) == 0 and np.array_equal(table.cpu().numpy(), tb) and np.array_equal(slots.cpu().numpy(), want[3])
        R.append(K, V, Ks, Vs, k, v, want[3])
        same_cache(cache, K, V, Ks, Vs)
        R.check(O, None, R.attention(Q.double().cpu().numpy(), K, V, Ks, Vs, tb, ctx, want[2]), str(adds))
        ctx = ctx + adds
        ctx_d += i32(adds)
    # request 0 ends: its pages go back on the stack and request 1 starts anew in them
    mine = tb[0, :-(-ctx[0] // page)]
    n = int(count[0])
    free[n:n + len(mine)] = i32(mine)
    count += len(mine)
    ctx[0], tb[0] = 0, -1
    ctx_d, table = i32(ctx), i32(tb)
    adds = np.array([90, 0, 0])
    cu, slots = i32(np.zeros(B + 1)), i32(np.zeros(90))
    want = ref_plan(ctx, adds, page, tb, free.cpu().numpy(), int(count[0]), 90)
    A.kv8_plan(ctx_d, i32(adds), page, table, free, count, count, cu, slots, status)
    assert int(status[0]) == 0 and np.array_equal(table.cpu().numpy(), want[1]) and int(count[0]) == want[4]
    kt, k = values(rng, 90, NKV, HD, "f16", 0.01)
    A.kv8_append(kt, kt, cache, slots)
    R.append(K, V, Ks, Vs, k, k, want[3])
    same_cache(cache, K, V, Ks, Vs, "pages taken again")


def test_a_captured_step_replays_on_new_lengths():
    """plan (count in place), append and attention as one graph; every replay against the same calls made eagerly on a copy,
    with eager work between; a second graph with its own workspace replayed in between."""
    NQ, NKV, HD = HEADS["q6"]
    page, B, P, T = 16, 4, 200, 2
    rng = np.random.default_rng(12)
    arrays = R.make_cache(rng, P, page, NKV, HD)
    mp = 700

    class Side:
        def __init__(s):
            s.cache = R.to_cache(A, *arrays)
            s.table, s.free, s.count, s.status = i32(np.full((B, mp // page + 1), -1)), i32(np.arange(P)), i32([P]), i32([0])
            s.ctx, s.add, s.cu, s.slots = i32([0] * B), i32([0] * B), i32([0] * (B + 1)), i32([0] * (B * T))
            s.k, s.v = (torch.zeros(B * T, NKV, HD, device="cuda", dtype=torch.bfloat16) for _ in range(2))
            s.Q, s.O = (torch.zeros(B * T, NQ, HD, device="cuda", dtype=torch.float16) for _ in range(2))
            s.ws = torch.empty(A.attn_kv8_workspace(B, T, B * T, NQ, NKV, HD, mp, 128), dtype=torch.uint8, device="cuda")

        def step(s):
            A.kv8_plan(s.ctx, s.add, page, s.table, s.free, s.count, s.count, s.cu, s.slots, s.status)
            A.kv8_append(s.k, s.v, s.cache, s.slots)
            A.attn_kv8(s.Q, s.cache, s.table, s.ctx, s.O, T, mp, cu=s.cu, chunk=128, ws=s.ws)
            s.ctx.add_(s.add)

    a, b, c = Side(), Side(), Side()
    graphs = {}
    for s in (a, c):                       # warm up on nothing (add = 0), then capture
        s.step()
        torch.cuda.synchronize()
        graphs[s] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[s]):
            s.step()
    for i in range(6):
        add = rng.integers(0, T + 1, B) if i else np.full(B, T)
        fresh = torch.randn(3, B * T, NKV, HD, device="cuda")
        q = torch.randn(B * T, NQ, HD, device="cuda").half()
        for s in (a, b, c):
            s.add.copy_(i32(add))
            s.k.copy_(fresh[0] * (i + 1)); s.v.copy_(fresh[1]); s.Q.copy_(q)
            s.O.fill_(5.0)
        graphs[a].replay()
        graphs[c].replay()
        b.step()
        torch.cuda.synchronize()
        for s in (a, c):
            assert torch.equal(s.O, b.O) and torch.equal(s.table, b.table) and torch.equal(s.count, b.count), i
            assert np.array_equal(R.codes(s.cache.K), R.codes(b.cache.K)) and np.array_equal(R.codes(s.cache.V), R.codes(b.cache.V)), i
        if i == 2:                         # longer contexts: more than one chunk
            for s in (a, b, c):
                s.ctx.copy_(i32([0] * B)); s.add.copy_(i32([0] * B))
                s.count.fill_(P); s.table.fill_(-1)
                big = [300, 129, 5, 640]
                cu, slots = i32([0] * (B + 1)), i32([0] * sum(big))
                A.kv8_plan(s.ctx, i32(big), page, s.table, s.free, s.count, s.count, cu, slots, s.status)
                g = torch.Generator(device="cuda").manual_seed(3)
                kv = torch.randn(2, sum(big), NKV, HD, device="cuda", generator=g)
                A.kv8_append(kv[0], kv[1], s.cache, slots)
                s.ctx.add_(i32(big))


def test_captured_prompts():
    """A prompt of the tile kernel at HD 512 (dynamic LDS past 64 KB) and a split one, each captured and replayed on new lengths."""
    rng = np.random.default_rng(21)
    for heads, T, ctx, mp in (("g16", 1700, 0, 1699), ("q6", 64, 2000, 3000)):
        NQ, NKV, HD = HEADS[heads]
        K, V, Ks, Vs = R.make_cache(rng, mp // 64 + 3, 64, NKV, HD)
        cache = R.to_cache(A, K, V, Ks, Vs)
        table = i32(rng.permutation(mp // 64 + 3)[None])
        Q = torch.randn(T, NQ, HD, device="cuda").half()
        c, cu = i32([ctx]), i32([0, T])
        ws = torch.empty(A.attn_kv8_workspace(1, T, T, NQ, NKV, HD, mp), dtype=torch.uint8, device="cuda")
        O, E = torch.zeros_like(Q), torch.zeros_like(Q)
        A.attn_kv8(Q, cache, table, c, E, T, mp, cu=cu, ws=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            A.attn_kv8(Q, cache, table, c, O, T, mp, cu=cu, ws=ws)
        for n in (T, T - 5, 1, T // 2):
            cu.copy_(i32([0, n]))
            c.copy_(i32([ctx + T - n]))
            O.fill_(2.0), E.fill_(2.0)
            g.replay()
            A.attn_kv8(Q, cache, table, c, E, T, mp, cu=cu, ws=torch.empty_like(ws))
            torch.cuda.synchronize()
            assert torch.equal(O, E), (heads, n)


def test_tables_with_strided_rows():
    """A table whose rows lie further apart than their columns, in all three operators."""
    NQ, NKV, HD = HEADS["s4"]
    rng = np.random.default_rng(22)
    K, V, Ks, Vs = R.make_cache(rng, 20, 16, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    big = i32(np.full((3, 40), -9))
    table = big[:, 4:11]
    ctx, add = np.array([0, 0, 0]), np.array([40, 0, 100])
    cu, slots, n, status = i32([0] * 4), i32([0] * 140), i32([20]), i32([0])
    free = rng.permutation(20)
    A.kv8_plan(i32(ctx), i32(add), 16, table, i32(free), n, n, cu, slots, status)
    want = ref_plan(ctx, add, 16, np.full((3, 7), -9), free, 20, 140)
    assert int(status[0]) == 0 and np.array_equal(table.cpu().numpy(), want[1]) and np.array_equal(slots.cpu().numpy(), want[3])
    assert bool((big[:, :4] == -9).all()) and bool((big[:, 11:] == -9).all())
    kt, k = values(rng, 140, NKV, HD, "bf16")
    A.kv8_append(kt, kt, cache, slots)
    R.append(K, V, Ks, Vs, k, k, want[3])
    for T, rows_of in ((100, [40, 0, 100]), (1, [1, 0, 1])):
        q = np.array(rows_of)
        c = ctx + add - q
        off = np.concatenate([[0], np.cumsum(q)])
        Q = torch.randn(int(off[-1]), NQ, HD, device="cuda").half()
        O = torch.empty_like(Q)
        A.attn_kv8(Q, cache, table, i32(c), O, T, 99, cu=i32(off))
        R.check(O, None, R.attention(Q.double().cpu().numpy(), K, V, Ks, Vs, want[1], c, off), str(T))


def test_what_the_binding_refuses_on_the_gpu():
    NQ, NKV, HD = HEADS["s4"]
    cache = A.KV8Cache.empty(4, 16, NKV, HD)
    Q = torch.zeros(2, NQ, HD, device="cuda").half()
    t, c = i32([[0], [1]]), i32([3, 4])
    good = dict(Q=Q, cache=cache, table=t, ctx=c, O=torch.empty_like(Q), T=1, max_pos=10)
    A.attn_kv8(**good)
    for bad in (dict(max_pos=16), dict(O=torch.empty_like(Q)[:1]), dict(Q=Q.float()), dict(Q=Q.transpose(0, 1).contiguous().transpose(0, 1)),
                dict(table=t.long()), dict(table=t.expand(2, 3)), dict(ctx=c.float()), dict(cu=i32([0, 2])), dict(anc=i32([1])),
                dict(lse=torch.empty(2, NQ, device="cuda").half()), dict(ws=torch.empty(8, device="cuda")), dict(cu=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises((ValueError, A.HipError)):
            A.attn_kv8(**dict(good, **bad))
    k = torch.zeros(3, NKV, HD, device="cuda")
    s = i32([0, 1, 2])
    A.kv8_append(k, k, cache, s)
    for bad in ((k.double(), k.double(), s), (k, k.half(), s), (k[:2], k, s), (k, k, s.long()), (k[..., ::2], k, s),
                (torch.zeros(3, NKV, HD + 1, device="cuda")[..., 1:], k, s), (k[:1].expand(3, NKV, HD), k, s)):
        with pytest.raises((ValueError, A.HipError)):
            A.kv8_append(bad[0], bad[1], cache, bad[2])


def test_statistics_of_the_append():
    """G4_KV_STATS=1 counts what is not finite and the largest stored magnitudes, as the other stores do."""
    import os
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = ["dgx-serving_amd", "tests"]
import torch, dgx_attn as A
c = A.KV8Cache.empty(3, 16, 2, 128)
k, v = torch.ones(20, 2, 128, device="cuda") * 3.3, torch.ones(20, 2, 128, device="cuda")
k[4, 1, 9] = -100.3; k[2, 0, 0] = float("nan"); v[3, 1, 5] = float("inf"); v[17, 0, 7] = float("-inf"); v[19, 1, 127] = 7.7
A.kv8_append(k, v, c, torch.arange(20, dtype=torch.int32, device="cuda"))
torch.cuda.synchronize()
s = A.kv_stats()
f = lambda u: torch.tensor([u], dtype=torch.int64).to(torch.int32).view(torch.float32).item()
print(s[0], s[1], f(s[2]), f(s[3]))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, G4_KV_STATS="1"), cwd=root, capture_output=True, text=True, timeout=110)
    assert out.returncode == 0, out.stderr
    # 100.3 under 2^-2 is 401.2, nearest code 416: 104. 7.7 under 2^-5 (7.7 <= 448 / 32) is 246.4, nearest 240 (step 16): 7.5
    assert out.stdout.split() == ["1", "2", "104.0", "7.5"], out.stdout


def test_streams_with_their_own_workspaces():
    """Two calls at once on two streams."""
    NQ, NKV, HD = HEADS["q6"]
    rng = np.random.default_rng(13)
    K, V, Ks, Vs = R.make_cache(rng, 300, 16, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    ctx = [900, 300, 700, 1100]
    table = i32(R.tables(rng, [n + 1 for n in ctx], 16, 300, 70))
    Q = [torch.randn(4, NQ, HD, device="cuda").half() for _ in range(2)]
    want = []
    for q in Q:
        O = torch.empty_like(q)
        A.attn_kv8(q, cache, table, i32(ctx), O, 1, 1100, chunk=64)
        want.append(O)
    n = A.attn_kv8_workspace(4, 1, 4, NQ, NKV, HD, 1100, 64)
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in st]
    out = [torch.empty_like(q) for q in Q]
    c = i32(ctx)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                A.attn_kv8(Q[i], cache, table, c, out[i], 1, 1100, chunk=64, ws=ws[i])
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
