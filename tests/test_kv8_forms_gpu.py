"""GPU tests of the prompt tiles of the attention over the paged 8-bit cache: tiles of 64 and 128 rows, in one pass and in key
splits, each call with the form that it is meant for (dgx_attn_kv8_form) and against the 64-bit form of kv8_ref, whose bounds
hold per element."""
import numpy as np
import pytest
import torch

import dgx_attn as A
import kv8_ref as R

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def form_of(heads, ctx, add, rows, window=0, chunk=0, max_pos=None):
    NQ, NKV, HD = heads
    mp = int((np.array(ctx) + np.array(add)).max()) - 1 if max_pos is None else max_pos
    return A.attn_kv8_form(len(ctx), int(np.max(add)), rows, NQ, NKV, HD, mp, chunk, window)


def call(seed, heads, page, io, ctx, add, tile, split, window=0, chunk=0, out=None, scale=0.0, spread=2, hurt=None, max_pos=None,
         change_q=None):
    """One call of the given form (tile rows; in splits or not); NaN codes in every token that is nobody's."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(seed)
    ctx, add = np.array(ctx), np.array(add)
    lens = np.maximum(np.where(add > 0, ctx + add, ctx), 0)
    P = int((-(-lens // page)).sum()) + 2
    mp = int((ctx + add).max()) - 1 if max_pos is None else max_pos
    table = R.tables(rng, lens, page, P, max(int(-(-lens.max() // page)), mp // page + 1) + 1)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD, spread)
    R.blank_tail(K, V, table, lens, page)
    if hurt:
        hurt(K, V, Ks, Vs, table)
    cu = np.concatenate([[0], np.cumsum(add)])
    rows = int(cu[-1]) + 3
    got = form_of(heads, ctx, add, rows, window, chunk, mp)
    assert got[0] == tile and (got[3] > 1) == split, got
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).to(R.DTYPES[io])
    if change_q:
        change_q(Q)
    O = torch.full((rows, NQ, HD), 77.0, dtype=R.DTYPES[out or io], device="cuda")
    lse = torch.full((rows, NQ), 77.0, device="cuda")
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(table), i32(ctx), O, int(add.max()), mp, cu=i32(cu), chunk=chunk, window=window,
               lse=lse, scale=scale)
    torch.cuda.synchronize()
    assert bool((O[int(cu[-1]):] == 77).all()) and bool((lse[int(cu[-1]):] == 77).all()), "rows behind the last request were written"
    ref = R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, table, ctx, cu, scale=scale, window=window)
    R.check(O, lse, ref, f"{heads} page {page} {io}")
    return O, lse, cu


# heads, page, type, ctx, add, window, chunk, tile, split. Enough heads for few tokens to fill the chip.
CALLS = {
    "64, HD 128": ((128, 64, 128), 16, "f16", [0, 33, 5], [70, 65, 90], 0, 0, 64, False),
    "64, HD 128, window": ((96, 48, 128), 64, "bf16", [150, 0], [70, 90], 33, 0, 64, False),
    "64, HD 256, groups of 6": ((192, 32, 256), 64, "bf16", [0, 70, 3], [101, 64, 130], 0, 0, 64, False),
    "64, HD 256, window": ((64, 32, 256), 16, "f16", [150, 0, 9], [100, 90, 77], 40, 0, 64, False),
    "64, HD 512": ((96, 32, 512), 64, "f16", [40, 0, 130], [65, 90, 70], 0, 0, 64, False),
    "64, HD 512, window": ((64, 64, 512), 32, "bf16", [40, 0, 200], [130, 90, 70], 25, 0, 64, False),
    "128, HD 128": ((512, 128, 128), 64, "bf16", [10, 0, 77], [101, 65, 90], 0, 0, 128, False),
    "128, HD 128, window": ((384, 64, 128), 16, "f16", [150, 0], [99, 90], 65, 0, 128, False),
    "128, HD 256, groups of 6": ((384, 64, 256), 64, "f16", [0, 130, 3], [120, 101, 129], 0, 0, 128, False),
    "128, HD 256, window, groups of 5": ((320, 64, 256), 32, "bf16", [90, 0, 250], [70, 66, 90], 50, 0, 128, False),
    "64 in splits, HD 128": ((128, 64, 128), 16, "bf16", [100, 0], [100, 65], 0, 128, 64, True),
    "64 in splits, HD 128, window": ((64, 32, 128), 64, "f16", [300, 0, 40], [90, 65, 80], 70, 64, 64, True),
    "64 in splits, HD 256": ((64, 64, 256), 64, "f16", [260, 0, 64], [70, 80, 65], 0, 192, 64, True),
    "64 in splits, HD 256, window": ((32, 32, 256), 16, "bf16", [260, 3], [130, 131], 100, 64, 64, True),
    "64 in splits, HD 512": ((32, 32, 512), 32, "bf16", [200, 0, 90], [190, 130, 180], 0, 64, 64, True),
    "64 in splits, HD 512, window": ((128, 64, 512), 64, "f16", [270, 0], [66, 90], 70, 128, 64, True),
    "128 in splits, HD 128": ((128, 64, 128), 32, "f16", [200, 0, 64], [100, 130, 65], 0, 64, 128, True),
    "128 in splits, HD 128, window": ((192, 64, 128), 16, "bf16", [330, 10], [130, 99], 120, 64, 128, True),
    "128 in splits, HD 256, groups of 6": ((192, 32, 256), 64, "bf16", [300, 0, 70], [100, 81, 129], 0, 128, 128, True),
    "128 in splits, HD 256, window": ((192, 64, 256), 64, "f16", [400, 2], [130, 90], 64, 64, 128, True),
}


@pytest.mark.parametrize("name", CALLS)
def test_prompt_tiles(name):
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS[name]
    call(1, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk)


@pytest.mark.parametrize("name", CALLS)
def test_prompt_tiles_of_other_types_and_a_scale_of_the_callers(name):
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS[name]
    call(2, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk, out="fp32", scale=0.11)


@pytest.mark.parametrize("G", [96, 130])
@pytest.mark.parametrize("window,chunk", [(0, 0), (40, 0), (0, 64), (70, 64)])
def test_tiles_of_fewer_rows_than_a_token_has(G, window, chunk):
    """Groups of 96 and 130 q-heads in 128-row tiles: a token's rows lie in one or two of them."""
    NKV = 16 if G == 96 else 12
    call(3, (G * NKV, NKV, 128), 16, "bf16", [50, 0], [66, 20] if chunk or window else [66, 30], 128, chunk > 0, window=window, chunk=chunk)


@pytest.mark.parametrize("name", ["64, HD 128", "64, HD 512", "128, HD 256, groups of 6", "64 in splits, HD 256, window", "128 in splits, HD 128",
                                  "64 in splits, HD 512"])
def test_nan_tokens_in_tiles(name):
    """NaN codes in K of a token in the middle, of the last token, and of a token behind some rows' windows: NaN in the rows that
    attend them and in no other."""
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS[name]

    def hurt(K, V, Ks, Vs, table):
        last = ctx[1] + add[1] - 1
        K[table[0, 60 // page], ::2, 60 % page] = 0x7F
        K[table[1, last // page], 0, last % page] = 0xFF
        if len(ctx) > 2:
            K[table[2, 0], 1, 0] = 0x7F
    O, lse, cu = call(4, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk, hurt=hurt)
    assert bool(torch.isnan(O[:int(cu[-1])].float()).any()) and not bool(torch.isnan(O[:int(cu[-1])].float()).all())


@pytest.mark.parametrize("name", ["64, HD 256, window", "64, HD 512", "128, HD 128", "64 in splits, HD 128", "128 in splits, HD 256, window",
                                  "64 in splits, HD 512, window"])
def test_tiles_with_rows_that_attend_nothing(name):
    """Positions below zero, a request all of whose pages lie outside the pool, and a gap in another's: O = 0 and lse = -inf for
    rows without a key."""
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS[name]
    ctx, add = list(ctx) + [-7, 20], list(add) + [30, 40]

    def hurt(K, V, Ks, Vs, table):
        table[-1, :] = 1 << 30
        table[0, 1] = -1
        table[0, 3] = K.shape[0]
    O, lse, cu = call(5, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk, hurt=hurt)
    n = int(cu[-3])
    assert bool((O[n:n + 7] == 0).all()) and bool(torch.isneginf(lse[n:n + 7]).all()) and bool(torch.isfinite(lse[n + 7:n + 30]).all())
    assert bool((O[n + 30:n + 70] == 0).all()) and bool(torch.isneginf(lse[n + 30:n + 70]).all())


@pytest.mark.parametrize("name", ["64, HD 128", "64, HD 512", "128, HD 128", "64 in splits, HD 256", "128 in splits, HD 128"])
def test_infinite_queries_stay_in_their_rows_of_a_tile(name):
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS[name]

    def spoil(Q):
        Q[1, 2, 5] = float("inf")
        Q[7, 0] = float("nan")
    a = call(6, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk)[0]
    same = torch.ones(a.shape[:2], dtype=torch.bool, device="cuda")
    same[1, 2] = same[7, 0] = False
    b = raw(6, heads, page, io, ctx, add, window, chunk, spoil)
    assert torch.equal(a[same], b[same]) and bool(torch.isnan(b[7, 0]).all())


def raw(seed, heads, page, io, ctx, add, window, chunk, change_q):
    """The call of call(), its inputs changed, without a check."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(seed)
    ctx, add = np.array(ctx), np.array(add)
    lens = ctx + add
    P = int((-(-lens // page)).sum()) + 2
    mp = int(lens.max()) - 1
    table = R.tables(rng, lens, page, P, max(int(-(-lens.max() // page)), mp // page + 1) + 1)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD)
    R.blank_tail(K, V, table, lens, page)
    cu = np.concatenate([[0], np.cumsum(add)])
    Q = torch.from_numpy(rng.standard_normal((int(cu[-1]) + 3, NQ, HD))).to(R.DTYPES[io])
    change_q(Q)
    O = torch.full(Q.shape, 77.0, dtype=Q.dtype, device="cuda")
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(table), i32(ctx), O, int(add.max()), mp, cu=i32(cu), chunk=chunk, window=window)
    return O


# Rows that attend pages of small scales only, beside rows of large ones: 2^40 between them, so nothing of the large ones may
# reach their sums, and the bound is that of the small values.
SMALL = {
    "single tokens": ((12, 2, 256), 16, "f16", [100, 90, 130], [1, 1, 1], 0, 0, 0, False),
    "single tokens in splits": ((8, 2, 128), 16, "bf16", [200, 190, 230], [1, 1, 1], 0, 64, 0, True),
    "short runs in a window": ((4, 2, 128), 16, "f16", [40, 90], [32, 32], 8, 0, 0, False),
    "short runs in a window, splits": ((16, 1, 512), 16, "f16", [40, 90], [8, 8], 8, 64, 0, True),
    "prompts in groups of rows": ((8, 2, 256), 16, "bf16", [0, 90], [90, 70], 8, 0, 0, False),
    "64-row tiles": ((96, 48, 128), 16, "f16", [0, 90], [90, 70], 8, 0, 64, False),
    "64-row tiles, HD 512": ((64, 64, 512), 16, "bf16", [40, 0, 200], [130, 90, 70], 8, 0, 64, False),
    "64-row tiles in splits": ((64, 32, 256), 16, "f16", [120, 0, 40], [90, 65, 80], 8, 64, 64, True),
    "128-row tiles": ((384, 64, 128), 16, "f16", [150, 0], [99, 90], 8, 0, 128, False),
    "128-row tiles in splits": ((192, 32, 256), 16, "bf16", [200, 0, 70], [130, 110, 129], 8, 64, 128, True),
}


@pytest.mark.parametrize("name", SMALL)
def test_small_scales_beside_large_ones(name):
    heads, page, io, ctx, add, window, chunk, tile, split = SMALL[name]
    small = np.float32(2.0 ** -30)

    def hurt(K, V, Ks, Vs, table):
        Ks[:] = 2.0 ** -8
        Vs[:] = 2.0 ** 10
        if window:                                                   # every other page: windows of 8 keys lie in one or two
            for b in range(len(ctx)):
                ids = table[b, ::2]
                Vs[ids[ids >= 0]] = small
        else:                                                        # every other request
            for b in range(0, len(ctx), 2):
                Vs[table[b][table[b] >= 0]] = small
    O, lse, cu = call(7, heads, page, io, ctx, add, tile, split, window=window, chunk=chunk, hurt=hurt, out="fp32")
    pos = np.concatenate([c + np.arange(a) for c, a in zip(ctx, add)])
    if window:
        # every key of the window in one page of an even column
        only = torch.from_numpy((pos // page == np.maximum(pos - window + 1, 0) // page) & (pos // page % 2 == 0))
    else:
        only = torch.from_numpy(np.repeat(np.arange(len(ctx)) % 2 == 0, add))
    top = O[:int(cu[-1])].abs().amax(dim=(1, 2)).cpu()
    assert int(only.sum()) > 1 and bool((top[only] <= 448 * float(small)).all()) and bool((top[only] > float(small)).all())
    assert bool((top[~only] > 1e-3).all())


def test_captured_tiles_in_splits():
    """128-row tiles in key splits, captured at the largest sizes and replayed on other lengths, against the same call made eagerly."""
    heads, page, io, ctx, add, window, chunk, tile, split = CALLS["128 in splits, HD 256, window"]
    NQ, NKV, HD = heads
    rng = np.random.default_rng(8)
    B, T, mp = 2, max(add), 531
    rows = B * T
    assert form_of(heads, ctx, [T, T], rows, window, chunk, mp)[0] == 128
    K, V, Ks, Vs = R.make_cache_fast(rng, 2 * (mp // page + 1), page, NKV, HD)
    cache = R.to_cache(A, K, V, Ks, Vs)
    table = i32(rng.permutation(2 * (mp // page + 1)).reshape(2, -1))
    Q = torch.randn(rows, NQ, HD, device="cuda").half()
    c, cu = i32(ctx), i32([0, T, 2 * T])
    O, E = torch.zeros_like(Q), torch.zeros_like(Q)
    ws = torch.empty(A.attn_kv8_workspace(B, T, rows, NQ, NKV, HD, mp, chunk, window), dtype=torch.uint8, device="cuda")
    A.attn_kv8(Q, cache, table, c, E, T, mp, cu=cu, chunk=chunk, ws=ws, window=window)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.attn_kv8(Q, cache, table, c, O, T, mp, cu=cu, chunk=chunk, ws=ws, window=window)
    for lens, news in (([400, 2], [130, 90]), ([0, 0], [1, 130]), ([401, 300], [130, 0]), ([63, 64], [65, 64])):
        c.copy_(i32(lens)), cu.copy_(i32(np.concatenate([[0], np.cumsum(news)])))
        ws.fill_(0xFF)                                               # NaN in every partial
        O.fill_(2.0), E.fill_(2.0)
        g.replay()
        A.attn_kv8(Q, cache, table, c, E, T, mp, cu=cu, chunk=chunk, window=window)
        torch.cuda.synchronize()
        assert torch.equal(O, E), lens
        n = sum(news)
        ref = R.attention_rows(Q.double().cpu().numpy(), K, V, Ks, Vs, table.cpu().numpy(), lens, np.concatenate([[0], np.cumsum(news)]), window=window)
        R.check(O, None, ref, str(lens))
        assert bool((O[n:] == 2).all())


@pytest.mark.parametrize("heads,add", [((24, 4, 256), [8, 5, 1]), ((16, 1, 512), [4, 4, 2]), ((8, 2, 128), [32, 17, 9])])
@pytest.mark.parametrize("window,chunk", [(5, 0), (40, 64), (200, 128)])
def test_trees_behind_a_window(heads, add, window, chunk):
    """Ancestor masks and a window together: tokens of the window that the tree leaves."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(9)
    page, ctx = 16, np.array([0, 70, 300])
    add = np.array(add)
    lens, cu = ctx + add, np.concatenate([[0], np.cumsum(add)])
    P, rows = int((-(-lens // page)).sum()), int(cu[-1])
    table = R.tables(rng, lens, page, P)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD)
    anc = rng.integers(0, 1 << 32, rows).astype(np.uint32)
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).half()
    O, lse = torch.empty(rows, NQ, HD, device="cuda").half(), torch.empty(rows, NQ, device="cuda")
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(table), i32(ctx), O, int(add.max()), int(lens.max()) - 1, cu=i32(cu),
               anc=torch.from_numpy(anc.view(np.int32)).cuda(), chunk=chunk, window=window, lse=lse)
    R.check(O, lse, R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, table, ctx, cu, window=window, anc=anc), f"{heads}")


@pytest.mark.parametrize("heads,page,add,window,chunk,tile", [
    ((24, 4, 256), 64, [1, 1, 1, 1], 1000, 0, 0), ((16, 8, 256), 16, [1, 1, 1, 1], 65, 64, 0), ((16, 8, 256), 16, [1, 1, 1], 66, 64, 0),
    ((16, 1, 512), 32, [8, 3, 1, 8], 700, 0, 0), ((8, 2, 128), 16, [32, 9, 1, 0], 1, 64, 0), ((8, 2, 128), 16, [32, 32, 20, 5], 2, 64, 0),
    ((16, 4, 128), 16, [13, 8, 16], 128, 128, 0), ((12, 2, 256), 64, [90, 3, 77], 130, 64, 0), ((4, 2, 256), 32, [300], 600, 0, 0),
    ((64, 32, 128), 64, [90, 65, 80], 70, 64, 64), ((128, 64, 512), 64, [66, 90], 129, 128, 64), ((192, 64, 256), 64, [130, 90], 64, 64, 128)])
def test_splits_behind_a_window_far_from_the_first_key(heads, page, add, window, chunk, tile):
    """Positions around 10^5 and 10^7, of which only the pages that the window reaches exist, in a workspace of exactly the size
    that is asked for: results, and bytes behind the workspace."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(window + HD)
    add = np.array(add)
    B, T = len(add), int(add.max())
    cu = np.concatenate([[0], np.cumsum(add)])
    rows = int(cu[-1])
    near = rng.integers(window + 64, window + 400, B)                # positions within the pages that exist
    near[0] = -(-(window + 100) // 128) * 128 + window - 2            # first key one before a split's border
    lens = near + add
    P = int((-(-lens // page)).sum())
    table = R.tables(rng, lens, page, P)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD)
    R.blank_tail(K, V, table, lens, page)
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).half()
    for shift in (0, 102400, 1 << 24):                                # multiples of every page and of the splits below
        mp = int(lens.max()) - 1 + shift
        form = A.attn_kv8_form(B, T, rows, NQ, NKV, HD, mp, chunk, window)
        assert form[0] == tile and (form[3] > 1 or chunk == 0), form
        n = A.attn_kv8_workspace(B, T, rows, NQ, NKV, HD, mp, chunk, window)
        ws = torch.full((n + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
        t = np.full((B, mp // page + 1), -1, np.int32)
        t[:, shift // page:] = table[:, :t.shape[1] - shift // page]
        O, lse = torch.full((rows, NQ, HD), 77.0, dtype=torch.float16, device="cuda"), torch.empty(rows, NQ, device="cuda")
        A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(t), i32(near + shift), O, T, mp, cu=i32(cu), chunk=chunk, window=window, lse=lse,
                   ws=ws[:n])
        torch.cuda.synchronize()
        assert bool((ws[n:] == 0xFF).all()), "bytes behind the workspace were written"
        ref = R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, table, near, cu, window=window)
        R.check(O, lse, ref, f"shift {shift}")
