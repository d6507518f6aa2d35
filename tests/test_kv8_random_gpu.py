"""GPU tests of the paged 8-bit cache with calls drawn at random: single operators, and a serving loop that accepts some of its
drafts, gives pages back and takes them again; all against the plain forms (codes, scales, tables and slots exactly, attention
within its bounds)."""
import numpy as np
import pytest
import torch

import dgx_attn as A
import kv8_ref as R
from test_kv8_gpu import ref_plan, same_cache

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def heads_of(rng):
    HD = int(rng.choice([128, 256, 512]))
    NKV = int(rng.choice([1, 2, 3, 8, 20, 64]))
    G = int(rng.choice([1, 2, 3, 4, 6, 8, 16, 17]))
    while G * NKV > 256:
        G = (G + 1) // 2
    return NKV * G, NKV, HD


@pytest.mark.parametrize("seed", range(60))
def test_attention(seed):
    rng = np.random.default_rng(1000 + seed)
    NQ, NKV, HD = heads_of(rng)
    page, io, out = int(rng.choice([16, 32, 64])), str(rng.choice(["f16", "bf16"])), str(rng.choice(["f16", "bf16", "fp32"]))
    B = int(rng.choice([1, 2, 5, 17]))
    kind = rng.choice(["one", "run", "tree", "prompt", "prompt"])
    top = {"one": 1, "run": int(rng.integers(2, 40)), "tree": int(rng.integers(2, 33)), "prompt": int(rng.integers(40, 200))}[kind]
    if kind == "prompt":
        B = min(B, 3)
    add = rng.integers(0, top + 1, B) if kind != "one" else rng.integers(0, 2, B)
    add[int(rng.integers(0, B))] = top
    uniform = bool(rng.random() < 0.3)
    if uniform:
        add[:] = top
    ctx = np.minimum(np.exp(rng.uniform(0, np.log(1200), B)).astype(int) - int(rng.integers(0, 3)), 1200)
    window = int(rng.choice([0, 0, 1, 7, 64, 100, 300]))
    chunk = int(rng.choice([0, 0, 64, 128, 192, 512, 1024]))
    lens = np.maximum(np.where(add > 0, ctx + add, ctx), 0)
    mp = max(int((ctx + add).max()) - 1, 0) + int(rng.choice([0, 0, 1, 500]))
    P = int((-(-lens // page)).sum()) + 2
    table = R.tables(rng, lens, page, P, mp // page + 1)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD)
    R.blank_tail(K, V, table, lens, page)
    if rng.random() < 0.3:                                           # a page that was given back
        table[int(rng.integers(0, B)), 0] = -1
    cu = np.concatenate([[0], np.cumsum(add)])
    rows = int(cu[-1]) + (0 if uniform else int(rng.integers(0, 4)))
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).to(R.DTYPES[io])
    anc = rng.integers(0, 1 << 32, rows).astype(np.uint32) if kind == "tree" else None
    O, lse = torch.full((rows, NQ, HD), 77.0, dtype=R.DTYPES[out], device="cuda"), torch.full((rows, NQ), 77.0, device="cuda")
    more = int(rng.choice([0, 0, 3]))                                # T is a bound
    T = top if uniform else min(32, top + 1) if kind == "tree" else top + more
    n = A.attn_kv8_workspace(B, T, rows, NQ, NKV, HD, mp, chunk, window, kind == "tree")
    ws = torch.full((n + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    what = f"{kind} {NQ}/{NKV}x{HD} page {page} ctx {ctx.tolist()} add {add.tolist()} window {window} chunk {chunk} T {T} max_pos {mp}"
    print(what, A.attn_kv8_form(B, T, rows, NQ, NKV, HD, mp, chunk, window, kind == "tree"), flush=True)
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), i32(table), i32(ctx), O, T, mp, cu=None if uniform else i32(cu), chunk=chunk, window=window,
               lse=lse, ws=ws[:n], anc=None if anc is None else torch.from_numpy(anc.view(np.int32)).cuda())
    torch.cuda.synchronize()
    assert bool((ws[n:] == 0xFF).all())
    assert bool((O[int(cu[-1]):] == 77).all()) and bool((lse[int(cu[-1]):] == 77).all())
    R.check(O, lse, R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, table, ctx, cu, window=window, anc=anc), what)


@pytest.mark.parametrize("seed", range(24))
def test_append(seed):
    """Runs of any length and place, far apart in magnitude, with skipped rows in and between them, strided sources."""
    rng = np.random.default_rng(2000 + seed)
    NKV, HD, page = int(rng.choice([1, 2, 5, 24])), int(rng.choice([128, 256, 512])), int(rng.choice([16, 32, 64]))
    dtype, runs = str(rng.choice(["fp32", "f16", "bf16"])), int(rng.choice([1, 4, 30]))
    slots = []
    for pid in rng.permutation(runs):
        off = int(rng.integers(0, page)) if rng.random() < 0.7 else 0
        n = int(rng.integers(1, page - off + 1))
        seg = list(pid * page + off + np.arange(n))
        for _ in range(int(rng.integers(0, 9)) if rng.random() < 0.5 else 0):
            seg.insert(int(rng.integers(0, len(seg) + 1)), int(rng.choice([-1, runs * page, 2 ** 31 - 1, -2 ** 31])))
        slots += seg
    rows, pad = len(slots), int(rng.choice([0, 8, 64]))
    K, V, Ks, Vs = R.make_cache(rng, runs, page, NKV, HD, 8)
    cache = R.to_cache(A, K, V, Ks, Vs)
    mag = 2.0 ** rng.integers(-9, 9 if dtype == "f16" else 30, (rows, 1, 1)) if rng.random() < 0.5 else 1.0
    big = [torch.from_numpy(rng.standard_normal((rows, NKV, HD)) * mag).to(R.DTYPES[dtype]) for _ in range(2)]
    if rng.random() < 0.3:
        big[int(rng.integers(0, 2))][int(rng.integers(0, rows)), int(rng.integers(0, NKV)), int(rng.integers(0, HD))] = float(rng.choice([np.nan, np.inf, -np.inf]))
    dev = []
    for t in big:                                                    # rows of a wider buffer
        w = torch.full((rows, NKV * HD + pad), 3.0, dtype=t.dtype, device="cuda")
        w[:, :NKV * HD] = t.view(rows, -1).cuda()
        dev.append(w[:, :NKV * HD].unflatten(1, (NKV, HD)))
    A.kv8_append(*dev, cache, i32(np.array(slots, np.int64)))
    R.append(K, V, Ks, Vs, big[0].double().numpy(), big[1].double().numpy(), slots)
    same_cache(cache, K, V, Ks, Vs, f"seed {seed}")


@pytest.mark.parametrize("seed,page,heads,window", [(0, 16, (8, 2, 128), 0), (1, 32, (4, 2, 256), 40), (2, 16, (16, 1, 512), 0), (3, 64, (12, 2, 256), 100),
                                                    (4, 16, (6, 6, 128), 25), (5, 16, (24, 4, 256), 0)])
def test_a_serving_loop(seed, page, heads, window):
    """Steps of prompts, single tokens and draft trees over requests that come and go. After a step some of a request's drafts are
    accepted and appended again at consecutive places; the pages behind them, those behind the window and those of ended
    requests go back on the stack. The counts of free pages take turns."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(3000 + seed)
    B, P, most = 5, 60, 400
    cols = most // page + 3
    K, V, Ks, Vs = R.make_cache(rng, P, page, NKV, HD)
    K[:], V[:] = 0x7F, 0x7F
    cache = R.to_cache(A, K, V, Ks, Vs)
    ctx, tb = np.zeros(B, int), np.full((B, cols), -1)
    stack, count = rng.permutation(P), P
    table, free, counts, status = i32(tb), i32(stack), [i32([P]), i32([-1])], i32([-1])
    refused = 0
    for step in range(24):
        tree = bool(rng.random() < 0.4)
        adds = rng.integers(0, 9, B) if tree else np.where(rng.random(B) < 0.3, rng.integers(0, 120, B), rng.integers(0, 2, B))
        adds = np.minimum(adds, most - ctx)
        if adds.sum() == 0:
            adds[0] = 1
        rows = int(adds.sum()) + int(rng.integers(0, 5))
        want = ref_plan(ctx, adds, page, tb, stack, count, rows)
        cin, cout = counts[step % 2], counts[1 - step % 2]
        cu, slots, ctx_d = i32(np.full(B + 1, -3)), i32(np.full(rows, -3)), i32(ctx)
        A.kv8_plan(ctx_d, i32(adds), page, table, free, cin, cout, cu, slots, status)
        kv = [torch.from_numpy(rng.standard_normal((rows, NKV, HD)) * 2.0 ** rng.integers(-4, 5)).to(torch.bfloat16) for _ in range(2)]
        A.kv8_append(kv[0].cuda(), kv[1].cuda(), cache, slots)
        Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).half()
        O = torch.full((rows, NQ, HD), 9.0, dtype=torch.float16, device="cuda")
        anc = None
        if tree:                                                     # each token and some of those before it
            anc = np.array([rng.integers(0, 1 << 32) for _ in range(rows)], np.uint64)
            for b in range(B):
                for i in range(adds[b]):
                    anc[want[2][b] + i] |= np.uint64(1 << i)
        mp, T = int((ctx + adds).max()) - 1, int(adds.max())
        A.attn_kv8(Q.cuda(), cache, table, ctx_d, O, T, mp, cu=cu, window=window, chunk=64 if step % 3 == 0 else 0,
                   anc=None if anc is None else torch.from_numpy(anc.astype(np.uint32).view(np.int32)).cuda())
        torch.cuda.synchronize()
        got = (int(status[0]), table.cpu().numpy(), cu.cpu().numpy(), slots.cpu().numpy(), int(cout[0]))
        for g, w, name in zip(got, want, ("status", "table", "cu", "slots", "count")):
            assert np.array_equal(g, w), f"step {step}: {name}"
        tb, count = want[1], want[4]
        if want[0]:                                                  # too few pages: nothing was done
            refused += 1
            assert bool((O == 9).all())
            gone = int(np.argmax(ctx))
            kept = np.zeros(B, int)
        else:
            k, v = (x.double().numpy() for x in kv)
            R.append(K, V, Ks, Vs, k, v, want[3])
            same_cache(cache, K, V, Ks, Vs, f"step {step}")
            R.check(O, None, R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, tb, ctx, want[2], window=window, anc=anc), f"step {step}")
            kept, gone = adds.copy(), int(rng.integers(0, B)) if rng.random() < 0.15 else -1
            if tree:                                                 # accepted drafts: some of each request's, in their order
                again = np.full(rows, -1)
                for b in range(B):
                    if not adds[b]:
                        continue
                    kept[b] = int(rng.integers(1, adds[b] + 1))
                    path = np.sort(rng.choice(adds[b], kept[b], replace=False))
                    pos = ctx[b] + np.arange(kept[b])
                    again[want[2][b] + path] = tb[b, pos // page] * page + pos % page
                A.kv8_append(kv[0].cuda(), kv[1].cuda(), cache, i32(again))
                R.append(K, V, Ks, Vs, k, v, again)
                same_cache(cache, K, V, Ks, Vs, f"step {step}, accepted drafts")
        # Pages go back: behind the accepted tokens, behind the window, of a request that ends.
        back = []
        for b in range(B):
            had = -(-(ctx[b] + (0 if want[0] else adds[b])) // page)
            ctx[b] += kept[b]
            if b == gone:
                ctx[b] = 0
            need = -(-ctx[b] // page)
            back += [p for p in tb[b, need:had] if p >= 0]           # (their entries stay in the table)
            if window and ctx[b] > window:
                first = (ctx[b] - window + 1) // page                 # the next token's first page
                back += [p for p in tb[b, :first] if p >= 0]
                tb[b, :first] = -1
        stack = stack.copy()
        stack[count:count + len(back)] = back
        count += len(back)
        table, free = i32(tb), i32(stack)
        cout.fill_(count)
    assert count + sum(int((tb[b, :-(-ctx[b] // page)] >= 0).sum()) for b in range(B)) == P, "pages were lost"
