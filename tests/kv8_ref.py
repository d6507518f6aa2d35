"""Plain 64-bit (numpy, CPU) forms of the paged 8-bit cache's operators, and the tolerances that their tests use.

The format: e4m3 codes, a scale 2^e for each page and KV head, e the least integer in [-40, 40] with amax <= 448 * 2^e."""
import numpy as np
import torch

E_MIN, E_MAX = -40, 40
DTYPES = {"fp32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def decode_table():
    """Values of the 256 e4m3 codes."""
    c = np.arange(256)
    s, e, m = np.where(c & 128, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    return np.where((e == 15) & (m == 7), np.nan, s * v)


TABLE = decode_table()
POSITIVE = TABLE[:127]                       # 0 .. 448, ascending


def encode(x):
    """Nearest codes of finite float64 values, ties to the even code, magnitudes past 448 to 448."""
    a = np.minimum(np.abs(x), 448.0)
    hi = np.searchsorted(POSITIVE, a)        # first code whose value is >= a
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - POSITIVE[lo], POSITIVE[hi] - a
    up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))
    return (np.where(up, hi, lo) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def exponent(amax):
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def append(K, V, Ks, Vs, k, v, slots):
    """The append of rows k, v [rows, NKV, HD] (float64) on code arrays K [P, NKV, page, HD], V [P, NKV, HD, page] and scales,
    in place."""
    P, NKV, page, HD = K.shape
    slots = np.asarray(slots)
    taken = (slots >= 0) & (slots < P * page)
    k, v, slots = k[taken], v[taken], slots[taken]
    r = 0
    while r < len(slots):
        s = int(slots[r])
        n = 1
        while r + n < len(slots) and slots[r + n] == s + n and (s + n) % page:
            n += 1
        pid, off = s // page, s % page
        for h in range(NKV):
            kk, vv = k[r:r + n, h], v[r:r + n, h]
            bad = ~np.isfinite(kk).all(1) | ~np.isfinite(vv).all(1)
            for x, C, S, tr in ((kk, K, Ks, False), (vv, V, Vs, True)):
                fin = np.isfinite(x)
                amax = np.abs(x[fin]).max() if fin.any() else 0.0
                old = int(round(np.log2(float(S[pid, h])))) if off else E_MIN
                e = max(exponent(amax), old)
                page_codes = C[pid, h].T if tr else C[pid, h]          # [page, HD], a view
                if off and e > old:
                    held = page_codes[:off]
                    val = TABLE[held]
                    page_codes[:off] = np.where(np.isnan(val), held, encode(np.nan_to_num(val) * 2.0 ** (old - e)))
                codes = encode(np.where(fin, x, 0.0) / 2.0 ** e)
                if not tr:
                    codes[bad] = 0x7F
                page_codes[off:off + n] = codes
                S[pid, h] = 2.0 ** e
        r += n


def attention(Q, K, V, Ks, Vs, table, ctx, cu, scale=0.0, window=0, anc=None, rows=None):
    """(O, lse, bound): float64 results for rows Q [rows, NQ, HD], and for each output element the largest error of a kernel that
      * sums q.k and the weighted values in fp32: every score off by at most HD 2^-24 sum |q k| + 2^-22 |s|,
      * rounds the weights once to f16 (2^-11 of each), or to nothing below 2^-30 of the largest,
    before the output's own rounding. Rows outside every request are NaN in O and lse."""
    rows_n, NQ, HD = Q.shape
    P, NKV, page, _ = K.shape
    G = NQ // NKV
    sc = scale if scale > 0 else 1.0 / np.sqrt(HD)
    O, lse, tol = np.full(Q.shape, np.nan), np.full((rows_n, NQ), np.nan), np.zeros(Q.shape)
    lse_tol = np.zeros((rows_n, NQ))
    for b in range(len(ctx)):
        n0, n = int(ctx[b]), int(cu[b + 1] - cu[b])
        if n <= 0:
            continue
        L = n0 + n
        ids = np.array([table[b, j // page] for j in range(L)], np.int64) if L > 0 else np.zeros(0, np.int64)
        ok = (ids >= 0) & (ids < P)
        ids, off = np.where(ok, ids, 0), np.arange(max(L, 0)) % page
        for h in range(NKV):
            k = TABLE[K[ids, h, off]] * Ks[ids, h].astype(np.float64)[:, None]
            v = TABLE[V[ids, h, :, off]] * Vs[ids, h].astype(np.float64)[:, None]
            for i in range(n):
                r, pos = int(cu[b]) + i, n0 + i
                j = np.arange(max(L, 0))
                att = ok & (j <= pos)
                if window > 0:
                    att &= j > pos - window
                if anc is not None:
                    d = j - n0
                    att &= (d < 0) | ((int(anc[r]) >> np.clip(d, 0, 31)) & 1).astype(bool)
                for q in range(h * G, (h + 1) * G):
                    if not att.any():
                        O[r, q], lse[r, q] = 0.0, -np.inf
                        continue
                    ka, va = k[att], v[att]
                    s = ka @ Q[r, q] * sc
                    w = np.exp(s - s.max())
                    l = w.sum()
                    O[r, q] = (w / l) @ va
                    lse[r, q] = s.max() + np.log(l)
                    ds = (HD * 2.0 ** -24 * (np.abs(ka) @ np.abs(Q[r, q])) * abs(sc) + 2.0 ** -22 * np.abs(s)).max() + 2.0 ** -21
                    nk = att.sum()
                    rel = 2.0 ** -11 + 2 * ds + 2 * nk * 2.0 ** -24
                    tol[r, q] = rel * ((w / l) @ np.abs(va)) + nk * 2.0 ** -30 * np.abs(va).max()
                    lse_tol[r, q] = ds + nk * 2.0 ** -24 + 2.0 ** -22 * abs(lse[r, q]) + 2.0 ** -20
    return O, lse, tol, lse_tol


def check(out, lse, ref, what=""):
    """Kernel outputs (torch tensors, or lse None) against attention()'s."""
    O, L, tol, ltol = ref
    got = out.double().cpu().numpy()
    live = ~np.isnan(L)
    nan = np.isnan(O) & live[..., None]
    assert np.array_equal(np.isnan(got)[live], nan[live]), f"{what}: NaN where none belongs, or none where one does"
    fine = live[..., None] & ~nan
    err = np.abs(got - O)
    lim = tol + HALF_STEP[out.dtype] * (np.abs(O) + tol) + 1e-30
    worst = (err / np.where(fine, lim, 1.0))[fine]
    assert worst.size == 0 or worst.max() <= 1.0, f"{what}: {worst.max():.3f} of the bound, err {err[fine].max():.3e}"
    if lse is not None:
        gl = lse.double().cpu().numpy()
        empty = live & np.isneginf(L)
        assert np.array_equal(np.isneginf(gl) & live, empty), f"{what}: lse of rows that attend nothing"
        m = live & ~empty & ~np.isnan(O).any(-1)
        if m.any():
            d = np.abs(gl[m] - L[m])
            assert (d <= ltol[m]).all(), f"{what}: lse off by {d.max():.3e}"


def codes(t):
    """uint8 numpy codes of a float8 tensor."""
    return t.view(torch.uint8).cpu().numpy().copy()


def make_cache(rng, P, page, NKV, HD, spread=2):
    """A pool whose every page holds normal values under scales 2^-6 .. 2^(spread - 6)."""
    K = encode(rng.standard_normal((P, NKV, page, HD)) * 60)
    V = encode(rng.standard_normal((P, NKV, HD, page)) * 60)
    Ks = 2.0 ** (rng.integers(0, spread + 1, (P, NKV)) - 6.0)
    Vs = 2.0 ** (rng.integers(0, spread + 1, (P, NKV)) - 6.0)
    return K, V, Ks.astype(np.float32), Vs.astype(np.float32)


def to_cache(A, K, V, Ks, Vs):
    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return A.KV8Cache(dev(K).view(torch.float8_e4m3fn), dev(V).view(torch.float8_e4m3fn), dev(Ks), dev(Vs))


def tables(rng, lens, page, P, cols=None):
    """Random pages for requests of `lens` tokens; -1 behind."""
    need = [-(-int(n) // page) for n in lens]
    ids = rng.permutation(P)
    assert sum(need) <= P
    t = np.full((len(lens), cols or max(max(need), 1)), -1, np.int32)
    for b, n in enumerate(need):
        t[b, :n], ids = ids[:n], ids[n:]
    return t


def blank_tail(K, V, table, lens, page, code=0x7F):
    """NaN codes into every token of the requests' pages that is no token of theirs, and into the pages of nobody."""
    P = K.shape[0]
    used = np.zeros((P, page), bool)
    for b, n in enumerate(lens):
        for j in range(int(n)):
            if 0 <= table[b, j // page] < P:
                used[table[b, j // page], j % page] = True
    p, o = np.nonzero(~used)
    K[p, :, o, :] = code
    V[p, :, :, o] = code


def attention_rows(Q, K, V, Ks, Vs, table, ctx, cu, scale=0.0, window=0, anc=None):
    """attention() for larger calls: the same values and the same bounds, a request and KV head at a time."""
    rows_n, NQ, HD = Q.shape
    P, NKV, page, _ = K.shape
    G = NQ // NKV
    sc = scale if scale > 0 else 1.0 / np.sqrt(HD)
    O, lse, tol = np.full(Q.shape, np.nan), np.full((rows_n, NQ), np.nan), np.zeros(Q.shape)
    lse_tol = np.zeros((rows_n, NQ))
    for b in range(len(ctx)):
        n0, n, r0 = int(ctx[b]), int(cu[b + 1] - cu[b]), int(cu[b])
        if n <= 0:
            continue
        L = max(n0 + n, 0)
        j, pos = np.arange(L), n0 + np.arange(n)
        ids = np.asarray(table[b], np.int64)[j // page]
        ok = (ids >= 0) & (ids < P)
        ids, off = np.where(ok, ids, 0), j % page
        att = ok & (j <= pos[:, None])
        if window > 0:
            att &= j > pos[:, None] - window
        if anc is not None:
            d = j - n0
            att &= (d < 0) | ((np.asarray(anc[r0:r0 + n], np.int64)[:, None] >> np.clip(d, 0, 31)) & 1).astype(bool)
        some, att = att.any(0), np.repeat(att, G, 0)                   # rows: token-major, then q-heads
        nk, empty = att.sum(1), ~att.any(1)
        for h in range(NKV):
            q = Q[r0:r0 + n, h * G:(h + 1) * G].reshape(n * G, HD)
            k = np.where(some[:, None], TABLE[K[ids, h, off]] * Ks[ids, h].astype(np.float64)[:, None], 0.0)
            v = np.where(some[:, None], TABLE[V[ids, h, :, off]] * Vs[ids, h].astype(np.float64)[:, None], 0.0)
            s = np.where(att, (q @ k.T) * sc, -np.inf)
            top = np.where(empty, 0.0, s.max(1, initial=-np.inf))
            w = np.exp(s - top[:, None])
            l = w.sum(1)
            w /= np.where(empty, 1.0, l)[:, None]
            ds = np.where(att, HD * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T) * sc + 2.0 ** -22 * np.abs(s), 0.0).max(1, initial=0.0) + 2.0 ** -21
            vmax = np.where(att, np.abs(v).max(1, initial=0.0), 0.0).max(1, initial=0.0)
            rel = 2.0 ** -11 + 2 * ds + 2 * nk * 2.0 ** -24
            at = (slice(r0, r0 + n), slice(h * G, (h + 1) * G))
            with np.errstate(divide="ignore"):
                L1 = np.where(empty, -np.inf, top + np.log(l))
            O[at], lse[at] = (w @ v).reshape(n, G, HD), L1.reshape(n, G)
            tol[at] = (rel[:, None] * (w @ np.abs(v)) + (nk * 2.0 ** -30 * vmax)[:, None]).reshape(n, G, HD)
            lse_tol[at] = np.where(empty, 0.0, ds + nk * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(empty, 0.0, L1)) + 2.0 ** -20).reshape(n, G)
    return O, lse, tol, lse_tol


def make_cache_fast(rng, P, page, NKV, HD, spread=2):
    """make_cache() with values drawn from 2^16 normal ones."""
    pool = encode(rng.standard_normal(1 << 16) * 60)
    K, V = (pool[rng.integers(0, 1 << 16, s)] for s in ((P, NKV, page, HD), (P, NKV, HD, page)))
    Ks, Vs = (2.0 ** (rng.integers(0, spread + 1, (P, NKV)) - 6.0) for _ in range(2))
    return K, V, Ks.astype(np.float32), Vs.astype(np.float32)
