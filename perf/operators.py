"""The 8-bit paged KV cache's operators, as a serving program calls them, and their plain forms.

The cache holds K and V as e4m3 codes in pages of `page` tokens, with one power-of-two scale 2^e for each page and KV
head (a value is code * scale), K pages as [NKV, page, HD] and V pages as [NKV, HD, page]. Three operators:
  plan       block tables and slot maps of a step from the requests' lengths, with new pages from a stack of free ones
  append     new K / V rows into the cache through the slot map: the page's scale grows where a new value needs it, and
             the codes that the page already held are rounded again to the grown scale
  attention  over the cache through the block tables: single tokens, draft trees and prompts

A case is a dict of plain values:
  kind       "plan", "append" or "attention"
  B          requests; `lo`..`hi` their cached lengths and `tlo`..`thi` their new tokens, drawn log-uniformly from the
             seed `lens` (they belong to the case: its work depends on them); T is the most new tokens of one request
  page       tokens of a page
  NQ, NKV, HD   query heads, KV heads, head dim;  io: type of Q and O;  src: type of appended rows
  window     sliding window in keys (0: causal);  tree: draft trees over the new tokens;  chunk: split chunk (0: own)

Head layouts are those of this repository's configurations: 24 q-heads over 4 KV heads of 256 (Qwen3.5 full attention),
16 over 8 of 256 (Gemma4 sliding layers), 16 over 1 of 512 (Gemma4 global layers), 16 over 4 of 128.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DT = {"fp32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "f16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn
E_MIN, E_MAX = -40, 40                     # exponents of the scales
HEADS = {"qwen": (24, 4, 256), "slide": (16, 8, 256), "global": (16, 1, 512), "small": (16, 4, 128)}


def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgx-serving_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dgx_attn
    return dgx_attn


def _case(kind, B, lo, hi, tlo, thi, page=64, heads="qwen", io="f16", src="bf16", window=0, tree=False, chunk=0, lens=1, name=None):
    NQ, NKV, HD = HEADS[heads]
    c = dict(kind=kind, B=B, lo=lo, hi=hi, tlo=tlo, thi=thi, page=page, NQ=NQ, NKV=NKV, HD=HD, io=io, src=src, window=window,
             tree=tree, chunk=chunk, lens=lens)
    return dict(c, name=name) if name else c


def listed():
    return [
        # The tables of a decode step: 256 running requests, a token each, a few of which begin a page.
        _case("plan", 256, 255, 8191, 1, 1, name="plan_decode"),
        # The tables of a step that takes in 96 prompts, on small pages.
        _case("plan", 96, 0, 512, 64, 4096, page=16, lens=2, name="plan_prompts"),
        # A decode step's rows: 16 requests, a token each, most into a page that holds some.
        _case("append", 16, 255, 8191, 1, 1, lens=2026, name="append_decode"),
        # A prompt of 1024 tokens, from fp32 projections.
        _case("append", 1, 0, 0, 1024, 1024, heads="slide", src="fp32", name="append_prompt"),
        # The prompts of a batch at once, some of them continued.
        _case("append", 24, 0, 1000, 700, 6000, page=32, heads="slide", lens=3, name="append_batch"),
        # One user, one token, a short context: latency and launches.
        _case("attention", 1, 511, 511, 1, 1, heads="small", name="decode_one"),
        # A full serving batch, one token per request.
        _case("attention", 16, 255, 8191, 1, 1, lens=2026, name="decode_batch"),
        # A global layer over long contexts: one KV head of 512.
        _case("attention", 8, 1023, 32767, 1, 1, heads="global", io="bf16", lens=13, name="decode_global"),
        # Speculative decoding: draft trees of 8 nodes for 16 requests.
        _case("attention", 16, 2048, 16384, 8, 8, tree=True, lens=5, name="tree_verify"),
        # A prompt of 1024 tokens.
        _case("attention", 1, 0, 0, 1024, 1024, heads="slide", io="bf16", name="prefill_causal"),
        # A long prompt through a sliding-window layer, on pages of 32.
        _case("attention", 1, 0, 0, 4096, 4096, page=32, heads="slide", io="bf16", window=1024, name="prefill_window"),
        # Prompts of several requests at once, odd lengths, behind cached prefixes.
        _case("attention", 6, 100, 2000, 200, 2500, lens=7, name="prefill_ragged"),
    ]


def draw(rng):
    def size(lo, hi):                      # spread over the logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kw = dict(page=rng.choice([16, 32, 64, 64]), lens=rng.randrange(1 << 20))
    kind = rng.choice(["plan", "append", "append", "decode", "decode", "decode", "verify", "verify", "prefill", "prefill", "prefill"])
    if kind == "plan":
        if rng.random() < 0.5:
            hi = size(64, 16384)
            return _case("plan", size(1, 512), min(hi, 15), hi, 1, rng.choice([1, 4]), **kw)
        top = size(64, 4096)
        return _case("plan", size(1, 96), 0, 512, max(1, top // 16), top, **kw)
    heads = rng.choice(["qwen", "qwen", "slide", "global", "small"])
    kw["io"] = kw["src"] = rng.choice(["f16", "bf16"])
    if kind == "append":
        kw["src"] = rng.choice(["fp32", "f16", "bf16"])
        if rng.random() < 0.5:
            hi = size(64, 8191)
            return _case("append", size(1, 64), min(hi, 15), hi, 1, size(1, 8), heads=heads, **kw)
        top = size(32, 4096)
        return _case("append", size(1, 8), 0, rng.choice([0, 1000]), max(1, top // 8), top, heads=heads, **kw)
    window = rng.choice([0, 0, 512, 1024])
    if kind == "decode":
        hi = size(64, 16384)
        return _case("attention", size(1, 16), max(1, hi // 16), hi, 1, 1, heads=heads, window=window, chunk=rng.choice([0, 0, 256, 512]), **kw)
    if kind == "verify":
        hi, t = size(64, 12000), rng.randint(2, 16)
        tree = rng.random() < 0.6
        return _case("attention", size(1, 16), max(1, hi // 8), hi, t if tree else 1, t, heads=heads, window=0 if tree else window, tree=tree, **kw)
    top = size(64, 2000)
    return _case("attention", rng.choice([1, 1, 2, 4]), 0, rng.choice([0, 0, 700, 3000]), max(1, top // 4), top, heads=heads, window=window, **kw)


# ---------------------------------------------------------------- inputs
def _lens(c):
    """Cached lengths and new tokens of the requests."""
    r = np.random.default_rng(c["lens"])

    def spread(lo, hi, n):
        x = np.exp(r.uniform(math.log(lo + 1), math.log(hi + 1), n)) - 1
        return np.clip(np.rint(x), lo, hi).astype(np.int64)

    ctx, add = spread(c["lo"], c["hi"], c["B"]), spread(c["tlo"], c["thi"], c["B"])
    add[0] = c["thi"]                       # the longest, so that it is the case's own
    return ctx, add


def _trees(c):
    """Draft trees as ancestor masks [B, T]: every node has at most two children, parents precede children."""
    r = np.random.default_rng(c["lens"] + 1)
    T = c["thi"]
    anc = np.zeros((c["B"], T), np.uint32)
    for b in range(c["B"]):
        par, kids = [-1], [0] * T
        for j in range(1, T):
            p = int(r.choice([p for p in range(j) if kids[p] < 2]))
            par.append(p)
            kids[p] += 1
        for j in range(T):
            x = j
            while x >= 0:
                anc[b, j] |= np.uint32(1 << x)
                x = par[x]
    return anc


def _pow2(e):
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _exponent(amax):
    """The least e with amax <= 448 * 2^e (448 = 0.875 * 2^9, the largest e4m3 value), within [E_MIN, E_MAX]."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _encode(x):
    """fp32 values, already divided by the scale, to the nearest e4m3 codes (ties to even)."""
    return x.clamp(-448.0, 448.0).to(F8)


def _fill(g, P, NKV, page, HD):
    """Pages of K (channels of uneven size) and V as a model's tokens leave them: codes [P, NKV, page, HD] and scales."""
    out = []
    for uneven in (0.5, 0.2):
        x = torch.randn(P, NKV, page, HD, device="cuda", generator=g)
        x *= torch.exp(uneven * torch.randn(1, NKV, 1, HD, device="cuda", generator=g))
        e = _exponent(x.abs().amax(dim=(2, 3)))
        out += [_encode(x * _pow2(-e)[:, :, None, None]), _pow2(e)]
    return out


def _inputs(c, seed):
    """The tensors of a case, the same for prepare() and exact()."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    r = np.random.default_rng(int(seed) * 7919 + 17)
    ctx, add = _lens(c)
    page, B, NKV, HD = c["page"], c["B"], c["NKV"], c["HD"]
    have, want = -(-ctx // page), -(-(ctx + add) // page)
    P = int(want.sum()) + 3
    cols = int(want.max()) + 1
    ids = r.permutation(P)
    table = np.full((B, cols), -1, np.int64)
    for b in range(B):
        n = int(have[b]) if c["kind"] == "plan" else int(want[b])
        table[b, :n], ids = ids[:n], ids[n:]
    rows = int(add.sum())
    cu = np.concatenate([[0], np.cumsum(add)])
    x = dict(ctx=ctx, add=add, cu=cu, table=table, rows=rows, P=P, cols=cols, T=int(add.max()), max_pos=int((ctx + add).max()) - 1)
    x["free"] = ids                         # a stack: the last is taken first
    if c["kind"] == "plan":
        x["cap"] = rows + 1 + rows % 61     # rows of the step's buffers; those behind the last token get no slot
        return x
    x["K"], x["Ks"], V, x["Vs"] = _fill(g, P, NKV, page, HD)
    x["V"] = V.transpose(2, 3).contiguous()
    if c["kind"] == "append":
        for name, sd in (("k", 1.3), ("v", 1.1)):
            x[name] = (sd * torch.randn(rows, NKV, HD, device="cuda", generator=g)).to(DT[c["src"]])
        seq = np.repeat(np.arange(B), add)
        pos = ctx[seq] + np.arange(rows) - cu[seq]
        x["slots"] = table[seq, pos // page] * page + pos % page
    else:
        x["Q"] = torch.randn(rows, c["NQ"], HD, device="cuda", generator=g).to(DT[c["io"]])
        x["anc"] = _trees(c) if c["tree"] else None
    return x


def prepare(case, seed):
    c, s = case, _inputs(case, seed)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()

    s["c"] = c
    for k in ("ctx", "add", "cu", "table", "free"):
        s[k] = dev(s[k])
    if c["kind"] == "plan":
        s["count"] = dev(np.array([s["free"].numel()]))
        s["left"], s["status"] = torch.empty_like(s["count"]), torch.empty_like(s["count"])
        s["cu"] = torch.empty(c["B"] + 1, dtype=torch.int32, device="cuda")
        s["slots"] = torch.empty(s["cap"], dtype=torch.int32, device="cuda")
    elif c["kind"] == "append":
        s["slots"] = dev(s["slots"])
    else:
        s["O"] = torch.empty_like(s["Q"])
        if s["anc"] is not None:
            s["anc"] = torch.from_numpy(s["anc"].reshape(-1).view(np.int32)).cuda()
    if own and c["kind"] != "plan":         # the handle, and the workspace that a server holds for its steps
        A = _lib()
        s["cache"] = A.KV8Cache(s["K"], s["V"], s["Ks"], s["Vs"])
        if c["kind"] == "attention":
            n = A.attn_kv8_workspace(c["B"], s["T"], s["rows"], c["NQ"], c["NKV"], c["HD"], s["max_pos"], c["chunk"], c["window"])
            s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return s


def run(state):
    s, c = state, state["c"]
    kind = c["kind"]
    if own:
        A = _lib()
        if kind == "plan":
            A.kv8_plan(s["ctx"], s["add"], c["page"], s["table"], s["free"], s["count"], s["left"], s["cu"], s["slots"], s["status"])
        elif kind == "append":
            A.kv8_append(s["k"], s["v"], s["cache"], s["slots"])
        else:
            A.attn_kv8(s["Q"], s["cache"], s["table"], s["ctx"], s["O"], s["T"], s["max_pos"], cu=s["cu"], anc=s["anc"],
                       chunk=c["chunk"], ws=s["ws"], window=c["window"])
    elif kind == "plan":
        _plain_plan(s, c)
    elif kind == "append":
        _plain_append(s, c)
    else:
        _plain_attention(s, c)
    if kind == "plan":
        return {"table": s["table"], "cu": s["cu"], "slots": s["slots"], "left": s["left"], "status": s["status"]}
    if kind == "append":                    # codes as e4m3 numbers, which the scales multiply
        return {"K": s["K"], "V": s["V"], "Ks": s["Ks"], "Vs": s["Vs"]}
    return {"O": s["O"]}


# ---------------------------------------------------------------- plain forms
def _plain_plan(s, c):
    page, dev = c["page"], s["ctx"].device
    ctx, add = s["ctx"].long(), s["add"].long()
    have, want = (ctx + page - 1) // page, (ctx + add + page - 1) // page
    before = torch.cumsum(want - have, 0) - (want - have)          # pages that earlier requests take
    cu = torch.nn.functional.pad(torch.cumsum(add, 0), (1, 0))
    enough = (want - have).sum() <= s["count"][0]
    fits = (want.max() <= s["table"].shape[1]) & (cu[-1] <= s["slots"].numel())
    good = enough & fits
    col = torch.arange(s["table"].shape[1], device=dev)
    new = (col >= have[:, None]) & (col < want[:, None]) & good
    at = s["count"].long() - 1 - (before[:, None] + col - have[:, None])
    s["table"].copy_(torch.where(new, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"]))
    row = torch.arange(s["slots"].numel(), device=dev)
    seq = (torch.searchsorted(cu, row, right=True) - 1).clamp(0, c["B"] - 1)
    pos = ctx[seq] + row - cu[seq]
    slot = s["table"][seq, (pos // page).clamp(0, s["table"].shape[1] - 1)].long() * page + pos % page
    s["slots"].copy_(torch.where((row < cu[-1]) & good, slot, torch.full_like(slot, -1)))
    s["cu"].copy_(torch.where(good, cu, torch.zeros_like(cu)))
    s["left"].copy_(s["count"] - torch.where(good, (want - have).sum(), torch.zeros_like(cu[0])))
    s["status"].copy_(torch.where(good, 0, 1).reshape(1))


def _plain_store(x, C, S, slots, page, transposed):
    """Rows x [rows, NKV, HD] into pages C of one tensor (codes) with scales S, at `slots`."""
    x = x.float()
    pid, off = slots // page, slots % page
    pages, at = torch.unique(pid, return_inverse=True)             # the touched pages, and each row's among them
    n = pages.numel()
    amax = torch.zeros(n, S.shape[1], device=x.device).index_reduce_(0, at, x.abs().amax(2), "amax")
    first = torch.full((n,), page, device=x.device).index_reduce_(0, at, off, "amin")
    old = torch.frexp(S[pages])[1] - 1
    e = torch.maximum(_exponent(amax), torch.where(first[:, None] > 0, old, torch.full_like(old, E_MIN)))
    codes = C.view(torch.uint8)[pages].view(F8)
    t = codes.transpose(2, 3) if transposed else codes             # [n, NKV, page, HD]
    again = _encode(t.float() * _pow2(old - e)[:, :, None, None])
    held = (torch.arange(page, device=x.device) < first[:, None])[:, None, :, None]
    t = torch.where(held, again.view(torch.uint8), t.contiguous().view(torch.uint8))
    t[at, :, off] = _encode(x * _pow2(-e)[at][:, :, None]).view(torch.uint8)
    C.view(torch.uint8)[pages] = t.transpose(2, 3) if transposed else t
    S[pages] = _pow2(e)


def _plain_append(s, c):
    slots = s["slots"].long()
    _plain_store(s["k"], s["K"], s["Ks"], slots, c["page"], False)
    _plain_store(s["v"], s["V"], s["Vs"], slots, c["page"], True)


def _plain_attention(s, c):
    B, T, NQ, NKV, HD, page = c["B"], s["T"], c["NQ"], c["NKV"], c["HD"], c["page"]
    G, dev = NQ // NKV, s["Q"].device
    cu, ctx = s["cu"].long(), s["ctx"].long()
    need = s["max_pos"] // page + 1
    ids = s["table"][:, :need].long().clamp(min=0)
    L = need * page

    def values(C, S, transposed):                                  # [B, NKV, L, HD]
        t = C.view(torch.uint8)[ids].view(F8)
        t = (t.transpose(3, 4) if transposed else t).float() * S[ids][..., None, None]
        return t.transpose(1, 2).reshape(B, NKV, L, HD)

    K, V = values(s["K"], s["Ks"], False), values(s["V"], s["Vs"], True)
    j = torch.arange(L, device=dev)
    pos = ctx[:, None] + torch.arange(T, device=dev)               # [B, T]
    ok = j <= pos[..., None]
    if c["window"]:
        ok &= j > pos[..., None] - c["window"]
    if s["anc"] is not None:
        d = j - ctx[:, None]                                       # [B, L]
        bit = (s["anc"].view(B, T)[..., None].long() >> d.clamp(0, 31)[:, None, :]) & 1
        ok &= (d < 0)[:, None, :] | (bit != 0)
    V = torch.where((j <= pos[:, -1:])[:, None, :, None], V, torch.zeros((), device=dev))   # unwritten rows weigh nothing
    row = (cu[:-1, None] + torch.arange(T, device=dev)).clamp(max=s["rows"] - 1)
    q = s["Q"][row].float().view(B, T, NKV, G, HD).transpose(1, 2).reshape(B, NKV, T * G, HD)
    w = torch.matmul(q, K.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(HD))
    w = w.view(B, NKV, T, G, L).masked_fill_(~ok[:, None, :, None, :], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, NKV, T * G, L), V).view(B, NKV, T, G, HD).transpose(1, 2).reshape(B, T, NQ, HD)
    r = torch.arange(s["rows"], device=dev)
    seq = torch.searchsorted(cu, r, right=True) - 1
    s["O"].copy_(o[seq, r - cu[seq]])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    ctx, add = _lens(c)
    page, NKV, HD = c["page"], c["NKV"], c["HD"]
    rows = int(add.sum())
    if c["kind"] == "plan":                 # lengths, free pages and begun pages in; table entries, offsets and slots out
        new = int((-(-(ctx + add) // page) - -(-ctx // page)).sum())
        return {"bytes": 4 * (2 * c["B"] + 2 * new + int((ctx % page > 0).sum()) + c["B"] + 4 + rows + 1 + rows % 61), "flops": 3 * rows}
    if c["kind"] == "append":               # rows in, codes and scales out; a page that holds tokens: its scale and codes may change
        pages = int((-(-(ctx + add) // page) - ctx // page).sum())
        return {"bytes": 2 * NKV * (rows * HD * (SIZE[c["src"]] + 1) + 4 * pages) + 4 * rows, "flops": 4 * rows * NKV * HD}
    w, pairs, keys = c["window"], 0, 0
    anc = _trees(c) if c["tree"] else None
    for b in range(c["B"]):
        pos = int(ctx[b]) + np.arange(int(add[b]), dtype=np.int64)
        lo = np.maximum(0, pos - w + 1) if w else np.zeros_like(pos)
        pairs += int((pos + 1 - lo).sum()) if anc is None else int(ctx[b]) * len(pos) + sum(bin(int(a)).count("1") for a in anc[b])
        keys += int(pos[-1] + 1 - lo[0])
    nbytes = 2 * keys * NKV * HD + 8 * NKV * (keys // page) + 2 * rows * c["NQ"] * HD * SIZE[c["io"]]
    return {"bytes": nbytes, "flops": 4 * HD * c["NQ"] * pairs}


# ---------------------------------------------------------------- 64-bit results
def _round8(x):
    """The e4m3 number nearest to each float64, ties to the even one: steps of 2^-9 below 2^-6, of 1/8 of the octave above."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None
    x = _inputs(c, seed)
    page = c["page"]
    if c["kind"] == "append":
        out = {}
        slots = torch.from_numpy(x["slots"]).cuda()
        off0, touched = np.full(x["P"], page), np.zeros(x["P"], bool)
        np.minimum.at(off0, x["slots"] // page, x["slots"] % page)
        touched[x["slots"] // page] = True
        off0, touched = torch.from_numpy(off0).cuda(), torch.from_numpy(touched).cuda()
        for name, C, S in (("k", "K", "Ks"), ("v", "V", "Vs")):
            new, scale = x[name].double(), x[S].double()
            cells = x[C].to(torch.float32).double()
            if C == "V":
                cells = cells.transpose(2, 3)
            # Tokens as values, [P, NKV, page, HD]: what the page held before its first new row, then the new rows.
            there = torch.zeros(x["P"] * page, *new.shape[1:], device="cuda", dtype=torch.float64)
            there[slots] = new
            there = there.view(x["P"], page, *new.shape[1:]).transpose(1, 2)
            top = there.abs().amax(dim=(2, 3))
            need = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))), torch.zeros_like(top))
            need = need.clamp(2.0 ** E_MIN, 2.0 ** E_MAX)
            need = torch.where((off0 > 0)[:, None], torch.maximum(need, scale), need)
            need = torch.where(touched[:, None], need, scale)
            is_new = torch.zeros(x["P"] * page, dtype=torch.bool, device="cuda")
            is_new[slots] = True
            is_new = is_new.view(x["P"], 1, page, 1)
            held = (torch.arange(page, device="cuda") < off0[:, None])[:, None, :, None] & touched[:, None, None, None]
            n4 = need[:, :, None, None]
            cells = torch.where(is_new, _round8(there / n4), torch.where(held, _round8(cells * (scale / need)[:, :, None, None]), cells))
            out[C], out[S] = (cells.transpose(2, 3).contiguous() if C == "V" else cells), need
        return out
    NQ, NKV, HD, w = c["NQ"], c["NKV"], c["HD"], c["window"]
    G = NQ // NKV
    out = torch.empty(x["Q"].shape, device="cuda", dtype=torch.float64)
    for b in range(c["B"]):
        n0, n = int(x["ctx"][b]), int(x["add"][b])
        r0, L = int(x["cu"][b]), n0 + n
        ids = torch.from_numpy(x["table"][b, :-(-L // page)]).cuda()
        for h in range(NKV):
            k = x["K"].view(torch.uint8)[ids, h].view(F8).float().double() * x["Ks"][ids, h].double()[:, None, None]
            v = x["V"].view(torch.uint8)[ids, h].view(F8).float().double() * x["Vs"][ids, h].double()[:, None, None]
            k, v = k.reshape(-1, HD)[:L], v.transpose(1, 2).reshape(-1, HD)[:L]
            for t0 in range(0, n, 512):
                t1 = min(n, t0 + 512)
                p = torch.arange(n0 + t0, n0 + t1, device="cuda")
                j0, j1 = (max(0, n0 + t0 - w + 1) if w else 0), n0 + (n if c["tree"] else t1)
                j = torch.arange(j0, j1, device="cuda")
                hide = j[None, :] > p[:, None]
                if w:
                    hide |= j[None, :] <= p[:, None] - w
                if x["anc"] is not None:
                    bits = torch.from_numpy(x["anc"][b, t0:t1].astype(np.int64)).cuda()
                    d = j - n0
                    hide |= (d >= 0)[None, :] & (((bits[:, None] >> d.clamp(0, 31)[None, :]) & 1) == 0)
                q = x["Q"][r0 + t0:r0 + t1, h * G:(h + 1) * G].double().reshape(-1, HD)
                sc = torch.mm(q, k[j0:j1].t().contiguous()) / math.sqrt(HD)
                sc.masked_fill_(hide.repeat_interleave(G, 0), -math.inf)
                out[r0 + t0:r0 + t1, h * G:(h + 1) * G] = torch.mm(torch.softmax(sc, -1), v[j0:j1].contiguous()).view(-1, G, HD)
    return {"O": out}
