// Prompt attention over the paged 8-bit cache on gfx950: causal and sliding-window rows of ragged requests, behind any
// cached prefix.
//
// A workgroup holds 64 or 128 query rows (token-major: tokens x q-heads of one KV head) and walks their keys in steps of 64
// at absolute positions. Its waves are RG row groups of 16 RB rows x KG key groups, which share a step's keys; the states of a
// row's key groups are merged at the end through LDS.
//   * K and V pages go to LDS as codes, 16 bytes per lane straight from memory (global_load_lds), two stages, one barrier a
//     step: half the LDS of 16-bit tiles, and half the bytes per fragment read. The 16-byte slots of a row are XOR-swizzled
//     (kf, vf below): K's 16-byte fragment reads meet every bank once, V's 8-byte ones take two turns, a third of the LDS
//     pipe's time in all.
//   * Fragments are converted to 16 bits (exact) as they are read; every conversion serves the wave's 16 RB rows.
//   * S^T = K Q^T on 16x16x32 with tile t (of 2) of a wave's 32 keys holding key 8 (rho / 4) + 4 t + rho % 4 in row rho:
//     lane group g then has the scores of keys 8 g .. 8 g + 7, which are the operand of O^T += V^T P^T as they stand, and
//     V's [dim][token] rows give the other one: 8 bytes per lane. Q and the accumulators stay in registers.
//   * Scales and softmax are those of the split-KV form (attn_kv8_decode.hip): the V scale is part of the weight.
// Workgroups take the tiles of all requests from the latest on: the causal tiles with the most keys start first. Consecutive
// workgroups take different KV heads, so that a head's pages are read through as few of the 8 L2s as there are heads for.
//
// Steps and key groups depend on positions alone and a step without keys for a row leaves its state as it was, so a row's
// bits do not depend on its place in the tile or on the rest of the batch; they do on the tile's form, which is chosen by the
// call's size, and with key splits on the split length.
//
// What bounds it: the vector and the matrix pipe share the issue slots. At HD 256 a wave of 32 rows takes, for 32 keys, 64 MFMAs
// of 16 cycles, 128 conversions of codes (each serves both row blocks) and about 120 other vector operations, most of them the
// softmax; two waves per SIMD (registers) let one multiply while the other one converts. 6 requests of up to 2500 tokens, 24
// q-heads over 4 of 256: 325 us, 924 TFLOP/s; 4096 tokens behind a window of 1024, 16 over 8: 80 us, 755 TFLOP/s.
#include "attn_kv8.h"
#include <algorithm>
#include <climits>

namespace dgx {

struct Kv8PrefArgs {
    Kv8Problem p;
    Kv8Partials part;
    uint32_t Cm;                      // div_magic(part.C)
    int ns;                           // key splits in the grid (1: none)
    float sl2;
};

// RB: 16-row blocks of a wave; RG x KG waves: row groups, and key groups that split a step; NSUB: 32-key sub-steps that a
// wave takes of a step; OCC: waves per SIMD that the registers are held to.
template <int HD, int RB_, int RG_, int KG_, int NSUB_, int OCC_>
struct Kv8PrefCfg {
    static constexpr int RB = RB_, RG = RG_, KG = KG_, NSUB = NSUB_, OCC = OCC_, NW = RG * KG, SK = 32 * NSUB * KG;
    static constexpr int RR = 16 * RB * RG;
    static constexpr int DC = HD / 64, DB = HD / 16, KS = HD / 32;
    static constexpr int SLOTS = HD / 16, VS = SK / 16;            // 16-byte slots of a K row, and of a V row
    static constexpr int NLD = SK * HD / 16 / (NW * 64);           // 16-byte loads per thread and step, K and V each
    static constexpr int HALF = SK * HD;                           // bytes of a K (or V) step
    static constexpr int STAGE = 2 * HALF;
    static constexpr int DK = DB / KG;                             // output blocks that a key group finishes
    static constexpr int XSTR = 16 * DK + 4;                       // exchange row, floats
    static constexpr size_t LDS_X = KG == 1 ? 0 : (size_t)NW * (KG - 1) * RB * 16 * XSTR * 4 + (size_t)2 * NW * RB * 16 * 4;
    static constexpr size_t LDS = 2 * STAGE > LDS_X ? 2 * STAGE : LDS_X;
    static_assert(NLD >= 1 && LDS <= 160 * 1024 && (SK == 16 * NW || SK == 8 * NW), "a wave loads keys of one 16-key piece");
    static_assert(VS == 4 || VS == 8, "V swizzle");
};

// 16 bytes per lane from its own address to LDS at `lds` + 16 * lane (lds: byte offset, the same in all lanes). The caller
// waits for it with vmcnt: the compiler does not know of it, which keeps it from waiting for a stage in flight before it
// reads the other one. (Nothing else in the kernel that includes this uses m0.)
__device__ __forceinline__ void load_to_lds16(const void *src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}

// LDS at a byte offset. (A pointer formed from an opaque offset is generic, and its loads go the slow flat way.)
template <class T> __device__ __forceinline__ __attribute__((address_space(3))) T *lds_at(unsigned off) {
    return (__attribute__((address_space(3))) T *)(uintptr_t)off;
}

template <int HD, class Cf, bool F16>
__global__ void __launch_bounds__(Cf::NW * 64, Cf::OCC) kv8_prefill_kernel(const Kv8PrefArgs a) {
    constexpr int RB = Cf::RB, KG = Cf::KG, NSUB = Cf::NSUB, NW = Cf::NW, SK = Cf::SK;
    constexpr int DC = Cf::DC, DB = Cf::DB, KS = Cf::KS, NLD = Cf::NLD, SLOTS = Cf::SLOTS, VS = Cf::VS, DK = Cf::DK;
    extern __shared__ __align__(16) unsigned char smem[];
    const Kv8Problem &p = a.p;
    const Kv8 &kc = p.c;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, ln = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rg = wave / KG, kg = wave % KG;
    const int G = p.NQ / kc.NKV;

    // Work item: KV head, key split, and the tile, tiles of all requests by the position of their last token from the latest
    // on (in units of a tile's tokens): the tiles with the most keys start first. S(X), the tiles at X or later, is a sum over
    // requests; the item's X is the last one with S(X) > its number.
    int rest = (int)blockIdx.x;
    const int h = rest % kc.NKV; rest /= kc.NKV;
    const int sp = rest % a.ns; rest /= a.ns;
    const int unit = max(1, Cf::RR / G);
    auto rows_of = [&](int b) {
        int r0, nr = 0;
        if (b < p.B) kv8_rows(p, b, r0, nr);
        return nr;
    };
    const int nr_0 = rows_of(lane), ctx_0 = lane < p.B ? p.ctx[lane] : 0;  // (held: the search below asks some ten times)
    auto later = [&](int b, long long X) {                             // tiles of request b at X or later
        const int nr = b < 64 ? nr_0 : rows_of(b);
        if (nr <= 0) return 0;
        const int n = (int)(((long long)nr * G + Cf::RR - 1) / Cf::RR);
        const long long t = X * unit - (b < 64 ? ctx_0 : p.ctx[b]);    // first token that counts
        return X <= 0 || t <= 0 ? n : t > nr - 1 ? 0 : n - (int)(t * G / Cf::RR);
    };
    auto later_all = [&](long long X) {
        int sum = 0;
        for (int s0 = 0; s0 < p.B; s0 += 64) sum += __builtin_amdgcn_readlane(wave_scan64(later(s0 + lane, X)), 63);
        return sum;
    };
    int seq = -1, tile = 0;
    if (p.B == 1) tile = __builtin_amdgcn_readfirstlane(later(0, 0)) - 1 - rest, seq = tile < 0 ? -1 : 0;
    else {
        long long x0 = 0, x1 = (long long)p.max_pos / unit + 2;        // S(x0) > rest >= S(x1), past max_pos all count as its end
        if (later_all(x1) > rest) x0 = x1;                             // (positions past max_pos: in the order of the requests)
        else if (later_all(x0) <= rest) return;
        while (x1 - x0 > 1) {
            const long long mid = (x0 + x1) >> 1;
            if (later_all(mid) > rest) x0 = mid; else x1 = mid;
        }
        if (x1 > x0) rest -= later_all(x1);
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            const int c0 = later(s0 + lane, x0), c1 = x1 > x0 ? later(s0 + lane, x1) : 0, n = c0 - c1, incl = wave_scan64(n);
            const unsigned long long hit = __ballot(incl > rest);
            if (hit) {
                const int l = __builtin_ctzll(hit), before = __builtin_amdgcn_readlane(incl - n, l);
                int r0, n_rows = 0;
                kv8_rows(p, s0 + l, r0, n_rows);
                const int tiles = (int)(((long long)n_rows * G + Cf::RR - 1) / Cf::RR);
                seq = s0 + l;
                tile = tiles - 1 - __builtin_amdgcn_readlane(c1, l) - (rest - before);
                break;
            }
            rest -= __builtin_amdgcn_readlane(incl, 63);
        }
    }
    if (seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(seq); tile = __builtin_amdgcn_readfirstlane(tile);
    int row0, nr;
    kv8_rows(p, seq, row0, nr);
    row0 = __builtin_amdgcn_readfirstlane(row0); nr = __builtin_amdgcn_readfirstlane(nr);
    const int p0 = min(scalar_load(p.ctx + seq), INT_MAX - nr);          // (kv8_first_pos)
    const int rho0 = tile * Cf::RR, nrows = min(nr * G - rho0, Cf::RR);
    const int tok_a = rho0 / G, tok_b = (rho0 + nrows - 1) / G;        // first and last token of the tile
    int j_lo = win_lo(p0 + tok_a, p.window), j_hi = min(p0 + tok_b, p.max_pos) + 1;
    if (a.ns > 1) {
        const int c = div_by(j_lo, a.part.C, a.Cm) + sp;               // (splits are counted from the tile's first)
        j_lo = max(j_lo, c * a.part.C);
        j_hi = min(j_hi - c * a.part.C, a.part.C) + c * a.part.C;
        if (j_lo >= j_hi) return;
    }
    const int s_lo = j_lo / SK, s_hi = j_hi > j_lo ? (j_hi - 1) / SK : s_lo - 1;
    const int page = kc.page, last_col = p.max_pos >> kc.lp;
    const int *tab = p.table + (size_t)seq * p.table_stride;
    auto safe = [&](int id) { return (unsigned)id < (unsigned)kc.pages ? id : 0; };

    // Step loads. K slot S = (wave NLD + u) 64 + lane: key S / SLOTS, 16-byte column (S % SLOTS) ^ kf(key); a wave's keys lie
    // in one 16-key piece. V slot S: dim S / VS, piece (S % VS) ^ vf(dim). kf and vf are made of bits of their argument, so
    // load u differs from load 0 by a constant XOR and offset.
    auto kf = [](int key) { return HD == 128 ? ((key >> 1) & 1) | ((key >> 3) & 3) << 1 : (key & 3) | ((key >> 3) & 3) << 2; };
    auto vf = [](int dim) { return VS == 4 ? (dim >> 2) & 3 : (dim >> 1) & 7; };
    constexpr int KPL = 64 / SLOTS, DPL = 64 / VS, KPW = SK / NW;      // keys and dims of one load, keys that a wave loads
    const unsigned lds0 = (unsigned)(uintptr_t)smem;
    const int key0 = lane / SLOTS, dim0 = wave * NLD * DPL + lane / VS;
    const unsigned koff = (unsigned)(key0 * HD + (((lane % SLOTS) ^ kf(KPW * wave + key0)) << 4));
    const int vp0 = (lane % VS) ^ vf(dim0);
    constexpr int NV = VS == 8 && NLD > 1 ? 2 : 1;                     // pieces of a lane's V loads: vp0, and vp0 ^ 4 in odd u
    static_assert(VS == 4 || NLD % 2 == 0, "V pieces by the parity of u");
    // A step's pages and scales, loaded a step or two ahead: of the wave's own pieces and of its K loads through the scalar
    // cache, of the lane's V loads as vectors. (Not picked from one list of all: the compiler puts a list that is indexed by
    // wave into memory, and reading it back waits for every load in flight.)
    auto piece_id = [&](int s, int piece) { return scalar_load(tab + min((SK * s + 16 * piece) >> kc.lp, last_col)); };
    struct Ids { int s[NSUB][2], k; };
    struct VIds { int v[NV]; };
    auto ids_of = [&](int s) {
        Ids q;
#pragma unroll
        for (int x = 0; x < NSUB; x++) { q.s[x][0] = piece_id(s, 2 * (kg * NSUB + x)); q.s[x][1] = piece_id(s, 2 * (kg * NSUB + x) + 1); }
        q.k = piece_id(s, KPW * wave / 16);
        return q;
    };
    auto v_ids_of = [&](int s) {
        VIds q;
#pragma unroll
        for (int x = 0; x < NV; x++) q.v[x] = tab[min((SK * s + 16 * (vp0 ^ (4 * x))) >> kc.lp, last_col)];
        return q;
    };
    struct Scales { float k[NSUB][2], v[NSUB][2]; bool ok[NSUB][2]; };
    auto scales_of = [&](const Ids &q) {
        Scales r;
#pragma unroll
        for (int x = 0; x < NSUB; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const size_t cell = (size_t)safe(q.s[x][y]) * kc.NKV + h;
                r.ok[x][y] = (unsigned)q.s[x][y] < (unsigned)kc.pages;
                r.k[x][y] = scalar_load(kc.Ks + cell); r.v[x][y] = scalar_load(kc.Vs + cell);
            }
        return r;
    };
    const size_t head_bytes = (size_t)page * HD;
    auto issue_k = [&](int s, const Ids &q) {
        const unsigned st = lds0 + (unsigned)(s & 1) * Cf::STAGE + (unsigned)wave * NLD * 1024;
        const uint8_t *kb = kc.K + ((size_t)safe(q.k) * kc.NKV + h) * head_bytes + (size_t)((SK * s + KPW * wave) & (page - 1)) * HD;
#pragma unroll
        for (int u = 0; u < NLD; u++) load_to_lds16(kb + ((koff ^ (unsigned)(kf(u * KPL) << 4)) + u * KPL * HD), st + u * 1024);
    };
    auto issue_v = [&](int s, const VIds &q) {
        const unsigned st = lds0 + (unsigned)(s & 1) * Cf::STAGE + Cf::HALF + (unsigned)wave * NLD * 1024;
#pragma unroll
        for (int x = 0; x < NV; x++) {
            const uint8_t *vb = kc.V + (size_t)(unsigned)(safe(q.v[x]) * kc.NKV + h) * head_bytes + (unsigned)(dim0 * page + ((SK * s + 16 * (vp0 ^ (4 * x))) & (page - 1)));
#pragma unroll
            for (int u = x; u < NLD; u += NV) load_to_lds16(vb + u * DPL * page, st + u * 1024);
        }
    };
    Ids nxt{};
    VIds vnxt{};
    Scales sn{};
    if (s_lo <= s_hi) {
        const Ids q = ids_of(s_lo);
        const VIds vq = v_ids_of(s_lo);
        nxt = ids_of(min(s_lo + 1, s_hi));
        vnxt = v_ids_of(min(s_lo + 1, s_hi));
        issue_k(s_lo, q); issue_v(s_lo, vq);
        sn = scales_of(q);
    }

    // Rows of this wave: block rb holds rows lrow .. lrow + 15 of the tile; lane ln the row lrow + ln.
    u32x4 qop[RB][KS];
    int rpos[RB], wlo[RB], whi[RB], lo_max[RB], pos_min[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int lrow = (rg * RB + rb) * 16, rho = rho0 + lrow + ln;
        const bool valid = lrow + ln < nrows;
        const int tok = valid ? rho / G : 0;
        rpos[rb] = valid ? p0 + tok : -1;
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p.Q) + ((size_t)(row0 + tok) * p.NQ + h * G + (valid ? rho % G : 0)) * HD + 16 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qop[rb][ks] = u32x4{0u, 0u, 0u, 0u};
            if (valid) qop[rb][ks] = *reinterpret_cast<const u32x4 *>(q + 64 * (ks >> 1) + 8 * (ks & 1));
        }
        wlo[rb] = INT_MAX; whi[rb] = -1; lo_max[rb] = 0; pos_min[rb] = INT_MAX;
        if (lrow < nrows) {
            const int pf = p0 + (rho0 + lrow) / G, pl = p0 + (rho0 + min(nrows, lrow + 16) - 1) / G;
            wlo[rb] = max(win_lo(pf, p.window), j_lo); whi[rb] = min(pl, j_hi - 1);
            lo_max[rb] = win_lo(pl, p.window); pos_min[rb] = pf;
        }
    }
    float m[RB], l[RB];
    f32x4 acc[RB][DB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        m[rb] = kNegInf; l[rb] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++) acc[rb][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr float head = 6.f, move = 14.f;                           // see attn_kv8_decode.hip
    // K fragment (t, d) of sub-step x: row key 32 (kg NSUB + x) + 8 (ln / 4) + 4 t + ln % 4, slot (4 d + g) ^ kf. kf leaves out
    // the bits of t and of the 32 keys, so it is the same in all.
    const int krow = 32 * NSUB * kg + 8 * (ln >> 2) + (ln & 3);
    const unsigned kaddr = lds0 + (unsigned)krow * HD + ((unsigned)(g ^ kf(krow)) << 4);
    const unsigned vaddr = lds0 + Cf::HALF + (unsigned)ln * SK + 8 * (g & 1);

    for (int s = s_lo; s <= s_hi; s++) {
        // (Scalar loads without a branch around them, taken over at the end of the step: they wait with the stage.)
        const Scales s2 = scales_of(nxt);
        const Ids n2 = ids_of(min(s + 2, s_hi));
        // Stage s has landed, from every wave. By the builtin, not asm: the compiler then knows that the Q and page id loads
        // have landed too, and does not wait for them, and with them for the next stage, at their uses (2048 tokens causal, 16
        // q-heads over 8, 76.2 -> 64.4 us; HD 512 295 -> 275). With two sub-steps a step is long enough for that not to
        // matter, and its registers suffer (HD 128 93 -> 98).
        if constexpr (NSUB == 1) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt 0
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const Scales &sc = sn;
        const VIds vcur = vnxt;
        const bool more = s < s_hi;
        if (more) {
            issue_k(s + 1, nxt);
            if (NSUB == 1) issue_v(s + 1, vcur);
        }
        vnxt = v_ids_of(min(s + 2, s_hi));
#pragma unroll
        for (int x = 0; x < NSUB; x++) {
            if (x == 1 && more) issue_v(s + 1, vcur);                   // (spread over the step: at once, the waves queue for the memory pipe)
            const int jw = SK * s + 32 * (kg * NSUB + x);
            bool any = false;
#pragma unroll
            for (int rb = 0; rb < RB; rb++) any |= jw <= whi[rb] && jw + 31 >= wlo[rb];
            if (!any) continue;                                        // (wave-uniform; no barrier below)
            f32x4 st[2][RB];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int rb = 0; rb < RB; rb++) st[t][rb] = f32x4{0.f, 0.f, 0.f, 0.f};
            // (opaque bases: the fragments' addresses are formed at their reads, not held across the loop)
            unsigned ka = kaddr + (unsigned)(s & 1) * Cf::STAGE + 32 * x * HD;
            unsigned va = (vaddr + (((unsigned)(2 * (kg * NSUB + x) + (g >> 1)) ^ (unsigned)vf(ln)) << 4)) + (unsigned)(s & 1) * Cf::STAGE;
            asm volatile("" : "+v"(ka), "+v"(va));
            // Fragment 2 d + t is read while the one before it is multiplied (one, not more: registers), and converted between
            // that one's products: the vector pipe then works under the matrix pipe. A wave at its products goes before the
            // one at its softmax, which fills the gaps (both together: 4096 behind a window 91 -> 85 us, 6 ragged prompts 352 ->
            // 348, 4 of 2000 at HD 128 108 -> 99).
            u32x4 kw[2];
            auto read_k = [&](int i) { kw[i & 1] = *lds_at<u32x4>((ka ^ (64 * (i >> 1))) + 4 * (i & 1) * HD); };
            read_k(0);
            __builtin_amdgcn_s_setprio(1);
            u32x4 k0 = e4m3_op<F16>(kw[0][0], kw[0][1]), k1;
#pragma unroll
            for (int i = 0; i < 2 * DC; i++) {
                const int d = i >> 1, t = i & 1;
                if (i + 1 < 2 * DC) read_k(i + 1);
                __builtin_amdgcn_sched_barrier(0);
                st[t][0] = mfma16<F16>(k0, qop[0][2 * d], st[t][0]);
                k1 = e4m3_op<F16>(kw[t][2], kw[t][3]);
#pragma unroll
                for (int rb = 1; rb < RB; rb++) st[t][rb] = mfma16<F16>(k0, qop[rb][2 * d], st[t][rb]);
                __builtin_amdgcn_sched_barrier(0);
                st[t][0] = mfma16<F16>(k1, qop[0][2 * d + 1], st[t][0]);
                if (i + 1 < 2 * DC) k0 = e4m3_op<F16>(kw[t ^ 1][0], kw[t ^ 1][1]);
#pragma unroll
                for (int rb = 1; rb < RB; rb++) st[t][rb] = mfma16<F16>(k1, qop[rb][2 * d + 1], st[t][rb]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            const bool up = g >= 2, ok = up ? sc.ok[x][1] : sc.ok[x][0];   // the lane's 8 keys are in piece g / 2 of the sub-step's
            // (the factor stays above zero: a hidden score is -inf before it is multiplied)
            const float f = fmaxf((up ? sc.k[x][1] : sc.k[x][0]) * a.sl2, 1e-37f), ev = up ? (float)exp_of(sc.v[x][1]) : (float)exp_of(sc.v[x][0]);
            const float iv = up ? pow2i(-exp_of(sc.v[x][1])) : pow2i(-exp_of(sc.v[x][0]));
            const bool part = jw < j_lo || jw + 32 > j_hi || !(sc.ok[x][0] & sc.ok[x][1]);
            u32x4 pf[RB];
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                float tv[8];
#pragma unroll
                for (int i = 0; i < 8; i++) tv[i] = st[i >> 2][rb][i & 3];
                const bool full = !part && jw >= lo_max[rb] && jw + 31 <= pos_min[rb];
                if (!full) {
                    const int kl = max(j_lo, win_lo(rpos[rb], p.window)) - jw - 8 * g, kh = ok ? min(j_hi - 1, rpos[rb]) - jw - 8 * g : -1;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if ((i < kl) | (i > kh)) tv[i] = kNegInf;
                }
                // Scores of a lane share their factor and addend, so the maximum is taken before them.
                float mx = tv[0];
#pragma unroll
                for (int i = 1; i < 8; i++) mx = fmaxf(mx, tv[i]);
                mx = __builtin_fmaf(mx, f, ev);
                if (__any(mx > m[rb] + move)) {                         // rare: only then the lane groups' maxima meet
                    mx = max_over_groups(mx);
                    const float mn = mx > m[rb] + move ? mx - head : m[rb];
                    const float al = mn == m[rb] ? 1.f : fast_exp2(m[rb] - mn);
                    l[rb] *= al; m[rb] = mn;
#pragma unroll
                    for (int d = 0; d < DB; d++) acc[rb][d] *= al;
                }
                const float mz = m[rb] == kNegInf ? 0.f : m[rb], e0 = ev - mz;   // (no key yet: every 2^(-inf) is 0)
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    tv[i] = fast_exp2(__builtin_fmaf(tv[i], f, e0));
                    sum += tv[i];
                }
                l[rb] = __builtin_fmaf(sum, iv, l[rb]);
                pf[rb] = u32x4{pack2<true>(tv[0], tv[1]), pack2<true>(tv[2], tv[3]), pack2<true>(tv[4], tv[5]), pack2<true>(tv[6], tv[7])};
            }
            if (part) {
                // Bytes that are no token of the request's weigh nothing, NaN codes neither: cleared in LDS, in the wave's own
                // 32 keys (the other row groups clear the same ones before they read them). Rare, and a mask in the loop below
                // would cost 2 operations per fragment of 8, a second copy of the loop 64 registers.
                const int k0 = ok ? max(j_lo - jw - 8 * g, 0) : 8, k1 = min(j_hi - jw - 8 * g, 8);
                u32x2 keep;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const int x0 = min(max(k0 - 4 * w, 0), 4), y0 = min(max(k1 - 4 * w, 0), 4);
                    keep[w] = (y0 >= 4 ? 0xffffffffu : (1u << (8 * y0)) - 1u) & ~(x0 >= 4 ? 0xffffffffu : (1u << (8 * x0)) - 1u);
                }
#pragma unroll 1
                for (int d = 0; d < DB; d++) {
                    const u32x2 w = *lds_at<u32x2>(va + 16 * SK * d);
                    *lds_at<u32x2>(va + 16 * SK * d) = w & keep;
                }
            }
            constexpr int VB = 4;                                      // dim blocks read ahead
            u32x2 vw[2][VB];
            auto read_v = [&](int b) {
#pragma unroll
                for (int y = 0; y < VB; y++) vw[b & 1][y] = *lds_at<u32x2>(va + 16 * SK * (b * VB + y));
            };
            read_v(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int b = 0; b < DB / VB; b++) {
                if (b + 1 < DB / VB) read_v(b + 1);
                __builtin_amdgcn_sched_barrier(0);
                u32x4 v = e4m3_op<true>(vw[b & 1][0][0], vw[b & 1][0][1]);
#pragma unroll
                for (int y = 0; y < VB; y++) {
                    acc[0][b * VB + y] = mfma16<true>(v, pf[0], acc[0][b * VB + y]);
                    u32x4 vn = v;
                    if (y + 1 < VB) vn = e4m3_op<true>(vw[b & 1][y + 1][0], vw[b & 1][y + 1][1]);
#pragma unroll
                    for (int rb = 1; rb < RB; rb++) acc[rb][b * VB + y] = mfma16<true>(v, pf[rb], acc[rb][b * VB + y]);
                    v = vn;
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        nxt = n2; sn = s2;
        __builtin_amdgcn_s_setprio(0);
    }

    // Merge of the key groups: each wave finishes DK blocks of 16 dims of its rows and hands the others over. Everything is
    // weighted and added in key-group order, whichever wave does it.
    float *xb = reinterpret_cast<float *>(smem), *stm = xb + (size_t)NW * (KG - 1) * RB * 16 * Cf::XSTR, *stl = stm + NW * RB * 16;
#pragma unroll
    for (int rb = 0; rb < RB; rb++) l[rb] = sum_over_groups(l[rb]);
    if constexpr (KG > 1) {
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            if (g == 0) { stm[(wave * RB + rb) * 16 + ln] = m[rb]; stl[(wave * RB + rb) * 16 + ln] = l[rb]; }
#pragma unroll
            for (int o = 0; o < KG; o++) {                             // blocks of key group o; slot o (o - 1 past the own one)
                if (o == kg) continue;
                float *x = xb + (((size_t)wave * (KG - 1) + (o > kg ? o - 1 : o)) * RB + rb) * 16 * Cf::XSTR + ln * Cf::XSTR + 4 * g;
#pragma unroll
                for (int d = 0; d < DK; d++) *reinterpret_cast<f32x4 *>(x + 16 * d) = acc[rb][o * DK + d];
            }
            // What the wave keeps, moved to the front (by value: a choice of addresses would put acc in memory).
#pragma unroll
            for (int d = 0; d < DK; d++) {
                f32x4 v = acc[rb][d];
#pragma unroll
                for (int o = 1; o < KG; o++)
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = kg == o ? acc[rb][o * DK + d][i] : v[i];
                acc[rb][d] = v;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int lrow = (rg * RB + rb) * 16 + ln, rho = rho0 + lrow;
        if (lrow >= nrows) continue;
        float M = m[rb], L = l[rb], f[KG];
        if constexpr (KG > 1) {
            M = kNegInf; L = 0.f;
#pragma unroll
            for (int o = 0; o < KG; o++) M = fmaxf(M, stm[((rg * KG + o) * RB + rb) * 16 + ln]);
#pragma unroll
            for (int o = 0; o < KG; o++) {
                const float lo = stl[((rg * KG + o) * RB + rb) * 16 + ln];
                f[o] = kv8_weight(stm[((rg * KG + o) * RB + rb) * 16 + ln], lo, M);
                L += lo * f[o];
            }
        }
        const size_t row = (size_t)(row0 + rho / G) * p.NQ + h * G + rho % G;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int dim = kg * DK * 16 + 4 * g;
        const size_t px = row * a.part.ns + (a.ns > 1 ? div_by(j_lo, a.part.C, a.Cm) - div_by(win_lo(p0, p.window), a.part.C, a.Cm) : 0);
#pragma unroll
        for (int d = 0; d < DK; d++) {
            f32x4 v = acc[rb][d];
            if constexpr (KG > 1) {
                const f32x4 mine = v;
                v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int o = 0; o < KG; o++) {
                    const float *x = xb + (((size_t)(rg * KG + o) * (KG - 1) + (kg > o ? kg - 1 : kg)) * RB + rb) * 16 * Cf::XSTR + ln * Cf::XSTR + 4 * g;
                    v += (o == kg ? mine : *reinterpret_cast<const f32x4 *>(x + 16 * d)) * f[o];
                }
            }
            if (a.ns > 1) *reinterpret_cast<f32x4 *>(a.part.acc + px * HD + dim + 16 * d) = v;
            else kv8_store4(p, row * HD + dim + 16 * d, v * inv);
        }
        if (kg == 0 && g == 0) {
            if (a.ns > 1) { a.part.m[px] = M; a.part.l[px] = L; }
            else if (p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
        }
    }
}

template <int HD, class Cf, bool F16>
static hipError_t launch_pre_k(const Kv8PrefArgs &a, hipStream_t st) {
    const long long G = a.p.NQ / a.p.c.NKV;
    const long long tiles = std::min((long long)a.p.B * ((a.p.T * G + Cf::RR - 1) / Cf::RR), (long long)a.p.rows * G / Cf::RR + a.p.B);
    const long long wgs = tiles * a.p.c.NKV * a.ns;
    if (!kv8_grid_ok(wgs, Cf::NW * 64)) return hipErrorInvalidConfiguration;
    if constexpr (Cf::LDS > 64 * 1024) {                               // (per device; setting it again changes nothing)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv8_prefill_kernel<HD, Cf, F16>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)Cf::LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((kv8_prefill_kernel<HD, Cf, F16>), dim3((unsigned)wgs), dim3(Cf::NW * 64), Cf::LDS, st, a);
    return hipGetLastError();
}
template <int HD, class Cf> static hipError_t launch_pre(const Kv8PrefArgs &a, hipStream_t st) {
    return a.p.q_dtype == DT_F16 ? launch_pre_k<HD, Cf, true>(a, st) : launch_pre_k<HD, Cf, false>(a, st);
}

hipError_t launch_kv8_prefill(const Kv8Problem &p, const Kv8Partials &part, const Kv8Plan &pl, hipStream_t st) {
    const Kv8PrefArgs a{p, part, part.C ? div_magic(part.C) : 0u, pl.ns, p.scale * kLog2e};
    // (128 rows at HD 256 take all 256 registers and spill three; one of them is read again at the V loads of every step, a wait for
    // the step's K loads with it.)
    const bool wide = pl.tile == 128;
    switch (p.c.HD) {
    case 128: return wide ? launch_pre<128, Kv8PrefCfg<128, 2, 4, 1, 2, 2>>(a, st) : launch_pre<128, Kv8PrefCfg<128, 2, 2, 2, 1, 3>>(a, st);
    case 256: return wide ? launch_pre<256, Kv8PrefCfg<256, 2, 4, 1, 2, 2>>(a, st) : launch_pre<256, Kv8PrefCfg<256, 2, 2, 2, 1, 2>>(a, st);
    case 512:                                                          // (64 rows in 8 waves; before later steps 4 of 1500 x 16 q-heads 299 us, in 4 waves 333, 32 rows 444; 277 now)
        return launch_pre<512, Kv8PrefCfg<512, 1, 4, 2, 1, 2>>(a, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dgx
