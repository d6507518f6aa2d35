// Prompt attention over the paged 8-bit cache on gfx950: causal and sliding-window rows of ragged requests, behind any
// cached prefix.
//
// A workgroup holds 64 RB query rows (token-major: tokens x q-heads of one KV head) and walks their keys in steps of 64 at
// absolute positions. Its 8 waves are 4 row groups (16 RB rows each) x 2 key groups (32 keys of a step each); the two
// states of a row are merged at the end through LDS.
//   * K and V pages go to LDS as codes, 16 bytes per lane straight from memory (global_load_lds), two stages, one barrier a
//     step: half the LDS of 16-bit tiles, and half the bytes per fragment read. The 16-byte slots of a row are XOR-swizzled
//     so that a fragment read meets every bank once (kf, vf below).
//   * Fragments are converted to 16 bits (exact) as they are read; every conversion serves the wave's 16 RB rows.
//   * S^T = K Q^T on 16x16x32 with tile t (of 2) of a wave's 32 keys holding key 8 (rho / 4) + 4 t + rho % 4 in row rho:
//     lane group g then has the scores of keys 8 g .. 8 g + 7, which are the operand of O^T += V^T P^T as they stand, and
//     V's [dim][token] rows give the other one: 8 bytes per lane. Q and the accumulators stay in registers.
//   * Scales and softmax are those of the split-KV form (attn_kv8_decode.hip): the V scale is part of the weight.
// Workgroups take a request's tiles from its last one on: the causal tiles with the most keys start first. Consecutive
// workgroups take different KV heads, so that a head's pages are read through as few of the 8 L2s as there are heads for.
//
// Steps and key groups depend on positions alone and a step without keys for a row leaves its state as it was, so a row's
// bits do not depend on its tile, its batch or how the prompt is cut; with key splits, on the split length too.
//
// What bounds it: per step and wave 64 RB MFMAs, 16 RB conversions of the softmax's order and 256 of codes at HD 256. VALU and matrix
// time are about equal at RB = 2 (a row group of 32).
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

template <int HD, int RB>
struct Kv8PrefCfg {
    static constexpr int NW = 8, RG = 4, SK = 64;
    static constexpr int RR = 16 * RB * RG;
    static constexpr int DC = HD / 64, DB = HD / 16, KS = HD / 32;
    static constexpr int SLOTS = HD / 16;              // 16-byte slots of a K row
    static constexpr int NLD = 4 * HD / (NW * 64);     // 16-byte loads per thread and step, K and V each
    static constexpr int HALF = SK * HD;               // bytes of a K (or V) step
    static constexpr int STAGE = 2 * HALF;
    static constexpr int XSTR = HD / 2 + 4;            // exchange row, floats
    static constexpr size_t LDS_X = (size_t)NW * RB * 16 * XSTR * 4 + (size_t)2 * NW * RB * 16 * 4;
    static constexpr size_t LDS = 2 * STAGE > LDS_X ? 2 * STAGE : LDS_X;
    static_assert(NLD >= 1 && LDS <= 160 * 1024, "tile");
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

template <int HD, int RB, bool F16>
__global__ void __launch_bounds__(512) kv8_prefill_kernel(const Kv8PrefArgs a) {
    using Cf = Kv8PrefCfg<HD, RB>;
    constexpr int DC = Cf::DC, DB = Cf::DB, KS = Cf::KS, NLD = Cf::NLD, SLOTS = Cf::SLOTS;
    extern __shared__ __align__(16) unsigned char smem[];
    const Kv8Problem &p = a.p;
    const Kv8 &kc = p.c;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, ln = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rg = wave >> 1, kg = wave & 1;
    const int G = p.NQ / kc.NKV;

    // Work item: KV head, key split, and the tile: tiles of request 0 from its last to its first, then request 1's, ..
    int rest = (int)blockIdx.x;
    const int h = rest % kc.NKV; rest /= kc.NKV;
    const int sp = rest % a.ns; rest /= a.ns;
    int seq = -1, tile = 0;
    for (int s0 = 0; s0 < p.B; s0 += 64) {
        int r0, nr = 0;
        if (s0 + lane < p.B) kv8_rows(p, s0 + lane, r0, nr);
        const int n = (int)(((long long)nr * G + Cf::RR - 1) / Cf::RR), incl = wave_scan64(n);
        const unsigned long long hit = __ballot(incl > rest);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            seq = s0 + l; tile = __builtin_amdgcn_readlane(incl, l) - 1 - rest;
            break;
        }
        rest -= __builtin_amdgcn_readlane(incl, 63);
    }
    if (seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(seq); tile = __builtin_amdgcn_readfirstlane(tile);
    int row0, nr;
    kv8_rows(p, seq, row0, nr);
    const int p0 = min(p.ctx[seq], INT_MAX - nr);
    const int rho0 = tile * Cf::RR, nrows = min(nr * G - rho0, Cf::RR);
    const int tok_a = rho0 / G, tok_b = (rho0 + nrows - 1) / G;        // first and last token of the tile
    int j_lo = win_lo(p0 + tok_a, p.window), j_hi = min(p0 + tok_b, p.max_pos) + 1;
    if (a.ns > 1) {
        const int c = div_by(j_lo, a.part.C, a.Cm) + sp;               // (splits are counted from the tile's first)
        j_lo = max(j_lo, c * a.part.C);
        j_hi = min(j_hi - c * a.part.C, a.part.C) + c * a.part.C;
        if (j_lo >= j_hi) return;
    }
    const int s_lo = j_lo / 64, s_hi = j_hi > j_lo ? (j_hi - 1) / 64 : s_lo - 1;
    const int page = kc.page, last_col = p.max_pos >> kc.lp;
    const int *tab = p.table + (size_t)seq * p.table_stride;
    auto safe = [&](int id) { return (unsigned)id < (unsigned)kc.pages ? id : 0; };
    // A step's pages and scales, loaded a step or two ahead: of the wave's two 16-key pieces and of its K loads through the
    // scalar cache, of the lane's V loads as a vector. (Not picked from one list of all four: the compiler puts a list that is
    // indexed by wave into memory, and reading it back waits for every load in flight.)
    auto piece_id = [&](int s, int piece) { return scalar_load(tab + min((64 * s + 16 * piece) >> kc.lp, last_col)); };
    struct Ids { int a, b, k, v; };
    auto ids_of = [&](int s) {
        return Ids{piece_id(s, 2 * kg), piece_id(s, 2 * kg + 1), piece_id(s, wave >> 1), tab[min((64 * s + 16 * ((lane & 3) ^ ((lane >> 4) & 3))) >> kc.lp, last_col)]};
    };
    struct Scales { float ka, kb, va, vb; bool oka, okb; };
    auto scales_of = [&](const Ids &q) {
        const size_t ca = (size_t)safe(q.a) * kc.NKV + h, cb = (size_t)safe(q.b) * kc.NKV + h;
        return Scales{scalar_load(kc.Ks + ca), scalar_load(kc.Ks + cb), scalar_load(kc.Vs + ca), scalar_load(kc.Vs + cb),
                      (unsigned)q.a < (unsigned)kc.pages, (unsigned)q.b < (unsigned)kc.pages};
    };

    // Step loads. K slot S = (wave NLD + u) 64 + lane: key S / SLOTS, 16-byte column (S % SLOTS) ^ kf(key); a wave's keys lie
    // in one 16-key piece (wave / 2). V slot S: dim S / 4, piece (S % 4) ^ (dim / 4 % 4), which is the same in all u.
    auto kf = [](int key) { return HD == 128 ? ((key >> 1) & 1) | ((key >> 3) & 3) << 1 : (key & 3) | ((key >> 3) & 3) << 2; };
    const int vpiece = (lane & 3) ^ ((lane >> 4) & 3), kpiece = wave >> 1;
    const unsigned lds0 = (unsigned)(uintptr_t)smem;
    unsigned koff[NLD];                                                // K: key in the piece's page rows, column
#pragma unroll
    for (int u = 0; u < NLD; u++) {
        const int S = (wave * NLD + u) * 64 + lane, key = S / SLOTS;
        koff[u] = (unsigned)((key & 15) * HD + (((S % SLOTS) ^ kf(key)) << 4));
    }
    const size_t head_bytes = (size_t)page * HD;
    auto issue = [&](int s, const Ids &q) {
        const unsigned st = lds0 + (unsigned)(s & 1) * Cf::STAGE + (unsigned)wave * NLD * 1024;
        const uint8_t *kb = kc.K + ((size_t)safe(q.k) * kc.NKV + h) * head_bytes + (size_t)((64 * s + 16 * kpiece) & (page - 1)) * HD;
        const uint8_t *vb = kc.V + (size_t)(unsigned)(safe(q.v) * kc.NKV + h) * head_bytes + (unsigned)((wave * NLD * 16 + (lane >> 2)) * page + ((64 * s + 16 * vpiece) & (page - 1)));
#pragma unroll
        for (int u = 0; u < NLD; u++) {
            load_to_lds16(kb + koff[u], st + u * 1024);
            load_to_lds16(vb + 16 * u * page, st + Cf::HALF + u * 1024);
        }
    };
    Ids nxt{0, 0, 0, 0};
    Scales sn{1.f, 1.f, 1.f, 1.f, true, true};
    if (s_lo <= s_hi) {
        const Ids q = ids_of(s_lo);
        nxt = ids_of(min(s_lo + 1, s_hi));
        issue(s_lo, q);
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
        for (int ks = 0; ks < KS; ks++)
            qop[rb][ks] = valid ? *reinterpret_cast<const u32x4 *>(q + 64 * (ks >> 1) + 8 * (ks & 1)) : u32x4{0u, 0u, 0u, 0u};
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
    // K fragment (t, d) of the lane: row key 32 kg + 8 (ln / 4) + 4 t + ln % 4, slot (4 d + g) ^ kf. kf does not depend on t
    // or kg at HD 256 and 512 and not on t at 128 either.
    const int krow = 32 * kg + 8 * (ln >> 2) + (ln & 3);
    const unsigned kaddr = (unsigned)krow * HD + ((unsigned)(g ^ kf(krow)) << 4);
    const unsigned vaddr = Cf::HALF + (unsigned)ln * 64 + ((unsigned)((2 * kg + (g >> 1)) ^ ((ln >> 2) & 3)) << 4) + 8 * (g & 1);

    for (int s = s_lo; s <= s_hi; s++) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // stage s has landed, from every wave
        __syncthreads();
        const Scales sc = sn;
        if (s < s_hi) {
            issue(s + 1, nxt);
            sn = scales_of(nxt);
            nxt = ids_of(min(s + 2, s_hi));
        }
        const int jw = 64 * s + 32 * kg;
        bool any = false;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) any |= jw <= whi[rb] && jw + 31 >= wlo[rb];
        if (!any) continue;                                            // (wave-uniform; the barriers are above)
        f32x4 st[2][RB];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int rb = 0; rb < RB; rb++) st[t][rb] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (opaque bases: the fragments' addresses are formed at their reads, not held across the loop)
        unsigned ka = lds0 + kaddr + (unsigned)(s & 1) * Cf::STAGE, va = lds0 + vaddr + (unsigned)(s & 1) * Cf::STAGE;
        asm volatile("" : "+v"(ka), "+v"(va));
        u32x4 kw[2][2];
        auto read_k = [&](int d) {
#pragma unroll
            for (int t = 0; t < 2; t++) kw[d & 1][t] = *lds_at<u32x4>((ka ^ (64 * d)) + 4 * t * HD);
        };
        read_k(0);
#pragma unroll
        for (int d = 0; d < DC; d++) {
            if (d + 1 < DC) read_k(d + 1);
            __builtin_amdgcn_sched_barrier(0);
            const u32x4 (&w)[2] = kw[d & 1];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const u32x4 k0 = e4m3_op<F16>(w[t][0], w[t][1]), k1 = e4m3_op<F16>(w[t][2], w[t][3]);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) st[t][rb] = mfma16<F16>(k0, qop[rb][2 * d], st[t][rb]);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) st[t][rb] = mfma16<F16>(k1, qop[rb][2 * d + 1], st[t][rb]);
            }
        }
        const bool up = g >= 2, ok = up ? sc.okb : sc.oka;             // the lane's 8 keys are in piece g / 2 of the wave's
        const float f = (up ? sc.kb : sc.ka) * a.sl2, ev = up ? (float)exp_of(sc.vb) : (float)exp_of(sc.va);
        const float iv = up ? pow2i(-exp_of(sc.vb)) : pow2i(-exp_of(sc.va));
        const bool part = jw < j_lo || jw + 32 > j_hi || !(sc.oka & sc.okb);
        u32x4 pf[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            float tv[8];
#pragma unroll
            for (int i = 0; i < 8; i++) tv[i] = __builtin_fmaf(st[i >> 2][rb][i & 3], f, ev);
            const bool full = !part && jw >= lo_max[rb] && jw + 31 <= pos_min[rb];
            if (!full) {
                const int kl = max(j_lo, win_lo(rpos[rb], p.window)) - jw - 8 * g, kh = ok ? min(j_hi - 1, rpos[rb]) - jw - 8 * g : -1;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if ((i < kl) | (i > kh)) tv[i] = kNegInf;
            }
            float mx = tv[0];
#pragma unroll
            for (int i = 1; i < 8; i++) mx = fmaxf(mx, tv[i]);
            mx = max_over_groups(mx);
            const float mn = mx > m[rb] + move ? mx - head : m[rb];
            if (__any(mn != m[rb])) {
                const float al = mn == m[rb] ? 1.f : fast_exp2(m[rb] - mn);
                l[rb] *= al; m[rb] = mn;
#pragma unroll
                for (int d = 0; d < DB; d++) acc[rb][d] *= al;
            }
            const float mz = m[rb] == kNegInf ? 0.f : m[rb];           // (no key yet: every 2^(-inf) is 0)
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                tv[i] = fast_exp2(tv[i] - mz);
                sum += tv[i];
            }
            l[rb] = __builtin_fmaf(sum, iv, l[rb]);
            pf[rb] = u32x4{pack2<true>(tv[0], tv[1]), pack2<true>(tv[2], tv[3]), pack2<true>(tv[4], tv[5]), pack2<true>(tv[6], tv[7])};
        }
        if (part) {
            // Bytes that are no token of the request's weigh nothing, NaN codes neither: cleared in LDS, in the wave's own 32
            // keys (the other row groups clear the same ones before they read them). Rare, and a mask in the loop below would
            // cost 2 operations per fragment of 8, a second copy of the loop 64 registers.
            const int k0 = ok ? max(j_lo - jw - 8 * g, 0) : 8, k1 = min(j_hi - jw - 8 * g, 8);
            u32x2 keep;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int x = min(max(k0 - 4 * w, 0), 4), y = min(max(k1 - 4 * w, 0), 4);
                keep[w] = (y >= 4 ? 0xffffffffu : (1u << (8 * y)) - 1u) & ~(x >= 4 ? 0xffffffffu : (1u << (8 * x)) - 1u);
            }
#pragma unroll 1
            for (int d = 0; d < DB; d++) {
                const u32x2 w = *lds_at<u32x2>(va + 1024 * d);
                *lds_at<u32x2>(va + 1024 * d) = w & keep;
            }
        }
        constexpr int VB = 4;                                          // dim blocks read ahead
        u32x2 vw[2][VB];
        auto read_v = [&](int b) {
#pragma unroll
            for (int x = 0; x < VB; x++) vw[b & 1][x] = *lds_at<u32x2>(va + 1024 * (b * VB + x));
        };
        read_v(0);
#pragma unroll
        for (int b = 0; b < DB / VB; b++) {
            if (b + 1 < DB / VB) read_v(b + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < VB; x++) {
                const u32x4 v = e4m3_op<true>(vw[b & 1][x][0], vw[b & 1][x][1]);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) acc[rb][b * VB + x] = mfma16<true>(v, pf[rb], acc[rb][b * VB + x]);
            }
        }
    }

    // Merge of the two key groups: each wave finishes half of the dims of its rows and hands the other half over.
    float *xb = reinterpret_cast<float *>(smem), *stm = xb + (size_t)Cf::NW * RB * 16 * Cf::XSTR, *stl = stm + Cf::NW * RB * 16;
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        l[rb] = sum_over_groups(l[rb]);
        if (g == 0) { stm[(wave * RB + rb) * 16 + ln] = m[rb]; stl[(wave * RB + rb) * 16 + ln] = l[rb]; }
        float *x = xb + ((size_t)(wave * RB + rb) * 16 + ln) * Cf::XSTR + 4 * g;
#pragma unroll
        for (int d = 0; d < DB / 2; d++) {
            const f32x4 a0 = acc[rb][d], a1 = acc[rb][DB / 2 + d];     // (by value: a choice of addresses would put acc in memory)
            f32x4 give;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                give[i] = kg ? a0[i] : a1[i];
                acc[rb][d][i] = kg ? a1[i] : a0[i];                    // what it keeps
            }
            *reinterpret_cast<f32x4 *>(x + 16 * d) = give;
        }
    }
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int lrow = (rg * RB + rb) * 16 + ln, rho = rho0 + lrow, o = (wave ^ 1) * RB + rb;
        if (lrow >= nrows) continue;
        const float mo = stm[o * 16 + ln], lo = stl[o * 16 + ln], M = fmaxf(m[rb], mo);
        const float f0 = kv8_weight(m[rb], l[rb], M), f1 = kv8_weight(mo, lo, M);
        // (the sum and each product in key-group order, whichever wave forms them)
        const float L = kg ? lo * f1 + l[rb] * f0 : l[rb] * f0 + lo * f1;
        const float *x = xb + ((size_t)o * 16 + ln) * Cf::XSTR + 4 * g;
        const size_t row = (size_t)(row0 + rho / G) * p.NQ + h * G + rho % G;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int dim0 = kg * (HD / 2) + 4 * g;
        const int c = a.ns > 1 ? div_by(j_lo, a.part.C, a.Cm) : 0;
        const size_t px = row * a.part.ns + c;
#pragma unroll
        for (int d = 0; d < DB / 2; d++) {
            const f32x4 mine = acc[rb][d], other = *reinterpret_cast<const f32x4 *>(x + 16 * d);
            f32x4 v = mine * f0 + other * f1;
            if (a.ns > 1) {
                *reinterpret_cast<f32x4 *>(a.part.acc + px * HD + dim0 + 16 * d) = v;
                continue;
            }
            v *= inv;
            kv8_store4(p, row * HD + dim0 + 16 * d, v);
        }
        if (kg == 0 && g == 0) {
            if (a.ns > 1) { a.part.m[px] = M; a.part.l[px] = L; }
            else if (p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
        }
    }
}

template <int HD, int RB, bool F16>
static hipError_t launch_pre_k(const Kv8PrefArgs &a, hipStream_t st) {
    using Cf = Kv8PrefCfg<HD, RB>;
    const long long G = a.p.NQ / a.p.c.NKV;
    const long long tiles = std::min((long long)a.p.B * ((a.p.T * G + Cf::RR - 1) / Cf::RR), (long long)a.p.rows * G / Cf::RR + a.p.B);
    const long long wgs = tiles * a.p.c.NKV * a.ns;
    if (wgs > INT_MAX) return hipErrorInvalidConfiguration;
    // (per device; setting it again changes nothing)
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv8_prefill_kernel<HD, RB, F16>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)Cf::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv8_prefill_kernel<HD, RB, F16>), dim3((unsigned)wgs), dim3(512), Cf::LDS, st, a);
    return hipGetLastError();
}
template <int HD, int RB> static hipError_t launch_pre(const Kv8PrefArgs &a, hipStream_t st) {
    return a.p.q_dtype == DT_F16 ? launch_pre_k<HD, RB, true>(a, st) : launch_pre_k<HD, RB, false>(a, st);
}

hipError_t launch_kv8_prefill(const Kv8Problem &p, const Kv8Partials &part, hipStream_t st) {
    Kv8PrefArgs a{p, part, part.C ? div_magic(part.C) : 0u, 1, p.scale * kLog2e};
    const long long G = p.NQ / p.c.NKV;
    if (part.C) {
        long long per = p.max_pos / part.C + 1;
        if (p.window > 0) per = std::min<long long>(per, ((long long)p.window + p.T - 2) / part.C + 2);
        a.ns = (int)std::max(2ll, per);
    }
    const long long big = ((long long)p.T * G + 127) / 128 * p.B * p.c.NKV * a.ns;
    const bool two = big >= 256;
    switch (p.c.HD) {
    case 128: return two ? launch_pre<128, 2>(a, st) : launch_pre<128, 1>(a, st);
    case 256: return two ? launch_pre<256, 2>(a, st) : launch_pre<256, 1>(a, st);
    case 512: return launch_pre<512, 1>(a, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dgx
