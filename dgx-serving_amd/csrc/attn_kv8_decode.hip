// Split-KV attention over the paged 8-bit cache on gfx950: single tokens, short runs, draft trees and prompts that do not fill
// the chip, and the merge of key splits.
//
// A workgroup owns one key chunk of one request and KV head and up to 16 NT of its query rows (token-major: tokens x q-heads
// of the KV head, so a byte of K or V is read once for the whole group). It walks the chunk in steps of 128 keys at absolute
// positions. Its NW waves split a step twice: each computes the scores of 16 KT of its keys against all rows, and, after the
// probabilities went through LDS, the product of all 128 keys with HD / NW of V's dims. So
//   * K and V go from memory to the matrix units through registers alone, and every code is loaded and converted to 16 bits
//     (exactly) once per workgroup: half the accumulators per wave would be twice the conversions, and the other way round;
//   * a wave holds 16 rows x HD / NW dims of the output (16 registers at HD 256 instead of the 64 of a wave that walks its
//     own keys), which leaves registers for 2 to 4 waves per SIMD (OCC below), and there is no merge of waves at the end;
//   * the price is two barriers a step: for the row maxima, and for the probabilities.
// S^T = K Q^T on 16x16x32: a lane's 16-byte load is 16 dims of one key, two operands. O^T += V^T P^T: V pages hold
// [dim][token], so a lane's 16-byte load is 16 consecutive tokens of one dim, and its P operand is 16 neighbouring
// probabilities of its row in LDS.
//
// The V scale 2^e of a key's page is part of its weight: P = 2^(s + e - m) multiplies the bare codes, with m the running
// maximum of s + e, and the row sum takes P 2^-e. So P in f16 (11 bits) is as exact relative to the largest contribution
// as it would be without scales, whatever the scales are. P is kept below 2^14 by holding the reference 2^6 under the
// maximum it was set from: f16's smallest step is then 2^-30 of the largest term.
//
// Chunks and steps lie at absolute keys and a step's wave depends on its position alone: a row's bits do not depend on the
// other requests of the batch.
//
// What bounds it: HBM bytes of K and V, where a call has enough of them (16 requests of 32K keys 5.8 TB/s, 16 of up to 8K 5.0
// without the merge; a kernel that does nothing but read reaches 7.1 here); the steps of the longest workgroup where it has not.
// Conversions (v_cvt_scalef32_pk_f16_fp8 issues at full rate: 4.7 cycles measured, as an fma) and MFMAs take about a tenth of
// their pipes' time at 6 TB/s.
#include "attn_kv8.h"
#include <algorithm>
#include <climits>

namespace dgx {

struct Kv8DecArgs {
    Kv8Problem p;
    Kv8Partials part;
    int C;                            // keys of a chunk
    uint32_t Cm;                      // div_magic(C)
    int nrg;                          // row groups of a KV head
    int spread;                       // > 0: (chunk, KV head) units, which the row groups take in turn
    int direct;                       // one chunk holds every key: O and lse are written here
    float sl2;                        // scale * log2(e)
};

// Work item `rest` -> request, its first chunk, the item's chunk and the keys [lo, hi) of the request's rows; the shorter of a
// request's first and last chunk come behind all others (the scheme and its reasons are find_item's).
// With `all`, a request whose rows have no key at all is an item too (its rows are written in the kernel).
__device__ __forceinline__ bool kv8_find(const Kv8Problem &p, int C, uint32_t M, bool all, int rest, int &seq, int &c_first, int &c, int &lo, int &hi) {
    const int lane = threadIdx.x & 63;
    for (int phase = 0; phase < 2; phase++)
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            int lo_s = 0, hi_s = 0, first = 0, n = 0;
            if (s0 + lane < p.B) {
                int r0, nr;
                kv8_rows(p, s0 + lane, r0, nr);
                const int p0 = kv8_first_pos(p, s0 + lane, nr), pl = p0 + nr - 1;
                lo_s = win_lo(p0, p.window); hi_s = nr > 0 ? min(pl, p.max_pos) + 1 : 0;
                first = div_by(lo_s, C, M);
                n = hi_s > lo_s ? div_by(hi_s - 1, C, M) - first + 1 : all && nr > 0 ? 1 : 0;
            }
            const int kf = min(hi_s, (first + 1) * C) - lo_s, kl = hi_s - max(lo_s, (first + n - 1) * C);
            const int sh = n >= 2 && kf >= kl ? n - 1 : 0;
            const int m = phase == 0 ? max(n - 1, 0) : min(n, 1), incl = wave_scan64(m);
            const unsigned long long hit = __ballot(incl > rest);
            if (hit) {
                const int l = __builtin_ctzll(hit), r = rest - (incl - m);
                const int cc = first + (phase == 1 ? sh : r < sh ? r : r + 1);
                seq = s0 + l;
                c_first = __builtin_amdgcn_readlane(first, l); c = __builtin_amdgcn_readlane(cc, l); lo = __builtin_amdgcn_readlane(lo_s, l); hi = __builtin_amdgcn_readlane(hi_s, l);
                return true;
            }
            rest -= __builtin_amdgcn_readlane(incl, 63);
        }
    return false;
}

template <int HD, int NT>
struct Kv8DecCfg {
    static constexpr int SK = 128;                     // keys of a step
    // Waves. 8 where 4 would not hold the accumulators. (HD 512 with one row group fits 244 registers of 4 waves; 8 take 158 of
    // them. 8 requests of up to 32K in five draws, geometric mean of the 512-key splits: 30.1 us in 4 waves, 27.8 in 8.)
    static constexpr int NW = HD == 512 && NT > 1 ? 8 : 4;
    static constexpr int KT = SK / 16 / NW;            // 16-key tiles of a wave
    static constexpr int RR = 16 * NT;                 // query rows
    static constexpr int DC = HD / 64;                 // 64-dim pieces of a key (one 16-byte load per lane each)
    static constexpr int DB = HD / NW / 16;            // 16-dim output blocks of a wave
    static constexpr int QSTR = HD + 8;                // Q row in LDS: 16 rows on distinct bank quads
    static constexpr int PSTR = SK + 8;                // P row, likewise
    // K through LDS (see load_k): a unit of 16 keys x 64 UD dims at a time, in a place of each wave's own.
    static constexpr bool KLDS = NT == 1 || (NT == 2 && HD <= 256);
    static constexpr int UD = DC < 4 ? DC : 4;
    static constexpr size_t LDS_Q = (size_t)RR * QSTR * 2, LDS_P = (size_t)RR * PSTR * 2, LDS_K = KLDS ? (size_t)NW * 16 * 64 * UD : 0;
    static constexpr size_t LDS_R = (size_t)NW * RR * 4;
    static constexpr size_t LDS = LDS_Q + LDS_P + LDS_R + LDS_K;
    // Waves per SIMD that the registers are held to. (HD 256 with four row groups takes all 256 and spills one, which is written
    // before the loop over the keys and read behind it.)
    static constexpr int OCC = NT > 1 || HD == 512 ? 2 : HD == 256 ? 3 : 4;
};

constexpr float kv8_head = 6.f, kv8_move = 14.f;       // the reference lies 2^6 under its maximum and moves above 2^14

// STREAM: no other workgroup reads these keys; non-temporal loads sustain a higher HBM rate.
template <int HD, int NT, bool F16, bool STREAM>
__global__ void __launch_bounds__((Kv8DecCfg<HD, NT>::NW * 64), (Kv8DecCfg<HD, NT>::OCC)) kv8_decode_kernel(const Kv8DecArgs a) {
    using Cf = Kv8DecCfg<HD, NT>;
    constexpr int NW = Cf::NW, KT = Cf::KT, DC = Cf::DC, DB = Cf::DB, SK = Cf::SK;
    constexpr bool KLDS = Cf::KLDS;
    extern __shared__ __align__(16) unsigned char smem[];
    const Kv8Problem &p = a.p;
    const Kv8 &kc = p.c;
    // Workgroups of one (chunk, KV head) and different row groups read the same keys: 8 apart, on one XCD, if there are enough
    // of them for all XCDs.
    int unit, rg;
    if (a.spread) { rg = a.nrg - 1 - (int)blockIdx.x / a.spread; unit = (int)blockIdx.x % a.spread; }
    else { unit = (int)(blockIdx.x / (8 * a.nrg)) * 8 + (int)(blockIdx.x & 7); rg = a.nrg - 1 - (int)(blockIdx.x >> 3) % a.nrg; }
    int seq, c_first, c, lo, hi;
    if (!kv8_find(p, a.C, a.Cm, a.direct, unit / kc.NKV, seq, c_first, c, lo, hi)) return;
    seq = __builtin_amdgcn_readfirstlane(seq); c = __builtin_amdgcn_readfirstlane(c);
    const int place = __builtin_amdgcn_readfirstlane(c - c_first);     // of the chunk among the request's
    lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi);
    const int h = unit % kc.NKV, G = p.NQ / kc.NKV;
    int row0, nr;
    kv8_rows(p, seq, row0, nr);
    row0 = __builtin_amdgcn_readfirstlane(row0); nr = __builtin_amdgcn_readfirstlane(nr);
    const int rho0 = rg * Cf::RR, nrows = min(nr * G - rho0, Cf::RR);
    if (nrows <= 0) return;
    // Keys of the chunk that some row of this group attends.
    const int p0 = min(scalar_load(p.ctx + seq), INT_MAX - nr) /* kv8_first_pos */, t_a = rho0 / G, t_b = (rho0 + nrows - 1) / G;
    const int j_lo = max(c * a.C, win_lo(p0 + t_a, p.window)), j_hi = min(min(hi, p0 + t_b + 1) - c * a.C, a.C) + c * a.C;
    if (j_lo >= j_hi && !a.direct) return;

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, ln = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int page = kc.page;
    const int *tab = p.table + (size_t)seq * p.table_stride;
    const int last_col = p.max_pos >> kc.lp;
    auto safe = [&](int id) { return (unsigned)id < (unsigned)kc.pages ? id : 0; };

    // A step's pages and scales, loaded a step or two ahead: of the wave's own KT 16-key pieces through the scalar cache, of
    // the lane's V columns (the pieces g and 4 + g) as vectors. (Not picked from one list of all eight: the compiler puts a list
    // that is indexed by wave into memory, and reading it back waits for every load in flight.)
    struct Own { int id[KT]; };
    struct Scales { float k[KT], v[KT]; };
    auto own_ids = [&](int s) {
        Own q;
#pragma unroll
        for (int t = 0; t < KT; t++) q.id[t] = scalar_load(tab + min((SK * s + 16 * (KT * wave + t)) >> kc.lp, last_col));
        return q;
    };
    auto scales_of = [&](const Own &q) {
        Scales r;
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const size_t cell = (size_t)safe(q.id[t]) * kc.NKV + h;
            r.k[t] = scalar_load(kc.Ks + cell); r.v[t] = scalar_load(kc.Vs + cell);
        }
        return r;
    };
    auto v_id = [&](int s, int k) { return tab[min((SK * s + 64 * k + 16 * g) >> kc.lp, last_col)]; };
    const size_t head_bytes = (size_t)page * HD;
    auto fetch = [](const uint8_t *q) {
        if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(q));
        else return *reinterpret_cast<const u32x4 *>(q);
    };
    u32x4 kr[KT][DC], vr[2][DB];
    // K of the wave, tile t: key 16 (KT wave + t) + ln of the step. A fragment is 16 dims of each of 16 keys: loaded as such,
    // a load touches 64 bytes of 16 rows and takes five times as long to issue as one of whole rows (32 of them 1.1 us a step
    // at HD 256, more than the rest of a step that waits for nothing). With few rows K is therefore loaded in whole rows
    // and goes through LDS, 16-byte slots XOR-swizzled by the key; with more, Q takes the LDS and its bandwidth.
    constexpr int UD = Cf::UD;
    auto kswz = [](int key) { return UD == 4 ? key : key >> 1; };
    unsigned klane[KLDS ? UD : 1];
#pragma unroll
    for (int u = 0; u < (KLDS ? UD : 1); u++) {
        const int S = 64 * u + lane;
        klane[u] = KLDS ? (unsigned)(S / (4 * UD) * HD + S % (4 * UD) * 16) : (unsigned)(ln * HD + 16 * g);
    }
    auto load_k = [&](int s, const Own &q) {
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const uint8_t *b = kc.K + ((size_t)safe(q.id[t]) * kc.NKV + h) * head_bytes + (size_t)((SK * s + 16 * (KT * wave + t)) & (page - 1)) * HD;
#pragma unroll
            for (int d = 0; d < DC; d++) kr[t][d] = fetch(b + (KLDS ? klane[d % UD] + 64 * UD * (d / UD) : klane[0] + 64 * d));
        }
    };
    const unsigned vlane = (unsigned)((wave * (HD / NW) + ln) * page + ((16 * g) & (page - 1)));
    auto load_v = [&](int k, int id) {                                 // dims of the wave, 16 tokens from 64 k + 16 g of the step
        const uint8_t *b = kc.V + (size_t)(unsigned)(safe(id) * kc.NKV + h) * head_bytes + vlane;
#pragma unroll
        for (int d = 0; d < DB; d++) vr[k][d] = fetch(b + 16 * d * page);
    };

    const int s1 = j_hi > j_lo ? (j_hi - 1) / SK : -1;
    int s = j_lo / SK;
    Own nxt{};
    Scales sn{};
    bool okn = true;                                                   // the wave's pages are in the pool
    int vi0 = 0, vi1 = 0, vn0 = 0, vn1 = 0;                            // V pages of this step and of the next one
    auto own_ok = [&](const Own &q) {
        bool r = true;
#pragma unroll
        for (int t = 0; t < KT; t++) r &= (unsigned)q.id[t] < (unsigned)kc.pages;
        return r;
    };
    Own cur{};
    if (s <= s1) {
        cur = own_ids(s);
        vi0 = v_id(s, 0); vi1 = v_id(s, 1);
        nxt = own_ids(min(s + 1, s1));
        load_k(s, cur);
        load_v(0, vi0); load_v(1, vi1);
        vn0 = v_id(min(s + 1, s1), 0); vn1 = v_id(min(s + 1, s1), 1);
        sn = scales_of(cur);
        okn = own_ok(cur);
    }
    // Q rows, zeros past the last.
    uint16_t *qs = reinterpret_cast<uint16_t *>(smem), *ps = reinterpret_cast<uint16_t *>(smem + Cf::LDS_Q);
    float *red = reinterpret_cast<float *>(smem + Cf::LDS_Q + Cf::LDS_P);
    unsigned char *ks = smem + Cf::LDS_Q + Cf::LDS_P + Cf::LDS_R + (size_t)wave * 16 * 64 * UD;
    unsigned kw[KLDS ? UD : 1];                                        // where the lane's loads go in a unit, and its fragment's row
#pragma unroll
    for (int u = 0; u < (KLDS ? UD : 1); u++) {
        const int S = 64 * u + lane, key = S / (4 * UD);
        kw[u] = (unsigned)(key * 64 * UD + ((S % (4 * UD) ^ kswz(key)) << 4));
    }
    const unsigned kfrag = (unsigned)(ln * 64 * UD + ((g ^ kswz(ln)) << 4));
    for (int i = tid; i < Cf::RR * (HD / 8); i += NW * 64) {
        const int R = i / (HD / 8), rho = rho0 + R;
        u32x4 v{0u, 0u, 0u, 0u};
        if (R < nrows)
            v = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(p.Q) + ((size_t)(row0 + rho / G) * p.NQ + h * G + rho % G) * HD + (i % (HD / 8)) * 8);
        *reinterpret_cast<u32x4 *>(qs + R * Cf::QSTR + (i % (HD / 8)) * 8) = v;
    }
    // Rows of the lane (16 nt + ln) and the bounds within which no row needs its mask.
    int rpos[NT];
    uint32_t ranc[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int R = 16 * nt + ln, t = R < nrows ? (rho0 + R) / G : 0;
        rpos[nt] = R < nrows ? p0 + t : -1;
        ranc[nt] = p.anc && R < nrows ? p.anc[row0 + t] : 0u;
    }
    const int lo_max = win_lo(p0 + t_b, p.window), pos_min = p.anc ? p0 - 1 : p0 + t_a;
    __syncthreads();

    float m[NT], l[NT];
    f32x4 acc[NT][DB];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = kNegInf; l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++) acc[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (; s <= s1; s++) {
        const int j0 = SK * s, jw = j0 + 16 * KT * wave;
        const Scales sc = sn;
        const Own now = cur, next = nxt;
        const bool pages_ok = okn;
        // (Without a branch around them, and taken over at the end of the step: the scalar loads then wait with the K loads.)
        const Scales s2 = scales_of(next);
        const Own n2 = own_ids(min(s + 2, s1));
        f32x4 st[KT][NT];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) st[t][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
        unsigned qo = (unsigned)(ln * Cf::QSTR + 16 * g);              // (opaque: the fragments are read here, not held across steps)
        asm volatile("" : "+v"(qo));
        if constexpr (KLDS) {
            // (A wave's LDS operations run in their order: no wait between a unit's writes, its reads and the next one's writes.)
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int x = 0; x < DC / UD; x++) {
#pragma unroll
                    for (int u = 0; u < UD; u++) *reinterpret_cast<u32x4 *>(ks + kw[u]) = kr[t][x * UD + u];
                    __builtin_amdgcn_wave_barrier();
                    u32x4 kf[UD];
#pragma unroll
                    for (int u = 0; u < UD; u++) kf[u] = *reinterpret_cast<const u32x4 *>(ks + (kfrag ^ (64 * u)));
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int u = 0; u < UD; u++) {
                        const u32x4 k0 = e4m3_op<F16>(kf[u][0], kf[u][1]), k1 = e4m3_op<F16>(kf[u][2], kf[u][3]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint16_t *q = qs + qo + 16 * nt * Cf::QSTR + 64 * (x * UD + u);
                            st[t][nt] = mfma16<F16>(k0, *reinterpret_cast<const u32x4 *>(q), st[t][nt]);
                            st[t][nt] = mfma16<F16>(k1, *reinterpret_cast<const u32x4 *>(q + 8), st[t][nt]);
                        }
                    }
                }
        } else {
#pragma unroll
            for (int d = 0; d < DC; d++) {
                u32x4 k0[KT], k1[KT];
#pragma unroll
                for (int t = 0; t < KT; t++) { k0[t] = e4m3_op<F16>(kr[t][d][0], kr[t][d][1]); k1[t] = e4m3_op<F16>(kr[t][d][2], kr[t][d][3]); }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const u32x4 q0 = *reinterpret_cast<const u32x4 *>(qs + qo + 16 * nt * Cf::QSTR + 64 * d);
                    const u32x4 q1 = *reinterpret_cast<const u32x4 *>(qs + qo + 16 * nt * Cf::QSTR + 64 * d + 8);
#pragma unroll
                    for (int t = 0; t < KT; t++) st[t][nt] = mfma16<F16>(k0[t], q0, st[t][nt]);
#pragma unroll
                    for (int t = 0; t < KT; t++) st[t][nt] = mfma16<F16>(k1[t], q1, st[t][nt]);
                }
            }
        }
        // (From here to the step's end a wave goes before one at its scores: its workgroup waits for it at the barriers. 1024
        // tokens causal 32.0 -> 29.6 us, tree verify 68.5 -> 66.3.)
        __builtin_amdgcn_s_setprio(1);
        int vf0 = 0, vf1 = 0;
        if (s < s1) {
            vf0 = v_id(min(s + 2, s1), 0); vf1 = v_id(min(s + 2, s1), 1);
            load_k(s + 1, next);
        }
        const bool full = pages_ok && jw >= j_lo && jw + 16 * KT <= j_hi && jw >= lo_max && jw + 16 * KT - 1 <= pos_min;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float mx = kNegInf;
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const float kf = sc.k[t] * a.sl2, ev = (float)exp_of(sc.v[t]);
#pragma unroll
                for (int i = 0; i < 4; i++) st[t][nt][i] = __builtin_fmaf(st[t][nt][i], kf, ev);
                if (!full) {
                    const int kb = jw + 16 * t + 4 * g, kl = max(j_lo, win_lo(rpos[nt], p.window)) - kb;
                    const int kh = (unsigned)now.id[t] < (unsigned)kc.pages ? min(j_hi - 1, rpos[nt]) - kb : -1;
                    // Bit i: key kb + i is hidden by the tree (tokens from 32 on, and those whose bit is not set).
                    const int d = kb - p0;
                    const uint32_t tree = !p.anc ? 0u : ~(uint32_t)((d <= -32 ? ~0ull : d < 0 ? ((uint64_t)ranc[nt] << -d) | ((1ull << -d) - 1) : d < 32 ? (uint64_t)(ranc[nt] >> d) : 0ull));
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if ((i < kl) | (i > kh) | (bool)((tree >> i) & 1u)) st[t][nt][i] = kNegInf;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[t][nt][i]);
            }
            mx = max_over_groups(mx);
            if (g == 0) red[wave * Cf::RR + 16 * nt + ln] = mx;
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float mx = red[16 * nt + ln];
#pragma unroll
            for (int w = 1; w < NW; w++) mx = fmaxf(mx, red[w * Cf::RR + 16 * nt + ln]);
            const float mn = mx > m[nt] + kv8_move ? mx - kv8_head : m[nt];
            if (__any(mn != m[nt])) {
                const float al = mn == m[nt] ? 1.f : fast_exp2(m[nt] - mn);
                l[nt] *= al; m[nt] = mn;
#pragma unroll
                for (int d = 0; d < DB; d++) acc[nt][d] *= al;
            }
            const float mz = m[nt] == kNegInf ? 0.f : m[nt];           // (no key yet: every 2^(-inf) is 0)
#pragma unroll
            for (int t = 0; t < KT; t++) {
                float pv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) pv[i] = fast_exp2(st[t][nt][i] - mz);
                l[nt] = __builtin_fmaf((pv[0] + pv[1]) + (pv[2] + pv[3]), pow2i(-exp_of(sc.v[t])), l[nt]);
                *reinterpret_cast<u32x2 *>(ps + (16 * nt + ln) * Cf::PSTR + 16 * (KT * wave + t) + 4 * g) =
                    u32x2{pack2<true>(pv[0], pv[1]), pack2<true>(pv[2], pv[3])};
            }
        }
        __syncthreads();
        const bool vok0 = (unsigned)vi0 < (unsigned)kc.pages, vok1 = (unsigned)vi1 < (unsigned)kc.pages;
        if (j0 < j_lo || j0 + SK > j_hi || __any(!(vok0 & vok1))) {    // bytes that are no token of the request's: any code, NaN too
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int jb = j0 + 64 * k + 16 * g;
                const int k0 = (k ? vok1 : vok0) ? max(j_lo - jb, 0) : 16, k1 = min(j_hi - jb, 16);
                u32x4 keep;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const int x = min(max(k0 - 4 * w, 0), 4), y = min(max(k1 - 4 * w, 0), 4);      // bytes [x, y) of word w
                    keep[w] = (y >= 4 ? 0xffffffffu : (1u << (8 * y)) - 1u) & ~(x >= 4 ? 0xffffffffu : (1u << (8 * x)) - 1u);
                }
#pragma unroll
                for (int d = 0; d < DB; d++) vr[k][d] &= keep;
            }
        }
        unsigned po = (unsigned)(ln * Cf::PSTR + 16 * g);
        asm volatile("" : "+v"(po));
#pragma unroll
        for (int k = 0; k < 2; k++) {
            u32x4 pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) pf[nt][e] = *reinterpret_cast<const u32x4 *>(ps + po + 16 * nt * Cf::PSTR + 64 * k + 8 * e);
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const u32x4 v0 = e4m3_op<true>(vr[k][d][0], vr[k][d][1]), v1 = e4m3_op<true>(vr[k][d][2], vr[k][d][3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[nt][d] = mfma16<true>(v0, pf[nt][0], acc[nt][d]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[nt][d] = mfma16<true>(v1, pf[nt][1], acc[nt][d]);
            }
        }
        if (s < s1) { load_v(0, vn0); load_v(1, vn1); }
        __builtin_amdgcn_s_setprio(0);
        vi0 = vn0; vi1 = vn1; vn0 = vf0; vn1 = vf1;
        cur = next; nxt = n2; sn = s2; okn = own_ok(next);
    }

    // Row sums over the waves, in their order; m is the same in all.
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        l[nt] = sum_over_groups(l[nt]);
        if (g == 0) red[wave * Cf::RR + 16 * nt + ln] = l[nt];
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int R = 16 * nt + ln, rho = rho0 + R;
        if (R >= nrows) continue;
        float L = red[R];
#pragma unroll
        for (int w = 1; w < NW; w++) L += red[w * Cf::RR + R];
        const size_t row = (size_t)(row0 + rho / G) * p.NQ + h * G + rho % G;
        const int dim0 = wave * (HD / NW) + 4 * g;
        if (a.direct) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int d = 0; d < DB; d++) kv8_store4(p, row * HD + dim0 + 16 * d, acc[nt][d] * inv);
            if (wave == 0 && g == 0 && p.lse) p.lse[row] = L == 0.f ? kNegInf : (m[nt] + __builtin_amdgcn_logf(L)) * kLn2;
        } else {
            const size_t x = row * a.part.ns + place;
#pragma unroll
            for (int d = 0; d < DB; d++) *reinterpret_cast<f32x4 *>(a.part.acc + x * HD + dim0 + 16 * d) = acc[nt][d];
            if (wave == 0 && g == 0) { a.part.m[x] = m[nt]; a.part.l[x] = L; }
        }
    }
}

// ---------------------------------------------------------------- merge of key splits
// One workgroup per (row, q-head, 128 dims): 32 threads hold 4 dims each and 8 phases take the splits in turn; the phases are
// added in their order. The weights of the splits are formed once, a thread each (256 at a time). Three dependent reads
// whatever the number of splits: 64 of them at HD 512 took 15.5 us when every thread walked the maxima and sums itself.
// Also writes the rows that attend nothing (O = 0, lse = -inf).
// Where there are many rows, a wave of its own for each (row, q-head, 256 dims) does it without a barrier.
struct Kv8CombArgs {
    Kv8Problem p;
    Kv8Partials part;
    uint32_t Cm;
    int by_row;                       // items are rows of the buffers, not the T rows that each request has at most
};

// The places [c0, c0 + n) of the splits of item bt's row among its request's, and the row's place among the partials' rows;
// false past the last row. All lanes of a wave ask for the same item.
__device__ __forceinline__ bool comb_row(const Kv8CombArgs &a, int bt, int head, size_t &row, int &c0, int &n) {
    const Kv8Problem &p = a.p;
    int b, i, row0, nr;
    if (a.by_row) {                                                    // the request: as many begin at or before the row
        const int lane = threadIdx.x & 63;
        b = -1;
        for (int s0 = 0; s0 < p.B; s0 += 64) b += __builtin_popcountll(__ballot(s0 + lane < p.B && p.cu[min(s0 + lane, p.B)] <= bt));
        if (b < 0) return false;
        kv8_rows(p, b, row0, nr);
        i = bt - row0;
    } else {
        b = bt / p.T; i = bt - b * p.T;
        kv8_rows(p, b, row0, nr);
    }
    if ((unsigned)i >= (unsigned)nr) return false;
    const int p0 = kv8_first_pos(p, b, nr), pos = p0 + i, lo = win_lo(pos, p.window), hi = min(pos, p.max_pos);
    const int c_lo = div_by(lo, a.part.C, a.Cm);
    row = (size_t)(row0 + i) * p.NQ + head;
    c0 = c_lo - div_by(win_lo(p0, p.window), a.part.C, a.Cm);
    n = hi >= lo ? div_by(hi, a.part.C, a.Cm) - c_lo + 1 : 0;
    return true;
}

__global__ void __launch_bounds__(256) kv8_combine_kernel(const Kv8CombArgs a) {
    __shared__ __align__(16) float red[8][128];
    __shared__ float wt[256], part_s[2][4];
    const Kv8Problem &p = a.p;
    const int HD = p.c.HD;
    size_t row;
    int c0, n;
    if (!comb_row(a, (int)blockIdx.x, (int)blockIdx.y, row, c0, n)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, d4 = tid & 31, ph = tid >> 5, dim = (int)blockIdx.z * 128 + 4 * d4;
    const float *pm = a.part.m + row * a.part.ns + c0, *pl = a.part.l + row * a.part.ns + c0;
    const float *pa = a.part.acc + (row * a.part.ns + c0) * HD + dim;
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f}, t[4];
    float M = kNegInf, L = 0.f, m0 = kNegInf, l0 = 0.f;
    if (n > 0) {                                                       // the first splits, before their weights are known
        m0 = pm[min(tid, n - 1)]; l0 = pl[min(tid, n - 1)];
#pragma unroll
        for (int x = 0; x < 4; x++) t[x] = *reinterpret_cast<const f32x4 *>(pa + (size_t)min(ph + 8 * x, n - 1) * HD);
    }
    M = m0;
    for (int c = tid + 256; c < n; c += 256) M = fmaxf(M, pm[c]);
#pragma unroll
    for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
    if (lane == 0) part_s[0][wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(part_s[0][0], part_s[0][1]), fmaxf(part_s[0][2], part_s[0][3]));
    for (int b0 = 0; b0 < n; b0 += 256) {
        if (b0) __syncthreads();
        if (b0 + tid < n) {
            const float lc = b0 ? pl[b0 + tid] : l0;
            wt[tid] = kv8_weight(b0 ? pm[b0 + tid] : m0, lc, M);
            L += lc * wt[tid];
        }
        __syncthreads();
        const int nb = min(256, n - b0);
        if (b0 == 0) {
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (ph + 8 * x < nb) v += t[x] * wt[ph + 8 * x];
        }
#pragma unroll 4
        for (int c = b0 ? ph : ph + 32; c < nb; c += 8) v += *reinterpret_cast<const f32x4 *>(pa + (size_t)(b0 + c) * HD) * wt[c];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) L += __shfl_xor(L, d);
    if (lane == 0) part_s[1][wave] = L;
    *reinterpret_cast<f32x4 *>(&red[ph][4 * d4]) = v;
    __syncthreads();
    if (ph) return;
    L = (part_s[1][0] + part_s[1][1]) + (part_s[1][2] + part_s[1][3]);
#pragma unroll
    for (int x = 1; x < 8; x++) v += *reinterpret_cast<const f32x4 *>(&red[x][4 * d4]);
    kv8_store4(p, row * HD + dim, v * (L == 0.f ? 0.f : 1.f / L));
    if (tid == 0 && blockIdx.z == 0 && p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
}

template <int NP>   // 2 (HD 128): the halves of the wave take the splits in turn
__global__ void __launch_bounds__(256) kv8_combine_rows_kernel(const Kv8CombArgs a, int item0, unsigned units) {
    const Kv8Problem &p = a.p;
    const int HD = p.c.HD, lane = threadIdx.x & 63, per = HD > 256 ? HD / 256 : 1;
    const unsigned u = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (u >= units) return;
    const int it = (int)(u / (unsigned)(p.NQ * per)), hs = (int)u - it * p.NQ * per, head = hs / per, bt = item0 + it;
    size_t row;
    int c0, n;
    if (!comb_row(a, bt, head, row, c0, n)) return;
    const float *pm = a.part.m + row * a.part.ns + c0, *pl = a.part.l + row * a.part.ns + c0;
    const int ph = NP == 2 ? lane >> 5 : 0, dim = (hs - head * per) * 256 + 4 * (NP == 2 ? lane & 31 : lane);
    const float *pa = a.part.acc + (row * a.part.ns + c0) * HD + dim;
    float M = kNegInf;
    for (int c = lane; c < n; c += 64) M = fmaxf(M, pm[c]);
#pragma unroll
    for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    for (int b0 = 0; b0 < n; b0 += 64) {
        const float lc = b0 + lane < n ? pl[b0 + lane] : 0.f;
        const float w = b0 + lane < n ? kv8_weight(pm[b0 + lane], lc, M) : 0.f;
        L += lc * w;
        const int nb = min(64, n - b0);
        for (int c = 0; c < nb; c += 8 * NP) {                         // eight loads in flight; past the last split: its value, no weight
            f32x4 t[8];
#pragma unroll
            for (int x = 0; x < 8; x++) t[x] = *reinterpret_cast<const f32x4 *>(pa + (size_t)(b0 + min(c + NP * x + ph, nb - 1)) * HD);
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const float wx = __shfl(w, min(c + NP * x + ph, 63));
                if (c + NP * x + ph < nb) v += t[x] * wx;
            }
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) L += __shfl_xor(L, d);
    if constexpr (NP == 2) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += __shfl_xor(v[e], 32);
        if (ph) return;
    }
    kv8_store4(p, row * HD + dim, v * (L == 0.f ? 0.f : 1.f / L));
    if (lane == 0 && hs == head * per && p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
}

hipError_t launch_kv8_combine(const Kv8Problem &p, const Kv8Partials &part, hipStream_t st) {
    const int per = p.c.HD > 256 ? p.c.HD / 256 : 1;
    const bool by_row = p.cu && (long long)p.B * p.T > p.rows;        // (ragged rows: most of B * T are none)
    const Kv8CombArgs a{p, part, div_magic(part.C), by_row ? 1 : 0};
    const int items = by_row ? p.rows : p.B * p.T;
    // 16 trees of 8 tokens x 24 q-heads in up to 16 splits at HD 256: 12.8 us in workgroups, 7.7 in waves.
    if ((long long)items * p.NQ * per < 1024) {
        hipLaunchKernelGGL(kv8_combine_kernel, dim3((unsigned)items, (unsigned)p.NQ, (unsigned)p.c.HD / 128), dim3(256), 0, st, a);
        return hipGetLastError();
    }
    const int most = (1 << 25) / (p.NQ * per);                         // items of a launch: 2^31 threads
    for (int i0 = 0;; i0 += most) {
        const int n = std::min(most, items - i0);
        const unsigned units = (unsigned)n * (unsigned)(p.NQ * per);
        const dim3 g4((units + 3) / 4);
        if (p.c.HD == 128) hipLaunchKernelGGL(kv8_combine_rows_kernel<2>, g4, dim3(256), 0, st, a, i0, units);
        else hipLaunchKernelGGL(kv8_combine_rows_kernel<1>, g4, dim3(256), 0, st, a, i0, units);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || items - i0 <= most) return e;
    }
}

// ---------------------------------------------------------------- launch
template <int HD, int NT, bool F16, bool STREAM>
static hipError_t launch_dec_k(const Kv8DecArgs &a, dim3 grid, hipStream_t st) {
    using Cf = Kv8DecCfg<HD, NT>;
    static_assert(Cf::LDS <= 64 * 1024, "LDS");
    hipLaunchKernelGGL((kv8_decode_kernel<HD, NT, F16, STREAM>), grid, dim3(Cf::NW * 64), Cf::LDS, st, a);
    return hipGetLastError();
}
template <int HD, int NT> static hipError_t launch_dec_n(const Kv8DecArgs &a, dim3 grid, hipStream_t st) {
    const bool f16 = a.p.q_dtype == DT_F16;
    if (a.nrg == 1) return f16 ? launch_dec_k<HD, NT, true, true>(a, grid, st) : launch_dec_k<HD, NT, false, true>(a, grid, st);
    return f16 ? launch_dec_k<HD, NT, true, false>(a, grid, st) : launch_dec_k<HD, NT, false, false>(a, grid, st);
}

Kv8Plan kv8_choose(int B, int T, int rows, int NQ, int NKV, int HD, int max_pos, int chunk, int window, bool tree) {
    const long long G = NQ / NKV, hr = T * G;                          // rows of a KV head and request
    long long keys = max_pos + 1ll;
    if (window > 0) keys = std::min<long long>(keys, (long long)window + T - 1);
    const int whole = (max_pos / 128 + 1) * 128;                       // a split that holds every key
    Kv8Plan pl{0, 0, chunk, 1};
    if (tree || hr <= 64) {
        pl.nt = hr <= 16 ? 1 : hr <= 32 || HD == 512 ? 2 : 4;
        // Keys of a split, by the call's K and V in heads of 256 dims. Short ones leave a call to the prologues of its
        // workgroups and the merge, long ones to the longest workgroup. us in 128 | 256 | 384 | 512 | 1024 keys, 24 q-heads over
        // 4 of 256, K and V not in any cache: one request of 9K keys (36K) 16.8, 15.0, 16.5, 19.2, 28.2; 4 of 9K (144K) 28.7,
        // 24.4, 22.0, 24.0, 29.4; 8 of 9K (288K) 45.6, 37.9, 33.2, 36.4, 36.0; 16 of up to 8K (524K) in three draws 33.1, 26.3,
        // 25.0, 25.8, 30.6 | 28.1, 24.7, 22.7, 24.6, 29.8 | 28.0, 21.7, 21.9, 24.1, 30.1; 16 of 9K (576K) 74.4, 65.6, 60.1, 58.8,
        // 59.6; 16 of 32K (2M) 239, 217, 199, 194, 182. At HD 512 8 of up to 32K in five draws 31.4 (geometric mean) in 256, 30.0
        // in 384, 30.1 in 512. With more than 16 rows the partials weigh more: 16 trees of 48 rows over 16K keys (1M) 343,
        // 208, 183, 161, 132; over up to 16K 165, 113, 101, 85.7, 65.9; 4 over 16K (256K) 87.3, 62.9, 59.0, 46.2, 52.0. Up to
        // four steps go without splits and their merge: 256 keys 8.4 us, 11.2 in two splits (4 heads of 128), 9.8 and 11.5 (4 of
        // 256); at 512 it is even at HD 128 (11.7, in four splits 11.2) and behind at HD 256 (14.8 and 12.3).
        const long long work = (long long)B * NKV * keys * HD / 256;
        if (chunk == 0) pl.C = work < 60000 ? 128 : work < 280000 ? 256 : work < 560000 && hr <= 16 && HD <= 256 ? 384 : work < (hr > 16 ? 700000 : 1500000) ? 512 : 1024;
        if (chunk == 0 && keys <= 512) pl.C = whole;
    } else {
        // Tiles of 64 rows. Where they do not fill the chip the split-KV form takes a prompt too: it walks 128 keys a step,
        // and its row groups can be smaller and its keys split. Best split-KV | tiles, us: causal 1400 x 16 q-heads over 8 (352
        // tiles) 41.5 | 46.9, 1500 (376) 46.9 | 50.5, 1024 x 24 over 4 (384) 38.9 | 38.9, 800 x 24 behind 2000 (300) 95.4 | 85.9, 1000
        // x 16 over 8 behind 2000 (250) 76.5 | 79.3; behind a window of 1024 500 x 16 over 8 (125) 30.9 | 38.9, 600 (150) 37.1 | 39.3;
        // HD 512 800 x 16 (200) 38.7 | 47.0, 1024 (256) 49.5 | 55.6, 1500 (375) 92.3 | 77.3.
        const long long n64 = std::min((long long)B * ((hr + 63) / 64), (long long)rows * G / 64 + B) * NKV;
        pl.tile = n64 >= (HD == 512 ? 250 : window > 0 && window <= max_pos ? 140 : keys <= 2304 ? 360 : 280) ? 64 : 0;
        if (!pl.tile) {
            // 200 x 16 q-heads over 8 without a prefix: groups of 16 rows 10.7 us, 32 13.4, 64 18.4; 1000 behind 1000: 74, 56 and
            // 66; 512 behind 4096: 64 rows in 1152-key splits 65, in 1536 72, in 1024 93, no split of 16 rows 93. Fewer workgroups
            // at HD 512: 500 x 16 over 1 behind 4000 113 us unsplit, 141 in 1536; 100 behind 4000 42 in 1024, 52 in 1536, 53 in 512,
            // 104 unsplit. (Groups of 16 or 32 rows for keys of 900 to 1280 are close: 1024 x 16 over 8 31.3 and 32.0, 900 x 24 over
            // 4 37.7 and 33.2, HD 512 800 x 16 43.2 and 38.7.)
            const long long n = HD == 512 ? n64 * 2 : n64, want = HD == 512 ? 200 : 450;
            pl.nt = HD == 512 ? 2 : 4;
            if (chunk == 0 && keys <= 1280) pl.nt = 1, pl.C = whole;
            else if (chunk == 0 && keys <= 2304 && n64 >= 128) pl.nt = 2, pl.C = whole;
            else if (chunk == 0) {
                const long long splits = std::max(1ll, (want + n / 2) / n);
                pl.C = splits == 1 ? whole : (int)std::min(2048ll, std::max(512ll, (keys / splits + 127) / 128 * 128));
            }
        }
    }
    if (pl.C) {
        pl.ns = max_pos / pl.C + 1;
        // The keys of a request's rows behind a window are window + T - 1 neighbours. (Where max_pos reaches a second split there
        // are two places at least: the form with one has no bounds but a request's own.)
        if (window > 0 && pl.ns > 2) pl.ns = (int)std::min<long long>(pl.ns, std::max(2ll, ((long long)window + T + pl.C - 3) / pl.C + 1));
    }
    if (!pl.tile) return pl;
    if (pl.ns == 1) pl.C = 0;
    // Tiles of 128 rows where there are two rounds of them for the 512 workgroups that run at once (one, under a window: its
    // tiles are equally long), else of 64. us of 128 | 64 rows, with the number of the former; HD 256: 6 requests of up to 2500
    // x 24 q-heads over 4 (1330) 331 | 364, other lengths (880) 193 | 216; causal 4096, 16 over 8 (512) 208 | 155, 24 over 4 (768)
    // 225 | 233, 8192 (1024) 524 | 551, two of 4096 (1024) 280 | 309; behind a window of 1024 3000 (375) 77 | 77, 3600 (450) 80 |
    // 83, 4096 (512) 84 | 90, 6000 (750) 137 | 130, 4096 x 24 (768) 135 | 128, behind 512 4096 (512) 56 | 66: best where the rounds
    // are whole. HD 128, 16 over 4: 2 of 2000 (500) 96 | 63, 8 of 1000 (1000) 63 | 69, 4 of 2000 (1000) 100 | 102, one of 8000 (1000)
    // 345 | 300, 4 of 3000 (1500) 191 | 199.
    const long long all = std::min((long long)B * T, (long long)rows) * NQ * pl.ns;
    if (HD < 512 && all >= 128 * (window > 0 && window < max_pos ? 500 : 960)) pl.tile = 128;
    return pl;
}

hipError_t launch_kv8_decode(const Kv8Problem &p, const Kv8Partials &part, const Kv8Plan &pl, hipStream_t st) {
    const int nt = pl.nt, G = p.NQ / p.c.NKV, rows = (int)std::min<long long>((long long)p.T * G, INT_MAX);
    Kv8DecArgs a{p, part, part.C, div_magic(part.C), (rows + 16 * nt - 1) / (16 * nt), 0, part.ns == 1, p.scale * kLog2e};
    const long long raw = (long long)pl.ns * p.B * p.c.NKV, units = a.nrg == 1 || raw < 64 ? raw : (raw + 7) / 8 * 8, wgs = units * a.nrg;
    if (a.nrg == 1 || raw < 64) a.spread = (int)raw;
    if (!kv8_grid_ok(wgs, p.c.HD == 512 && nt > 1 ? 512 : 256)) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs);
    switch (p.c.HD) {
    case 128: return nt == 1 ? launch_dec_n<128, 1>(a, grid, st) : nt == 2 ? launch_dec_n<128, 2>(a, grid, st) : launch_dec_n<128, 4>(a, grid, st);
    case 256: return nt == 1 ? launch_dec_n<256, 1>(a, grid, st) : nt == 2 ? launch_dec_n<256, 2>(a, grid, st) : launch_dec_n<256, 4>(a, grid, st);
    case 512: return nt == 1 ? launch_dec_n<512, 1>(a, grid, st) : launch_dec_n<512, 2>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dgx
