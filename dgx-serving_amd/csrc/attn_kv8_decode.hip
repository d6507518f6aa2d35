// Split-KV attention over the paged 8-bit cache on gfx950: single tokens, short runs and draft trees, and the merge of key
// splits.
//
// A workgroup owns one key chunk of one request and KV head and up to 16 NT of its query rows (token-major: tokens x q-heads
// of the KV head, so a byte of K or V is read once for the whole group). Its waves take the chunk's steps of 64 keys in turn
// and run independent online softmaxes, merged at the end. Per step and wave everything goes from memory to the matrix
// units through registers alone:
//   * S^T = K Q^T on 16x16x32. Tile t (of 4) of a step holds the keys 16 (rho / 4) + 4 t + rho % 4 in its rows rho, so lane
//     group g gets the scores of the 16 consecutive keys 16 g .. 16 g + 15 (4 t + i) of query row ln. A lane's 16-byte load
//     is 16 dims of one key: two MFMA operands after the conversion to 16 bits, which is exact.
//   * O^T += V^T P^T: V pages hold [dim][token], so a lane's 16-byte load is 16 consecutive tokens of one dim, the same 16
//     keys whose probabilities the lane group holds. P never leaves its lane.
// The V scale 2^e of a key's page is part of its weight: P = 2^(s + e - m) multiplies the bare codes, with m the running
// maximum of s + e, and the row sum takes P 2^-e. So P in f16 (11 bits) is as exact relative to the largest contribution
// as it would be without scales, whatever the scales are. P is kept below 2^14 by holding the reference 2^6 under the
// maximum it was set from: f16's smallest step is then 2^-30 of the largest term.
//
// Chunks and steps lie at absolute keys and a step's wave depends on its position alone: a row's bits do not depend on the
// other requests of the batch.
//
// What bounds it: HBM bytes of K and V. Conversions take 1/16 of the VALU's time at 6 TB/s (v_cvt_scalef32_pk_f16_fp8 issues
// at full rate: 4.7 cycles measured, as an fma), MFMAs about a tenth of theirs.
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
    int direct;                       // one chunk holds every key: O and lse are written here
    float sl2;                        // scale * log2(e)
};

// Work item `rest` -> request, chunk and the keys [lo, hi) of the request's rows; the shorter of a request's first and
// last chunk come behind all others (the scheme and its reasons are find_item's).
// With `all`, a request whose rows have no key at all is an item too (its rows are written in the kernel).
__device__ __forceinline__ bool kv8_find(const Kv8Problem &p, int C, uint32_t M, bool all, int rest, int &seq, int &c, int &lo, int &hi) {
    const int lane = threadIdx.x & 63;
    for (int phase = 0; phase < 2; phase++)
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            int lo_s = 0, hi_s = 0, first = 0, n = 0;
            if (s0 + lane < p.B) {
                int r0, nr;
                kv8_rows(p, s0 + lane, r0, nr);
                const int p0 = p.ctx[s0 + lane], pl = min(p0, INT_MAX - nr) + nr - 1;
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
                c = __builtin_amdgcn_readlane(cc, l); lo = __builtin_amdgcn_readlane(lo_s, l); hi = __builtin_amdgcn_readlane(hi_s, l);
                return true;
            }
            rest -= __builtin_amdgcn_readlane(incl, 63);
        }
    return false;
}

template <int HD, int NT>
struct Kv8DecCfg {
    static constexpr int NW = 4;                       // waves
    static constexpr int RR = 16 * NT;                 // query rows
    static constexpr int DC = HD / 64;                 // 64-dim pieces of a key (one 16-byte load per lane each)
    static constexpr int DB = HD / 16;                 // 16-dim output blocks
    static constexpr int QSTR = HD + 8;                // Q row in LDS: 16 rows on distinct bank quads
    static constexpr int BSTR = HD + 4;
    static constexpr size_t LDS_Q = (size_t)RR * QSTR * 2;
    static constexpr size_t LDS_M = ((size_t)2 * NW * RR + (size_t)RR * BSTR) * 4;
    static constexpr size_t LDS = LDS_Q > LDS_M ? LDS_Q : LDS_M;       // the merge reuses Q's place
    // Two waves per SIMD where K, V and the accumulators of a wave fit 256 registers.
    static constexpr int OCC = HD / 16 * 4 * NT + HD / 2 + 16 * NT <= 208 ? 2 : 1;
};

constexpr float kv8_head = 6.f, kv8_move = 14.f;       // the reference lies 2^6 under its maximum and moves above 2^14

template <int HD, int NT, bool F16, int OT>
__global__ void __launch_bounds__(256, (Kv8DecCfg<HD, NT>::OCC)) kv8_decode_kernel(const Kv8DecArgs a) {
    using Cf = Kv8DecCfg<HD, NT>;
    constexpr int NW = Cf::NW, DC = Cf::DC, DB = Cf::DB;
    extern __shared__ __align__(16) unsigned char smem[];
    const Kv8Problem &p = a.p;
    const Kv8 &kc = p.c;
    // Workgroups of one (chunk, KV head) and different row groups read the same keys: 8 apart, on one XCD.
    const int unit = (int)(blockIdx.x / (8 * a.nrg)) * 8 + (int)(blockIdx.x & 7), rg = (int)(blockIdx.x >> 3) % a.nrg;
    int seq, c, lo, hi;
    if (!kv8_find(p, a.C, a.Cm, a.direct, unit / kc.NKV, seq, c, lo, hi)) return;
    seq = __builtin_amdgcn_readfirstlane(seq); c = __builtin_amdgcn_readfirstlane(c);
    lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi);
    const int h = unit % kc.NKV, G = p.NQ / kc.NKV;
    int row0, nr;
    kv8_rows(p, seq, row0, nr);
    const int rho0 = rg * Cf::RR, nrows = min(nr * G - rho0, Cf::RR);
    const int j_lo = max(c * a.C, lo), j_hi = min(hi - c * a.C, a.C) + c * a.C;
    if (nrows <= 0 || (j_lo >= j_hi && !a.direct)) return;

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, ln = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int p0 = p.ctx[seq], page = kc.page;
    const int *tab = p.table + (size_t)seq * p.table_stride;
    const int last_col = p.max_pos >> kc.lp;

    // The pages of a step: of the lane's K rows (16-key piece ln / 4), and of its scores and V columns (piece g).
    struct Pages { int k, v; };
    auto pages_of = [&](int s) {
        Pages q;
        q.k = tab[min((64 * s + 16 * (ln >> 2)) >> kc.lp, last_col)];
        q.v = tab[min((64 * s + 16 * g) >> kc.lp, last_col)];
        return q;
    };
    u32x4 kr[4][DC], vr[DB];
    float ksc, vsc;
    bool vok;
    auto safe = [&](int id) { return (unsigned)id < (unsigned)kc.pages ? id : 0; };
    auto load_k = [&](int s, const Pages &q) {
        const int key = 64 * s + 16 * (ln >> 2) + (ln & 3);
        const uint8_t *b = kc.K + (((size_t)safe(q.k) * kc.NKV + h) * page + (key & (page - 1))) * HD + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int d = 0; d < DC; d++) kr[t][d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(b + 4 * t * HD + 64 * d));
    };
    auto load_v = [&](int s, const Pages &q) {
        const size_t cell = (size_t)safe(q.v) * kc.NKV + h;
        const uint8_t *b = kc.V + (cell * HD + ln) * page + ((64 * s + 16 * g) & (page - 1));
        ksc = kc.Ks[cell]; vsc = kc.Vs[cell];
        vok = (unsigned)q.v < (unsigned)kc.pages;
#pragma unroll
        for (int d = 0; d < DB; d++) vr[d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(b + (size_t)16 * d * page));
    };

    // Wave w takes the steps w, w + NW, .. of the chunk's.
    const int sc = c * (a.C / 64), s1 = j_hi > j_lo ? (j_hi - 1) / 64 : -1;
    int s = j_lo / 64;
    s += (wave - (s - sc)) & (NW - 1);
    Pages pg{0, 0}, pn{0, 0};
    if (s <= s1) {
        pg = pages_of(s);
        pn = pages_of(min(s + NW, s1));
    }
    // Q rows, zeros past the last.
    uint16_t *qs = reinterpret_cast<uint16_t *>(smem);
    {
        constexpr int N = Cf::RR * (HD / 8) / (NW * 64);
        u32x4 v[N];
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int i = tid + NW * 64 * u, R = i / (HD / 8), rho = rho0 + R;
            v[u] = u32x4{0u, 0u, 0u, 0u};
            if (R < nrows)
                v[u] = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(p.Q) +
                                                        ((size_t)(row0 + rho / G) * p.NQ + h * G + rho % G) * HD + (i % (HD / 8)) * 8);
        }
        if (s <= s1) { load_k(s, pg); load_v(s, pg); }
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int i = tid + NW * 64 * u;
            *reinterpret_cast<u32x4 *>(qs + (i / (HD / 8)) * Cf::QSTR + (i % (HD / 8)) * 8) = v[u];
        }
    }
    RowMask rm[NT];
    int lo_max = 0, pos_min = INT_MAX;
    {
        const int t0 = rho0 / G, t1 = (rho0 + nrows - 1) / G;
        lo_max = win_lo(p0 + t1, p.window);
        pos_min = p.anc ? p0 - 1 : p0 + t0;                            // tree keys: per row
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int rho = rho0 + 16 * nt + ln;
            rm[nt].valid = 16 * nt + ln < nrows;
            const int t = rm[nt].valid ? rho / G : 0;
            rm[nt].pos = p0 + t; rm[nt].lo = win_lo(p0 + t, p.window); rm[nt].tb = p0; rm[nt].tree = p.anc != nullptr;
            rm[nt].anc = p.anc ? p.anc[row0 + t] : 0u;
        }
    }
    __syncthreads();

    float m[NT], l[NT];
    f32x4 acc[NT][DB];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = kNegInf; l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++) acc[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (; s <= s1; s += NW) {
        const int j0 = 64 * s;
        const bool more = s + NW <= s1;
        f32x4 st[4][NT];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) st[t][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DC; d++) {
            u32x4 q[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) q[nt][e] = *reinterpret_cast<const u32x4 *>(qs + (16 * nt + ln) * Cf::QSTR + 64 * d + 16 * g + 8 * e);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const u32x4 k0 = e4m3_op<F16>(kr[t][d][0], kr[t][d][1]), k1 = e4m3_op<F16>(kr[t][d][2], kr[t][d][3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) st[t][nt] = mfma16<F16>(k0, q[nt][0], st[t][nt]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) st[t][nt] = mfma16<F16>(k1, q[nt][1], st[t][nt]);
            }
        }
        const float kf = ksc * a.sl2, ev = (float)exp_of(vsc), iv = pow2i(-exp_of(vsc));
        const bool ok = vok;
        if (more) load_k(s + NW, pn);
        const bool part = j0 < j_lo || j0 + 64 > j_hi || __any(!ok);   // keys of the step outside the chunk's, or without a page
        const bool full = !part && j0 >= lo_max && j0 + 63 <= pos_min;
        u32x2 pf[NT][4];                                               // P of tile t: the lane's keys 16 g + 4 t ..
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float tv[16];
#pragma unroll
            for (int i = 0; i < 16; i++) tv[i] = __builtin_fmaf(st[i >> 2][nt][i & 3], kf, ev);
            if (!full) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = j0 + 16 * g + i;
                    if (!(ok & (key >= j_lo) & (key < j_hi) & rm[nt].attends(key))) tv[i] = kNegInf;
                }
            }
            float mx = tv[0];
#pragma unroll
            for (int i = 1; i < 16; i++) mx = fmaxf(mx, tv[i]);
            mx = max_over_groups(mx);
            const float mn = mx > m[nt] + kv8_move ? mx - kv8_head : m[nt];
            if (__any(mn != m[nt])) {
                const float al = mn == m[nt] ? 1.f : fast_exp2(m[nt] - mn);
                l[nt] *= al; m[nt] = mn;
#pragma unroll
                for (int d = 0; d < DB; d++) acc[nt][d] *= al;
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (full) tv[i] = fast_exp2(tv[i] - m[nt]);
                else tv[i] = tv[i] == kNegInf ? 0.f : fast_exp2(tv[i] - m[nt]);        // (a row without a key yet: m = -inf)
                sum += tv[i];
            }
            l[nt] = __builtin_fmaf(sum, iv, l[nt]);
#pragma unroll
            for (int t = 0; t < 4; t++) pf[nt][t] = u32x2{pack2<true>(tv[4 * t], tv[4 * t + 1]), pack2<true>(tv[4 * t + 2], tv[4 * t + 3])};
        }
        if (part) {                                                    // bytes that are no token of the request's: any code, NaN too
            const int k0 = ok ? max(j_lo - j0 - 16 * g, 0) : 16, k1 = min(j_hi - j0 - 16 * g, 16);
            u32x4 keep;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int x = min(max(k0 - 4 * w, 0), 4), y = min(max(k1 - 4 * w, 0), 4);      // bytes [x, y) of word w
                const uint32_t below = y >= 4 ? 0xffffffffu : (1u << (8 * y)) - 1u, under = x >= 4 ? 0xffffffffu : (1u << (8 * x)) - 1u;
                keep[w] = below & ~under;
            }
#pragma unroll
            for (int d = 0; d < DB; d++) vr[d] &= keep;
        }
        if (more) pg = pn;
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const u32x4 v0 = e4m3_op<true>(vr[d][0], vr[d][1]), v1 = e4m3_op<true>(vr[d][2], vr[d][3]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
                acc[nt][d] = mfma16<true>(v0, u32x4{pf[nt][0][0], pf[nt][0][1], pf[nt][1][0], pf[nt][1][1]}, acc[nt][d]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
                acc[nt][d] = mfma16<true>(v1, u32x4{pf[nt][2][0], pf[nt][2][1], pf[nt][3][0], pf[nt][3][1]}, acc[nt][d]);
        }
        if (more) {
            load_v(s + NW, pg);
            pn = pages_of(min(s + 2 * NW, s1));
        }
    }

    // Merge the waves' states in their order.
    float *redm = reinterpret_cast<float *>(smem), *redl = redm + NW * Cf::RR, *buf = redl + NW * Cf::RR;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) l[nt] = sum_over_groups(l[nt]);
    __syncthreads();
    if (g == 0)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) { redm[wave * Cf::RR + 16 * nt + ln] = m[nt]; redl[wave * Cf::RR + 16 * nt + ln] = l[nt]; }
    __syncthreads();
    for (int w = 0; w < NW; w++) {
        if (wave == w)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (16 * nt + ln >= nrows) continue;
                float M = kNegInf;
#pragma unroll
                for (int x = 0; x < NW; x++) M = fmaxf(M, redm[x * Cf::RR + 16 * nt + ln]);
                const float f = kv8_weight(m[nt], l[nt], M);
#pragma unroll
                for (int d = 0; d < DB; d++) {
                    f32x4 *dst = reinterpret_cast<f32x4 *>(buf + (16 * nt + ln) * Cf::BSTR + 16 * d + 4 * g);
                    f32x4 v = acc[nt][d] * f;
                    if (w > 0) v += *dst;
                    *dst = v;
                }
            }
        __syncthreads();
    }
    auto state_of = [&](int R, float &M, float &L) {
        M = kNegInf; L = 0.f;
        for (int x = 0; x < NW; x++) M = fmaxf(M, redm[x * Cf::RR + R]);
        for (int x = 0; x < NW; x++) {
            const float mx = redm[x * Cf::RR + R], lx = redl[x * Cf::RR + R];
            L += mx == kNegInf ? lx * 0.f : lx * fast_exp2(mx - M);
        }
    };
    for (int i = tid; i < nrows * (HD / 4); i += NW * 64) {
        const int R = i / (HD / 4), d4 = i % (HD / 4), rho = rho0 + R;
        const size_t row = (size_t)(row0 + rho / G) * p.NQ + h * G + rho % G;
        f32x4 v = *reinterpret_cast<const f32x4 *>(buf + R * Cf::BSTR + 4 * d4);
        float M, L;
        state_of(R, M, L);
        if (a.direct) {
            v *= L == 0.f ? 0.f : 1.f / L;
            if constexpr (OT == DT_FP32) *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(p.O) + row * HD + 4 * d4) = v;
            else *reinterpret_cast<u32x2 *>(reinterpret_cast<uint16_t *>(p.O) + row * HD + 4 * d4) =
                u32x2{pack2<OT == DT_F16>(v[0], v[1]), pack2<OT == DT_F16>(v[2], v[3])};
            if (d4 == 0 && p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
        } else {
            const size_t x = row * a.part.ns + c;
            *reinterpret_cast<f32x4 *>(a.part.acc + x * HD + 4 * d4) = v;
            if (d4 == 0) { a.part.m[x] = M; a.part.l[x] = L; }
        }
    }
}

// ---------------------------------------------------------------- merge of key splits
// One workgroup per (row, q-head): HD / 4 threads hold 4 dims each and 256 / (HD / 4) phases take the splits in turn; the
// phases are added in their order. Also writes the rows that attend nothing (O = 0, lse = -inf).
struct Kv8CombArgs {
    Kv8Problem p;
    Kv8Partials part;
    uint32_t Cm;
};

template <int HD, int OT>
__global__ void __launch_bounds__(256) kv8_combine_kernel(const Kv8CombArgs a) {
    constexpr int TPR = HD / 4, PH = 256 / TPR;
    __shared__ __align__(16) float red[PH][HD];
    const Kv8Problem &p = a.p;
    const int b = (int)blockIdx.x / p.T, i = (int)blockIdx.x - b * p.T, head = blockIdx.y;
    int row0, nr;
    kv8_rows(p, b, row0, nr);
    if (i >= nr) return;
    const int pos = min(p.ctx[b], INT_MAX - i) + i, lo = win_lo(pos, p.window), hi = min(pos, p.max_pos);
    const size_t row = (size_t)(row0 + i) * p.NQ + head;
    const int c0 = div_by(lo, a.part.C, a.Cm), c1 = hi >= lo ? div_by(hi, a.part.C, a.Cm) : c0 - 1;
    const int tid = threadIdx.x, d4 = tid % TPR, ph = tid / TPR;
    const float *pm = a.part.m + row * a.part.ns, *pl = a.part.l + row * a.part.ns;
    const float *pa = a.part.acc + row * a.part.ns * HD + 4 * d4;
    float M = kNegInf;
    for (int c = c0; c <= c1; c++) M = fmaxf(M, pm[c]);
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    for (int c = c0; c <= c1; c++) L += pl[c] * kv8_weight(pm[c], pl[c], M);
    for (int c = c0 + ph; c <= c1; c += PH) v += *reinterpret_cast<const f32x4 *>(pa + (size_t)c * HD) * kv8_weight(pm[c], pl[c], M);
    if constexpr (PH > 1) {
        *reinterpret_cast<f32x4 *>(&red[ph][4 * d4]) = v;
        __syncthreads();
        if (ph) return;
#pragma unroll
        for (int x = 1; x < PH; x++) v += *reinterpret_cast<const f32x4 *>(&red[x][4 * d4]);
    }
    v *= L == 0.f ? 0.f : 1.f / L;
    if constexpr (OT == DT_FP32) *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(p.O) + row * HD + 4 * d4) = v;
    else *reinterpret_cast<u32x2 *>(reinterpret_cast<uint16_t *>(p.O) + row * HD + 4 * d4) =
        u32x2{pack2<OT == DT_F16>(v[0], v[1]), pack2<OT == DT_F16>(v[2], v[3])};
    if (d4 == 0 && p.lse) p.lse[row] = L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * kLn2;
}

template <int HD> static hipError_t combine_t(const Kv8CombArgs &a, dim3 grid, hipStream_t st) {
    switch (a.p.o_dtype) {
    case DT_FP32: hipLaunchKernelGGL((kv8_combine_kernel<HD, DT_FP32>), grid, dim3(256), 0, st, a); break;
    case DT_F16: hipLaunchKernelGGL((kv8_combine_kernel<HD, DT_F16>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((kv8_combine_kernel<HD, DT_BF16>), grid, dim3(256), 0, st, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv8_combine(const Kv8Problem &p, const Kv8Partials &part, hipStream_t st) {
    const Kv8CombArgs a{p, part, div_magic(part.C)};
    const dim3 grid((unsigned)p.B * (unsigned)p.T, (unsigned)p.NQ);
    switch (p.c.HD) {
    case 128: return combine_t<128>(a, grid, st);
    case 256: return combine_t<256>(a, grid, st);
    case 512: return combine_t<512>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

// ---------------------------------------------------------------- launch
template <int HD, int NT, bool F16, int OT>
static hipError_t launch_dec_k(const Kv8DecArgs &a, dim3 grid, hipStream_t st) {
    using Cf = Kv8DecCfg<HD, NT>;
    static_assert(Cf::LDS <= 160 * 1024, "LDS");
    if constexpr (Cf::LDS > 64 * 1024) {                               // per device; setting it again changes nothing
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv8_decode_kernel<HD, NT, F16, OT>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)Cf::LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((kv8_decode_kernel<HD, NT, F16, OT>), grid, dim3(Cf::NW * 64), Cf::LDS, st, a);
    return hipGetLastError();
}
template <int HD, int NT, bool F16> static hipError_t launch_dec_o(const Kv8DecArgs &a, dim3 grid, hipStream_t st) {
    switch (a.p.o_dtype) {
    case DT_FP32: return launch_dec_k<HD, NT, F16, DT_FP32>(a, grid, st);
    case DT_F16: return launch_dec_k<HD, NT, F16, DT_F16>(a, grid, st);
    default: return launch_dec_k<HD, NT, F16, DT_BF16>(a, grid, st);
    }
}
template <int HD, int NT> static hipError_t launch_dec_n(const Kv8DecArgs &a, dim3 grid, hipStream_t st) {
    return a.p.q_dtype == DT_F16 ? launch_dec_o<HD, NT, true>(a, grid, st) : launch_dec_o<HD, NT, false>(a, grid, st);
}

Kv8Plan kv8_choose(int B, int T, int rows, int NQ, int NKV, int HD, int max_pos, int chunk, int window, bool tree) {
    (void)rows;
    const long long hr = (long long)T * (NQ / NKV);                    // rows of a KV head and request
    Kv8Plan pl{!tree && hr > 64, chunk, 1};
    long long keys = max_pos + 1ll;
    if (window > 0) keys = std::min<long long>(keys, (long long)window + T - 1);
    if (pl.prefill) {
        if (chunk == 0) return pl;
    } else if (chunk == 0) {
        const long long units = (long long)B * NKV, want = std::max(1ll, 512 / units);
        pl.C = (int)std::min<long long>(std::max<long long>((keys / want + 255) / 256 * 256, 256), 1024);
    }
    pl.ns = max_pos / pl.C + 1;
    if (pl.prefill && pl.ns == 1) pl.C = 0;
    return pl;
}

hipError_t launch_kv8_decode(const Kv8Problem &p, const Kv8Partials &part, hipStream_t st) {
    const int G = p.NQ / p.c.NKV, rows = (int)std::min<long long>((long long)p.T * G, INT_MAX);
    const int nt = p.c.HD == 512 || rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    Kv8DecArgs a{p, part, part.C, div_magic(part.C), (rows + 16 * nt - 1) / (16 * nt), part.ns == 1, p.scale * kLog2e};
    long long per = p.max_pos / part.C + 1;
    if (p.window > 0) per = std::min<long long>(per, ((long long)p.window + p.T - 2) / part.C + 2);
    const long long units = (per * p.B * p.c.NKV + 7) / 8 * 8, wgs = units * a.nrg;
    if (wgs > INT_MAX) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs);
    switch (p.c.HD) {
    case 128: return nt == 1 ? launch_dec_n<128, 1>(a, grid, st) : nt == 2 ? launch_dec_n<128, 2>(a, grid, st) : launch_dec_n<128, 4>(a, grid, st);
    case 256: return nt == 1 ? launch_dec_n<256, 1>(a, grid, st) : nt == 2 ? launch_dec_n<256, 2>(a, grid, st) : launch_dec_n<256, 4>(a, grid, st);
    case 512: return launch_dec_n<512, 1>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dgx
