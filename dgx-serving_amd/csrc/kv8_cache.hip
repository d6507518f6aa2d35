// Writing the paged 8-bit KV cache on gfx950: the block tables and slot maps of a step, and the quantising append.
#include "attn_kv8.h"
#include <algorithm>

namespace dgx {

// ---------------------------------------------------------------- block tables and slot maps
// Requests b = 0 .. B-1 hold ctx[b] tokens and get add[b] more: with have = ceil(ctx / page) and want = ceil((ctx + add) /
// page) request b takes want - have pages from the top of the free stack, in the order of the requests; row cu[b] + i (its
// i-th new token, at position ctx[b] + i) gets slot page_id * page + position % page. New pages begin exactly at the rows
// whose position is a multiple of the page, so that row writes the table's entry too and nothing else walks the pages.
//
// All or nothing: a step that needs more free pages, columns or rows than there are, or has a negative length, takes nothing
// (status tells which), gives every row slot -1 and every request no rows.
//
// Bound by latency: lengths, scan, free ids, slots (256 requests of one token 3.1 us, 96 prompts of 109K rows in all 5.9). The
// scans take one workgroup's time whatever the grid, so every workgroup does them (lengths come from the L2) and takes its
// share of the rows, from 2048 each on: the 96 prompts take 97 us a call in one workgroup and 8 in 54. A second launch behind a
// one-workgroup scan would cost more than the scan. One workgroup alone does it all where the free count is updated in place
// (another workgroup could read it late).
struct PlanArgs {
    const int *ctx, *add, *free_pages, *free_in;
    int *table, *free_out, *cu, *slots, *status;
    long table_stride;
    int B, lp, cols, rows, free_cap;
};

constexpr int kPlanThreads = 1024;

// Lengths are clamped to what a step can hold (and the step is refused): with at most kNarrow rows and columns the sums of
// 1024 requests fit 32 bits, whose scans are a fifth of the work.
constexpr int kNarrow = 1 << 20;
__device__ __forceinline__ int scan_wave(int v) { return wave_scan64(v); }
__device__ __forceinline__ long long scan_wave(long long v) {     // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

template <class T>
__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const PlanArgs a) {
    __shared__ T w_pages[kPlanThreads / 64], w_rows[kPlanThreads / 64];
    __shared__ int s_row[kPlanThreads + 1], s_page[kPlanThreads], s_ctx[kPlanThreads], bad_s;
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6, page = 1 << a.lp;
    const int count = a.free_in[0];
    int flags = count < 0 || count > a.free_cap ? 8 : 0;
    // Lengths of request b: pages and rows that it takes.
    auto lengths = [&](int b, int &ctx, T &pages, T &rows) {
        ctx = 0; pages = rows = 0;
        if (b >= a.B) return;
        const int c = a.ctx[b], n = a.add[b];
        const long long have = ((long long)c + page - 1) >> a.lp, want = ((long long)c + n + page - 1) >> a.lp;
        const int f = (c < 0 || n < 0 ? 8 : 0) | (want > a.cols ? 2 : 0) | (n > a.rows ? 4 : 0);
        flags |= f;
        if (f) return;
        ctx = c; pages = (T)(want - have); rows = n;
    };
    // Workgroup-wide inclusive scans of pages and rows, and the totals.
    auto scan = [&](T &pages, T &rows, T &all_pages, T &all_rows) {
        pages = scan_wave(pages); rows = scan_wave(rows);
        if (lane == 63) { w_pages[wave] = pages; w_rows[wave] = rows; }
        __syncthreads();
        all_pages = all_rows = 0;
        T before_p = 0, before_r = 0;
        for (int w = 0; w < nt / 64; w++) {
            if (w == wave) { before_p = all_pages; before_r = all_rows; }
            all_pages += w_pages[w]; all_rows += w_rows[w];
        }
        pages += before_p; rows += before_r;
    };
    if (tid == 0) bad_s = 0;
    int ctx;
    T pages, rows, ap, ar;
    lengths(tid, ctx, pages, rows);
    T mine = pages;
    scan(pages, rows, ap, ar);                                     // (its barrier is behind bad_s = 0 too)
    long long need_pages = ap, need_rows = ar;
    for (int t0 = nt; t0 < a.B; t0 += nt) {                        // totals over the requests behind the first tile
        int c;
        T x, y, xp, yr;
        lengths(t0 + tid, c, x, y);
        __syncthreads();
        scan(x, y, xp, yr);
        need_pages += xp; need_rows += yr;
    }
    if (need_pages > max(count, 0)) flags |= 1;
    if (need_rows > a.rows) flags |= 4;
    if (flags) atomicOr(&bad_s, flags);
    __syncthreads();
    const int bad = bad_s;
    const long long r_per = ((long long)a.rows + gridDim.x - 1) / gridDim.x;
    const long long r_lo = r_per * blockIdx.x, r_hi = min((long long)a.rows, r_lo + r_per);
    if (blockIdx.x == 0) {
        if (tid == 0) {
            a.status[0] = bad;
            a.free_out[0] = bad ? count : count - (int)need_pages;
            a.cu[0] = 0;
        }
        if (bad)
            for (int b = tid; b < a.B; b += nt) a.cu[b + 1] = 0;
    }
    for (long long r = max(r_lo, bad ? 0ll : need_rows) + tid; r < r_hi; r += nt) a.slots[r] = -1;
    if (bad) return;
    long long base_pages = 0, base_rows = 0;
    for (int t0 = 0;;) {                                           // a tile of requests at a time; the first one's scan is done
        s_row[tid + 1] = (int)(base_rows + rows);                  // (at most a.rows: checked above)
        if (tid == 0) s_row[0] = (int)base_rows;
        s_page[tid] = (int)(base_pages + pages - mine);
        s_ctx[tid] = ctx;
        if (blockIdx.x == 0 && t0 + tid < a.B) a.cu[t0 + tid + 1] = (int)(base_rows + rows);
        __syncthreads();
        const int nb = min(nt, a.B - t0);
        const long long lo = max(r_lo, base_rows), hi = min(r_hi, base_rows + ar);
        for (long long r = lo + tid; r < hi; r += nt) {
            int x = 0, y = nb;                                     // the request: s_row[x] <= r < s_row[x + 1]
            while (y - x > 1) {
                const int mid = (x + y) >> 1;
                if (s_row[mid] <= (int)r) x = mid; else y = mid;
            }
            const int c0 = s_ctx[x];
            const long long pos = (long long)c0 + ((int)r - s_row[x]);
            const int col = (int)(pos >> a.lp), off = (int)(pos & (page - 1)), have = (int)(((long long)c0 + page - 1) >> a.lp);
            int *cell = a.table + (size_t)(t0 + x) * a.table_stride + col;
            const int id = col < have ? *cell : a.free_pages[count - 1 - (s_page[x] + col - have)];
            if (off == 0) *cell = id;
            a.slots[r] = id >= 0 && id <= (0x7fffffff >> a.lp) - 1 ? (id << a.lp) + off : -1;
        }
        base_pages += ap; base_rows += ar;
        t0 += nt;
        if (t0 >= a.B) break;
        __syncthreads();
        lengths(t0 + tid, ctx, pages, rows);
        mine = pages;
        scan(pages, rows, ap, ar);
    }
}

hipError_t launch_kv8_plan(const int *ctx, const int *add, int B, int lp, int *table, long table_stride, int cols,
                           const int *free_pages, int free_cap, const int *free_in, int *free_out, int *cu, int *slots, int rows,
                           int *status, hipStream_t st) {
    const PlanArgs a{ctx, add, free_pages, free_in, table, free_out, cu, slots, status, table_stride, B, lp, cols, rows, free_cap};
    const int grid = free_in == free_out || rows <= 2048 ? 1 : (int)std::min(128ll, (rows + 2047ll) / 2048);
    // Fewer waves meet sooner at the barriers: 16 requests of a token 2.9 us in 256 threads, 3.5 in 1024 (one after another in a
    // graph), 256 of a token 3.3 and 4.0; 256 of four tokens take several rounds of rows, 6.0 and 4.2.
    const int threads = B <= 256 && rows <= 1024 ? 256 : kPlanThreads;
    if (rows <= kNarrow && cols <= kNarrow) hipLaunchKernelGGL(kv8_plan_kernel<int>, dim3(grid), dim3(threads), 0, st, a);
    else hipLaunchKernelGGL(kv8_plan_kernel<long long>, dim3(grid), dim3(threads), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- quantising append
// Row r of k_src / v_src goes to token slots[r] % page of page slots[r] / page; rows with a slot outside the pool are
// skipped. Rows that follow each other into one page are a run, and one workgroup takes a run of one KV head, K and V:
//   1. it holds the run's values in registers (4 tokens x 8 dims per thread, page * HD / 32 threads), takes the largest
//      finite magnitude of each tensor and notes the tokens that hold a value that is not finite;
//   2. e = max(exponent of that magnitude, the page's own exponent if the run starts behind token 0);
//   3. if the page's exponent grew, the codes before the run are rounded again to the new one;
//   4. the new codes: K rows as they come, V through LDS into rows of the head dim (4x4 byte transposes in registers, then
//      whole 16-byte pieces of 16 tokens; single bytes where the run covers a piece in part).
// A token with a value that is not finite gets K codes NaN and 0 in place of V's values that are not finite: a score with it
// is NaN, so every row that attends it comes out NaN, and rows that do not are left alone (a NaN code in V would reach the
// other rows of a matrix tile through 0 * NaN).
// Bound by memory: 66K rows x 8 heads x 256 from bf16 read 2 bytes and write 1 per element, 173 us, 4.73 TB/s (a large copy
// reaches 4.82). Small calls by latency: 16 rows of a token each 5.2 us, a prompt of 1024 from fp32 8.8 (128 workgroups, one of
// each run and head, on half of the CUs: its chain of load, maximum, transpose and store).
struct AppendArgs {
    const void *k, *v;
    long ks, vs;                      // row strides in elements
    Kv8 c;
    const int *slots;
    unsigned *stats;                  // {non-finite K, V, max |K|, max |V|} or null
    int rows, win, lv, windows;       // win: rows of a workgroup's window; lv = log2(HD / 8)
};

// 8 values of a source row.
template <int ST> struct Src8 {
    u32x4 w[ST == DT_FP32 ? 2 : 1];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (ST == DT_FP32) return __uint_as_float(w[i >> 2][i & 3]);
        else {
            const uint16_t h = (uint16_t)(w[0][i >> 1] >> (16 * (i & 1)));
            if constexpr (ST == DT_F16) return f16_bits_to_f32(h);
            else return bf16_bits_to_f32(h);
        }
    }
    __device__ __forceinline__ void put(int i, float x) {              // x: a value of the type
        if constexpr (ST == DT_FP32) w[i >> 2][i & 3] = __float_as_uint(x);
        else {
            const uint32_t h = f32_to_op(x, ST == DT_F16);
            w[0][i >> 1] = (i & 1) ? (w[0][i >> 1] & 0xffffu) | (h << 16) : (w[0][i >> 1] & 0xffff0000u) | h;
        }
    }
};

// Four codes times f, rounded again; NaN codes stay as they are.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, r, true);
    const uint32_t nan = ((((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u) * 255u;
    return ((uint32_t)r & ~nan) | (w & nan);
}

template <int ST, int MOST>
__global__ void __launch_bounds__(MOST) kv8_append_kernel(const AppendArgs a) {
    using SE = typename Elem<ST>::T;
    extern __shared__ __align__(16) unsigned char tile[];          // V codes of the run, [HD][page], swizzled
    __shared__ float red[2][16];
    __shared__ int bad_s[64], nonfin[2], rows_s[64];
    const Kv8 &c = a.c;
    const int page = c.page, HD = c.HD, PQ = page / 4;
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, nw = (nt + 63) >> 6;
    // Workgroups go round-robin over the 8 XCDs and runs begin at regular distances: each XCD takes an eighth of the windows.
    const unsigned unit = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int h = (int)(unit % (unsigned)c.NKV);
    if (unit / (unsigned)c.NKV >= (unsigned)a.windows) return;
    const int w0 = (int)(unit / (unsigned)c.NKV) * a.win;
    const int total = c.pages << c.lp;                             // host: at most INT_MAX
    auto slot_of = [&](int r) { return (unsigned)r < (unsigned)a.rows ? a.slots[r] : -1; };
    // A row begins a run unless the last row before it that is not skipped holds the token before its own, in the same page.
    unsigned long long starts;
    {
        const int r = w0 + lane, s = lane < a.win ? slot_of(r) : -1, prev = lane < a.win ? slot_of(r - 1) : -1;
        const bool ok = (unsigned)s < (unsigned)total, inner = (s & (page - 1)) != 0;
        starts = __ballot(ok && !(prev == s - 1 && inner));
        if (__ballot(ok && inner && r > 0 && (unsigned)prev >= (unsigned)total)) {   // rare: skipped rows to look behind
            const int s2 = slot_of(w0 - (64 - a.win) + lane);          // the window's rows are the last lanes'
            const bool ok2 = (unsigned)s2 < (unsigned)total;
            const unsigned long long below = __ballot(ok2) & ((1ull << lane) - 1);
            const int last = __shfl(s2, below ? 63 - __builtin_clzll(below) : lane);
            starts = __ballot(ok2 && lane >= 64 - a.win && !(below && last == s2 - 1 && (s2 & (page - 1)) != 0)) >> (64 - a.win);
        }
    }
    const int dv = tid & ((1 << a.lv) - 1), tg = tid >> a.lv;      // 8 dims from 8 dv, tokens 4 tg .. 4 tg + 3 of the run
    for (; starts; starts &= starts - 1) {
        const int r0 = w0 + __builtin_ctzll(starts), s0 = __builtin_amdgcn_readfirstlane(a.slots[r0]);
        const int off = s0 & (page - 1), pid = s0 >> c.lp;
        // Its n tokens: the rows from r0 on with the slots s0, s0 + 1, .. within the page; skipped rows may lie between them.
        int n;
        bool dense = true;                                             // none do
        {
            const int sa = slot_of(r0 + lane);
            const unsigned long long next = ~__ballot(sa == s0 + lane && off + lane < page);
            n = next ? __builtin_ctzll(next) : 64;
            if (off + n < page && (n == 64 || (__ballot((unsigned)sa >= (unsigned)total) >> n & 1)) && r0 + n < a.rows) {   // rare: a skipped row is next
                const unsigned long long under = (1ull << lane) - 1;
                int k = 0;
                for (int part = 0; part < 2; part++) {
                    const int sx = part ? slot_of(r0 + 64 + lane) : sa, kx = k + __popcll(__ballot((unsigned)sx < (unsigned)total) & under);
                    const bool taken = (unsigned)sx < (unsigned)total, in = sx == s0 + kx && off + kx < page;
                    const unsigned long long stop = __ballot(taken && !in), mine = __ballot(taken && in) & (stop ? (stop & -stop) - 1 : ~0ull);
                    if (mine >> lane & 1) rows_s[kx] = 64 * part + lane;
                    k += __popcll(mine);
                    if (stop) break;
                }
                dense = k == n;
                n = k;
            }
        }
        for (int i = tid; i < 64; i += nt) bad_s[i] = 0;
        if (tid < 2) nonfin[tid] = 0;
        // (Tokens behind the run repeat its last one: its magnitudes change nothing, and no load waits for a branch.)
        Src8<ST> x[2][4];
        const bool live = 4 * tg < n;
        if (live) {
            int row[4];
#pragma unroll
            for (int i = 0; i < 4; i++) row[i] = min(4 * tg + i, n - 1);
            if (!dense) {                                              // (all waves write the same rows_s and each reads what it wrote)
#pragma unroll
                for (int i = 0; i < 4; i++) row[i] = rows_s[row[i]];
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const SE *p = reinterpret_cast<const SE *>(t ? a.v : a.k) + (size_t)(r0 + row[i]) * (size_t)(t ? a.vs : a.ks) + h * HD + 8 * dv;
#pragma unroll
                    for (int q = 0; q < (ST == DT_FP32 ? 2 : 1); q++) x[t][i].w[q] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p) + q);
                }
        }
        const size_t cell = (size_t)pid * c.NKV + h;
        const float oldk = c.Ks[cell], oldv = c.Vs[cell];
        __syncthreads();
        constexpr uint32_t kInf = 0x7f800000u;
        uint32_t top[2] = {0u, 0u};                                     // bits of the largest magnitude (they order as the values)
        if (live) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) top[t] = max(top[t], __float_as_uint(x[t][i].get(e)) & 0x7fffffffu);
                if (top[t] >= kInf) {                                   // rare: something here is not finite
                    top[t] = 0u;
                    int nf = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t m = __float_as_uint(x[t][i].get(e)) & 0x7fffffffu;
                            if (m < kInf) top[t] = max(top[t], m);
                            else {
                                bad_s[4 * tg + i] = 1;
                                nf += 4 * tg + i < n ? 1 : 0;
                                x[t][i].put(e, 0.f);
                            }
                        }
                    if (nf && a.stats) atomicAdd(&nonfin[t], nf);
                }
            }
        }
        float amax[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            amax[t] = __uint_as_float(top[t]);
#pragma unroll
            for (int d = 32; d; d >>= 1) amax[t] = fmaxf(amax[t], __shfl_xor(amax[t], d));
            if (lane == 0) red[t][tid >> 6] = amax[t];
        }
        __syncthreads();
        int e_old[2], e[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float m = 0.f;
            for (int w = 0; w < nw; w++) m = fmaxf(m, red[t][w]);
            e_old[t] = off > 0 ? min(max(exp_of(t ? oldv : oldk), kv8_emin), kv8_emax) : kv8_emin;
            e[t] = max(kv8_exponent(m), e_old[t]);
            if (tid == 0) {
                (t ? c.Vs : c.Ks)[cell] = pow2i(e[t]);
                if (a.stats) {                                      // rounding is monotone: the largest stored value is the largest one's
                    const float s = fminf(m * pow2i(-e[t]), 448.f);
                    const float q = __builtin_amdgcn_cvt_pk_f32_fp8(__builtin_amdgcn_cvt_pk_fp8_f32(s, 0.f, 0, false), false)[0];
                    atomicMax(&a.stats[2 + t], __float_as_uint(q * pow2i(e[t])));
                    if (nonfin[t]) atomicAdd(&a.stats[t], (unsigned)nonfin[t]);
                }
            }
        }
        uint8_t *Kp = c.K + cell * ((size_t)page * HD), *Vp = c.V + cell * ((size_t)page * HD);
        // A grown exponent: the page's earlier tokens, 16 codes at a time. (V's pieces hold tokens from off on too, which
        // keep their bytes here; the waits put these stores before the bytes written below.)
        if (off > 0 && (e[0] > e_old[0] || e[1] > e_old[1])) {
            const float fk = pow2i(max(e_old[0] - e[0], -126)), fv = pow2i(max(e_old[1] - e[1], -126));
            if (e[0] > e_old[0])
                for (int i = tid; i < off * HD / 16; i += nt) {
                    u32x4 *q = reinterpret_cast<u32x4 *>(Kp) + i;
                    u32x4 w = *q;
#pragma unroll
                    for (int d = 0; d < 4; d++) w[d] = rescale4(w[d], fk);
                    *q = w;
                }
            if (e[1] > e_old[1])
                for (int i = tid; i < page * HD / 16; i += nt) {
                    const int t0 = (i & (page / 16 - 1)) * 16;
                    if (t0 >= off) continue;
                    u32x4 *q = reinterpret_cast<u32x4 *>(Vp) + i;
                    u32x4 w = *q;
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const int k = off - t0 - 4 * d;             // bytes of this word that are earlier tokens
                        const uint32_t m = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
                        w[d] = (rescale4(w[d], fv) & m) | (w[d] & ~m);
                    }
                    *q = w;
                }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const float ik = pow2i(-e[0]), iv = pow2i(-e[1]);
        if (ST != DT_F16 && live && (e[0] == kv8_emax || e[1] == kv8_emax)) {   // the largest scale may be too small: values past 448 of it
            const float top_v = 448.f * pow2i(kv8_emax);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int q = 0; q < 8; q++) x[t][i].put(q, __builtin_amdgcn_fmed3f(x[t][i].get(q), -top_v, top_v));
        }
        uint32_t *tw = reinterpret_cast<uint32_t *>(tile);
        if (live) {
            uint32_t vc[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int tok = 4 * tg + i;
                const bool nan = bad_s[tok] != 0;
                u32x2 kc;
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    kc[q] = to_e4m3x4(x[0][i].get(4 * q) * ik, x[0][i].get(4 * q + 1) * ik, x[0][i].get(4 * q + 2) * ik, x[0][i].get(4 * q + 3) * ik);
                    vc[i][q] = to_e4m3x4(x[1][i].get(4 * q) * iv, x[1][i].get(4 * q + 1) * iv, x[1][i].get(4 * q + 2) * iv, x[1][i].get(4 * q + 3) * iv);
                    if (nan) kc[q] = 0x7f7f7f7fu;
                }
                if (tok < n) *reinterpret_cast<u32x2 *>(Kp + (size_t)(off + tok) * HD + 8 * dv) = kc;
            }
            // [4 tokens][8 dims] -> [8 dims][4 tokens]. Word (dim d, tokens 4 tq ..) of the tile sits at d * PQ + (tq ^ (d / 8 %
            // PQ)): the lanes of a wave hold dims 8 apart, which would all share a bank.
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const uint32_t l01 = __builtin_amdgcn_perm(vc[1][q], vc[0][q], 0x05010400u), h01 = __builtin_amdgcn_perm(vc[1][q], vc[0][q], 0x07030602u);
                const uint32_t l23 = __builtin_amdgcn_perm(vc[3][q], vc[2][q], 0x05010400u), h23 = __builtin_amdgcn_perm(vc[3][q], vc[2][q], 0x07030602u);
                const uint32_t b[4] = {__builtin_amdgcn_perm(l23, l01, 0x05040100u), __builtin_amdgcn_perm(l23, l01, 0x07060302u),
                                       __builtin_amdgcn_perm(h23, h01, 0x05040100u), __builtin_amdgcn_perm(h23, h01, 0x07060302u)};
#pragma unroll
                for (int d = 0; d < 4; d++) tw[(8 * dv + 4 * q + d) * PQ + (tg ^ (dv & (PQ - 1)))] = b[d];
            }
        }
        __syncthreads();
        const int whole = off == 0 ? n >> 4 : 0;                    // 16-token pieces that the run covers
        if (whole)
            for (int i = tid; i < page * HD / 16; i += nt) {
                const int ch = i & (page / 16 - 1), d = i / (page / 16), g = (d >> 3) & (PQ - 1);
                if (ch >= whole) continue;
                u32x4 w = *reinterpret_cast<const u32x4 *>(tw + d * PQ + 4 * (ch ^ (g >> 2)));
                if (g & 1) w = u32x4{w[1], w[0], w[3], w[2]};
                if (g & 2) w = u32x4{w[2], w[3], w[0], w[1]};
                *reinterpret_cast<u32x4 *>(Vp + (size_t)i * 16) = w;
            }
        const int t1 = 16 * whole;
        for (int i = tid; i < (n - t1) * HD; i += nt) {
            const int d = i & (HD - 1), t = t1 + i / HD, g = (d >> 3) & (PQ - 1);
            Vp[(size_t)d * page + off + t] = tile[(d * PQ + ((t >> 2) ^ g)) * 4 + (t & 3)];
        }
        __syncthreads();                                            // the next run reuses the tile
    }
}

template <int ST>
static hipError_t launch_append_t(const AppendArgs &a, dim3 grid, int threads, hipStream_t st) {
    // (fp32 rows need 165 registers, more than 1024 threads have: 2000 rows x 8 heads of 256 20.7 us, 22.1 with spills)
    constexpr int few = ST == DT_FP32 ? 512 : 1024;
    if (threads <= few) hipLaunchKernelGGL((kv8_append_kernel<ST, few>), grid, dim3(threads), (size_t)a.c.page * a.c.HD, st, a);
    else hipLaunchKernelGGL((kv8_append_kernel<ST, 1024>), grid, dim3(threads), (size_t)a.c.page * a.c.HD, st, a);
    return hipGetLastError();
}

hipError_t launch_kv8_append(const void *k, const void *v, int src_dtype, long k_stride, long v_stride, const Kv8 &c,
                             const int *slots, int rows, unsigned *stats, hipStream_t st) {
    AppendArgs a{k, v, k_stride, v_stride, c, slots, stats, rows, 1, 0, 0};
    while ((8 << a.lv) < c.HD) a.lv++;
    // A workgroup looks for runs among `win` rows, and takes those that begin there one after another. Windows of 1 | 4 | 16
    // rows, us: 16 requests of a token x 4 heads (64 units) 5.2 | 13.3 | 46.1, 256 of a token x 4 (1024) 13.1 | 15.8 | 46.7, 512
    // of up to 4 x 8 (10K) 56.8 | 49.6 | 60.0, a prompt of 1024 x 8 (8K) from bf16 11.4 | 7.5 | 8.3, from fp32 16.7 | 8.7 | 7.4, 66K rows
    // of prompts x 8 (532K) 383 | 212 | 165: most workgroups of a prompt find none.
    const long long units = (long long)rows * c.NKV;
    a.win = units <= 4096 ? 1 : units <= 32768 ? 4 : 16;
    a.windows = (rows - 1) / a.win + 1;
    const long long wgs = ((long long)a.windows * c.NKV + 7) / 8 * 8;
    const int threads = c.page * c.HD / 32;
    if (!kv8_grid_ok(wgs, threads)) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs);
    switch (src_dtype) {
    case DT_FP32: return launch_append_t<DT_FP32>(a, grid, threads, st);
    case DT_F16: return launch_append_t<DT_F16>(a, grid, threads, st);
    case DT_BF16: return launch_append_t<DT_BF16>(a, grid, threads, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dgx
