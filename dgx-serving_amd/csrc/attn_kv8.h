// The paged 8-bit KV cache: descriptors shared by its kernels and the C-ABI layer, and the device-side arithmetic of its
// format.
//
// K and V are OCP e4m3 codes in pages of `page` tokens (16, 32 or 64), with a scale 2^e of each (page, KV head) for K and
// for V: value = code * 2^e, e in [kv8_emin, kv8_emax]. A power of two, because then
//   * x / 2^e is exact, so a stored value is off by one rounding to e4m3 and by nothing else,
//   * a page whose scale grows keeps the bits of its codes but for those that leave the normal range,
//   * the attention kernels fold the K scale into the factor that the scores are multiplied by anyway and the V scale into
//     the exponent of the probabilities (P = 2^(s + e - m) multiplies the bare codes): neither costs an operation per element.
// Layout, chosen for the matrix operands (16 bytes per lane straight from memory, no transpose in any kernel):
//   K  [pages][NKV][page][HD]      V  [pages][NKV][HD][page]      Ks, Vs  [pages][NKV]
#pragma once
#include "attn_device.h"
#include "attn_internal.h"
#include <climits>

namespace dgx {

struct Kv8 {
    uint8_t *K, *V;
    float *Ks, *Vs;
    int pages, page, lp;              // lp = log2(page)
    int NKV, HD;
};

constexpr int kv8_emin = -40, kv8_emax = 40;

// The least e with amax <= 448 * 2^e, within the bounds: 448 = 1.75 * 2^8, so amax = m * 2^k takes e = k - 8 while its
// mantissa is at most 1.75. amax is finite and not negative.
__device__ __forceinline__ int kv8_exponent(float amax) {
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return min(max(e, kv8_emin), kv8_emax);
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
// Exponent of a scale, at most 126: the scale of a page that holds no token yet may be anything, its keys weigh 0, and 0 times
// 2^-exponent has to stay 0.
__device__ __forceinline__ int exp_of(float scale) { return min((int)((__float_as_uint(scale) >> 23) & 255u), 253) - 127; }

// Two e4m3 codes (bytes 2 * HI, 2 * HI + 1 of w) as a packed pair of 16-bit MFMA operands; exact in either format.
template <bool F16, bool HI> __device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
}
// Eight codes as one MFMA operand (8 consecutive elements of the reduction).
template <bool F16> __device__ __forceinline__ u32x4 e4m3_op(uint32_t w0, uint32_t w1) {
    return u32x4{e4m3_pair<F16, false>(w0), e4m3_pair<F16, true>(w0), e4m3_pair<F16, false>(w1), e4m3_pair<F16, true>(w1)};
}
// Four values of at most 448 to e4m3 codes: nearest, ties to even.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// One call of the attention: row r of Q / O / lse belongs to request b for r in [cu[b], cu[b + 1]) (cu null: T rows each),
// its position is ctx[b] + r - cu[b], its keys are those of the request's pages in `table`.
struct Kv8Problem {
    Kv8 c;
    const void *Q; int q_dtype;
    void *O; int o_dtype;
    float *lse;
    int B, T, rows, NQ;
    const int *ctx, *cu, *table;
    long table_stride;
    const uint32_t *anc;              // tree masks [rows], relative to the request's first row
    int max_pos;
    float scale;
    int window;
};

// Row range of request b: at most T rows, within the `rows` of the buffers.
__device__ __forceinline__ void kv8_rows(const Kv8Problem &p, int b, int &r0, int &n) {
    if (p.cu) {
        r0 = min(max(p.cu[b], 0), p.rows);
        n = min(min(max(p.cu[b + 1], r0), p.rows) - r0, p.T);
    } else {
        r0 = b * p.T;
        n = p.T;
    }
}

// Position of request b's first row, which leaves its n rows below INT_MAX.
__device__ __forceinline__ int kv8_first_pos(const Kv8Problem &p, int b, int n) { return min(p.ctx[b], INT_MAX - n); }

// Partials of a split call: index (r * NQ + head) * ns + split; acc[HD], reference exponent m and sum l: the row's output is
// sum acc 2^(m - M) / sum l 2^(m - M) over the splits, M the largest m. Splits lie at absolute keys c C .., but are counted from
// the one with the first key of the request's first row: behind a window the room that a row needs does not grow with the
// positions (16 drafts of 8 tokens, 16 q-heads over 8 of 256, window 1024, max_pos 131071: 13 MB, counted from key 0 1082).
struct Kv8Partials {
    float *m, *l, *acc;
    int ns, C;                        // splits that a row has room for, keys of a split (0: none, the kernel writes O itself)
};

// A value that is the same in all lanes and that no kernel of this library writes while this one runs, through the scalar
// cache: page ids and scales then cost no vector registers and no wait behind the vector loads in flight.
template <class T> __device__ __forceinline__ T scalar_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(uintptr_t)p;
}

// Four neighbouring dims of an output row, rounded once to the type of O.
__device__ __forceinline__ void kv8_store4(const Kv8Problem &p, size_t at, const f32x4 &v) {
    if (p.o_dtype == DT_FP32) *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(p.O) + at) = v;
    else *reinterpret_cast<u32x2 *>(reinterpret_cast<uint16_t *>(p.O) + at) =
        p.o_dtype == DT_F16 ? u32x2{pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3])} : u32x2{pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3])};
}

// Merge weight of a partial state (m, l) under the common reference M >= m. A state that saw no key has m = -inf and
// l = 0; one whose only keys were NaN has m = -inf and l = NaN, which must reach the result.
__device__ __forceinline__ float kv8_weight(float m, float l, float M) { return m == kNegInf ? l * 0.f : fast_exp2(m - M); }

// A launch holds less than 2^32 threads.
inline bool kv8_grid_ok(long long wgs, int threads) { return wgs <= 0x7fffffff && wgs * threads <= 0xffffffffll; }

hipError_t launch_kv8_plan(const int *ctx, const int *add, int B, int lp, int *table, long table_stride, int cols,
                           const int *free_pages, int free_cap, const int *free_in, int *free_out, int *cu, int *slots, int rows,
                           int *status, hipStream_t st);
hipError_t launch_kv8_append(const void *k, const void *v, int src_dtype, long k_stride, long v_stride, const Kv8 &c,
                             const int *slots, int rows, unsigned *stats, hipStream_t st);

// Split-KV form: single tokens, short runs, trees, small prompts (any T; rows of a KV head in groups of 16 nt, nt 1, 2 or 4;
// at HD 512 1 or 2).
struct Kv8Plan;
hipError_t launch_kv8_decode(const Kv8Problem &p, const Kv8Partials &part, const Kv8Plan &pl, hipStream_t st);
// Prompt form: 64 or 128 rows of a KV head per workgroup, no tree masks.
hipError_t launch_kv8_prefill(const Kv8Problem &p, const Kv8Partials &part, const Kv8Plan &pl, hipStream_t st);
hipError_t launch_kv8_combine(const Kv8Problem &p, const Kv8Partials &part, hipStream_t st);

// What a call runs: the rows of a prompt tile (0: the split-KV form, in groups of 16 nt rows), the keys of a split (0: the
// prompt form's one pass) and how many splits the keys of one request's rows reach at most (1: the kernel writes O, no
// workspace).
struct Kv8Plan { int tile, nt, C, ns; };
Kv8Plan kv8_choose(int B, int T, int rows, int NQ, int NKV, int HD, int max_pos, int chunk, int window, bool tree);

}  // namespace dgx
