// logprobs.hip — log probabilities of given tokens, the entropy of their distributions and the
// most likely alternatives, from rows of logits x:
//
//   lse = M + ln S,  S = sum_j e^(x_j - M),  M = max x
//   log p_j = (x_j - M) - ln S,   H = -sum p ln p = ln S - sum_j e^(x_j - M) (x_j - M) / S
//
// Both terms of H are positive, so that sharp distributions cancel nothing.
//
// The logits are read once.  A block takes a segment of kSeg values of a row in registers, 64
// to a lane (bf16: two to a register): first the maximum, then S and the sum of H in its terms,
// and the segment's alternatives.  These are found by a bound that at least k values reach (in
// every wave the maxima of k / 4 lanes do): the few values that do go to LDS and are ranked by
// counting.  Where more reach it than LDS holds (many equal values), they are taken one
// after the other.  Order: larger first, equal ones by position, a whole number of both.
// A second launch joins the segments of a row (one segment: none).
//
// Exponents are z = x log2(e) - c, one instruction, c = M log2(e) rounded: all are off by the
// same r = M log2(e) - c, which S, T and H are rid of at the end (S 2^-r).  (From 2^20 on r is
// not small: differences first.)
//
// Errors, e = 2^-24, u = M - x: a term by 2 e (exponential) and 1.3 e u (z's rounding and log2(e)'s;
// differences 2.3, a segment's factor 1 more), its sum by 18 roundings (8 terms, 3 steps, 6 over a wave,
// 2 over waves).  The mean of u is at most H, so ln S is off by (22 + 3.3 H) e; T by 24 e of itself and 3.3 e
// of the mean of u^2, at most 30 H: H by (24 + 128 H) e.
//
// Bound by vector instructions (14 a bf16 value with entropy and alternatives, 90 % of the cycles)
// for bf16, by HBM for f32; small calls by two launches' latency.  500 rows of 151665, 20
// alternatives: bf16 45-47 us (3.3 TB/s; without alternatives 34), f32 61-62 us (4.9); one row of
// 32000 f32 9.1 us.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kEach = 64;
constexpr int kSeg = kThreads * kEach;
static_assert(kThreads == 256, "four waves");
// S and T of a lane, each so many sums side by side: in one chain of 64 equal terms the roundings are
// alike and add up (ln p 2.7e-6 off, entropies 1e-5; so 4e-7 and 3e-6, at 44.7 against 44.2 us for 500
// rows of 151665 bf16).
constexpr int kSums = 8;
constexpr int kCand = 512;              // candidates that LDS holds for a block
constexpr int kGroups = 128;            // and groups of 8 values with one
constexpr int kHeld = 512;              // keys of a row's segments that its joining wave holds

struct LpJob {
    int vocab, k, n_seg;
    const void *x;
    int64_t ld;
    const int32_t *token;
    float *lp, *entropy, *top_lp;
    int32_t *top;
    float *part;                        // [row][seg][4]: M, S, T, r
    uint64_t *list;                     // [row][seg][k]
};

typedef uint64_t u64;

// A value and its position as one whole number: larger values first, then lower positions.
// 0: nothing (-inf and NaN are no alternatives).
__device__ __forceinline__ u64 key_of(float x, int i)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x > -__builtin_inff() ? (u64)(b ^ (b >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~i : 0;
}
__device__ __forceinline__ float value_of(u64 key)
{
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ u64 wave_max64(u64 v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const u64 u = __shfl_xor(v, o, 64);
        v = u > v ? u : v;
    }
    return v;
}

template <bool BF16>
__device__ __forceinline__ float logit(const void *x, int64_t at)
{
    if constexpr (BF16) return __uint_as_float((uint32_t)((const uint16_t *)x)[at] << 16);
    else return ((const float *)x)[at];
}

// e^x, |x| <= 0.35, to 2e-10: the series' terms up to x^8.
__device__ __forceinline__ double exp_near(double x)
{
    double y = 1.0 / 40320;
    y = fma(y, x, 1.0 / 5040);
    y = fma(y, x, 1.0 / 720);
    y = fma(y, x, 1.0 / 120);
    y = fma(y, x, 1.0 / 24);
    y = fma(y, x, 1.0 / 6);
    y = fma(y, x, 0.5);
    y = fma(y, x, 1.0);
    return fma(y, x, 1.0);
}

// ln s of a sum, from its exponent e and the rest f, of 1 to 2: g = log2 f by the f32 instruction,
// then f 2^-g - 1, which is ln f - g ln 2 but for its square.  (With the library's functions of 64
// bits, here and in put_right, a launch took 0.3 us more.)
__device__ __forceinline__ double ln_of(double s)
{
    constexpr double ln2 = 0.6931471805599453;
    const uint64_t b = (uint64_t)__double_as_longlong(s);
    const int e = (int)(b >> 52);
    // 0, infinite and NaN sums as f32 has them
    if (e <= 0 || e >= 0x7ff) return (double)__builtin_amdgcn_logf((float)s);
    const double f = __longlong_as_double((long long)((b & 0xfffffffffffffull) | 0x3ff0000000000000ull));
    const double g = (double)__builtin_amdgcn_logf((float)f);
    const double d = fma(f, 0.7071067811865476 * exp_near(ln2 * (0.5 - g)), -1.0);
    return fma(ln2, g + (double)(e - 1023), d);
}

// A row's results from M, S, T (in units of ln 2), the given token's logit and the sorted
// alternatives.
__device__ __forceinline__ void finish(const LpJob &J, int64_t row, float m, double s, double t, int token,
                                       float given, const u64 *best, int tid)
{
    // The largest logit's own term is 1, but rounded here (its z is r), so that a sum of little else may
    // come out below: ln S >= 0 and H >= 0 are kept.  (A sum of 0, nothing but -inf, stays -inf.)
    double ln_s = ln_of(s);
    if (s > 0.0 && ln_s < 0.0) ln_s = 0.0;
    if (tid == 0) {
        if (J.lp)
            J.lp[row] = token >= 0 && token < J.vocab ? (float)((double)given - (double)m - ln_s)
                                                      : -__builtin_inff();
        if (J.entropy) {
            // t / s: the f32 reciprocal and a step of Newton's
            const double y = (double)__builtin_amdgcn_rcpf((float)s);
            const double h = ln_s - 0.6931471805599453 * (t * (y * fma(-s, y, 2.0)));
            J.entropy[row] = h < 0.0 ? 0.0f : (float)h;
        }
    }
    if (tid < J.k) {
        const u64 key = best[tid];
        J.top[row * J.k + tid] = key ? index_of(key) : -1;
        J.top_lp[row * J.k + tid] = key ? (float)((double)value_of(key) - (double)m - ln_s)
                                        : -__builtin_inff();
    }
}

// S and T of terms whose exponents are all off by r
__device__ __forceinline__ void put_right(double r, double &s, double &t)
{
    const double f = exp_near(-0.6931471805599453 * r);         // (|r| < 0.1)
    t = f * (t - r * s);
    s = f * s;
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// (the compiler makes a number of __ballot's argument first)
__device__ __forceinline__ uint64_t ballot(bool b) { return __builtin_amdgcn_ballot_w64(b); }

// best[0..k): the largest of n different keys in order, 0 where there are fewer (as best is).
// cand: 16-byte aligned, 8 zeros behind the keys.  Thread tid of `threads`.
__device__ __forceinline__ void rank(u64 *cand, int n, u64 *best, int k, int tid, int threads)
{
    for (int i = tid; i < n; i += threads) {
        const u64 mine = cand[i];
        int r = 0;
        for (int j = 0; j < n; j += 8) {
            u64 y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = cand[j + e];
#pragma unroll
            for (int e = 0; e < 8; e++) r += y[e] > mine;
        }
        if (r < k && mine) best[r] = mine;
    }
}

// A bound that the maxima of k lanes of a wave reach, in 16 bits of a float's order (-inf: fewer
// lanes have one).
__device__ __forceinline__ float reached(float top, int k)
{
    const uint32_t b = __float_as_uint(top + 0.0f);
    const uint32_t key = top > -__builtin_inff() ? b ^ (b >> 31 ? 0xffffffffu : 0x80000000u) : 0;
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--)
        if ((int)__popcll(ballot(key >= (t | 1u << bit))) >= k) t |= 1u << bit;
    return t ? __uint_as_float(t >> 31 ? t ^ 0x80000000u : ~t) : -__builtin_inff();
}

// TOP, ENT: whether alternatives and entropies are wanted.
template <bool BF16, bool TOP, bool ENT>
__global__ __launch_bounds__(kThreads, 4) void logprob_kernel(LpJob J)
{
    constexpr int V = BF16 ? 8 : 4, NV = kEach / V, NX = BF16 ? kEach / 2 : kEach;
    __shared__ __align__(16) u64 cand[TOP ? kCand + 8 : 1];
    __shared__ u64 best[EAKVD_TOP_MAX], wbest[kThreads / 64];
    __shared__ float red[3][kThreads / 64];
    __shared__ int n_cand, n_group[kThreads / 64];
    __shared__ uint16_t groups[kThreads / 64][TOP ? kGroups : 1];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    if constexpr (TOP) {
        for (int i = tid; i < kCand + 8; i += kThreads) cand[i] = 0;
        if (tid < EAKVD_TOP_MAX) best[tid] = 0;
        if (tid == 0) n_cand = 0;
    }
    const int64_t row = blockIdx.x / J.n_seg;
    const int seg = (int)(blockIdx.x - row * J.n_seg);
    // vectors are aligned: value i of the row is at place i + shift
    const int64_t at = row * J.ld;
    const int shift = (int)(((uintptr_t)J.x / (BF16 ? 2 : 4) + (uint64_t)at) % V);
    const int i0 = seg * kSeg + V * tid - shift;        // of the lane's first vector
    const float none = -__builtin_inff();
    uint32_t raw[NX];
    auto x = [&](int e) __attribute__((always_inline)) {
        if constexpr (BF16) return __uint_as_float(e & 1 ? raw[e >> 1] & 0xffff0000u : raw[e >> 1] << 16);
        else return __uint_as_float(raw[e]);
    };
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = i0 + j * kThreads * V;
        v4u y;
        if (i >= 0 && i + V <= J.vocab) {
            y = __builtin_nontemporal_load((const v4u *)((const uint8_t *)J.x + (at + i) * (BF16 ? 2 : 4)));
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                auto word = [&](int k) {
                    return i + k >= 0 && i + k < J.vocab ? __float_as_uint(logit<BF16>(J.x, at + i + k)) : 0xff800000u;
                };
                if constexpr (BF16) y[e] = word(2 * e) >> 16 | word(2 * e + 1);
                else y[e] = word(e);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) raw[j * 4 + e] = y[e];
    }
    // (two values of a register are taken apart where they are used, not kept apart)
    auto hold = [&]() __attribute__((always_inline)) {
        if constexpr (BF16)
#pragma unroll
            for (int k = 0; k < NX; k++) asm("" : "+v"(raw[k]));
    };
    float high[kEach / 8];                              // of 8 values each
#pragma unroll
    for (int j = 0; j < kEach / 8; j++)
        high[j] = max3(max3(max3(x(8 * j), x(8 * j + 1), x(8 * j + 2)), x(8 * j + 3), x(8 * j + 4)),
                       max3(x(8 * j + 5), x(8 * j + 6), x(8 * j + 7)), x(8 * j + 7));
    const float top = max3(max3(max3(high[0], high[1], high[2]), high[3], high[4]), max3(high[5], high[6], high[7]),
                           high[7]);
    hold();
    const float bound = TOP ? reached(top, (J.k + 3) / 4) : none;
    float m = wave_max(top);
    if (lane == 0) {
        red[0][w] = m;
        red[1][w] = bound;
    }
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float thr = fminf(fminf(red[1][0], red[1][1]), fminf(red[1][2], red[1][3]));
    __syncthreads();
    if (TOP && thr == none) {
        // a wave has too few: what k lanes of one reach
        const float b = reached(top, J.k);
        if (lane == 0) red[2][w] = b;
        __syncthreads();
        thr = fmaxf(fmaxf(red[2][0], red[2][1]), fmaxf(red[2][2], red[2][3]));
    }
    // (nothing but -inf: every term is 0)
    const float from = m == none ? 0.0f : m;
    const float c = from * EAKV_LOG2E;
    float r = fmaf(from, EAKV_LOG2E, -c), s8[kSums] = {}, t8[kSums] = {};
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const float z = fmaf(x(e), EAKV_LOG2E, -c), p = __builtin_amdgcn_exp2f(z);
        s8[e % kSums] += p;
        if constexpr (ENT) t8[e % kSums] = fmaf(p, fmaxf(z, -1000.0f), t8[e % kSums]);  // (a term of 0, not NaN, for -inf)
    }
#pragma unroll
    for (int n = kSums / 2; n >= 1; n /= 2)
#pragma unroll
        for (int k = 0; k < n; k++) {
            s8[k] += s8[k + n];
            t8[k] += t8[k + n];
        }
    float s = s8[0], t = t8[0];
    if (!(fabsf(from) < 0x1p20f)) {
        // r is not small: from differences, read again
        double sd = 0.0, td = 0.0;
        for (int i = max(seg * kSeg - shift, 0) + tid; i < min((seg + 1) * kSeg - shift, J.vocab); i += kThreads) {
            const float z = (logit<BF16>(J.x, at + i) - from) * EAKV_LOG2E, p = __builtin_amdgcn_exp2f(z);
            sd += (double)p;
            td = fma((double)p, (double)fmaxf(z, -1000.0f), td);
        }
        s = (float)sd;
        t = (float)td;
        r = 0.0f;
    }
    hold();
    s = wave_sum(s);
    if constexpr (ENT) t = wave_sum(t);
    if (lane == 0) {
        red[0][w] = s;
        red[1][w] = t;
    }
    // groups of 8 with a value that reaches the bound
    if constexpr (TOP) {
        int found = 0;
#pragma unroll
        for (int j = 0; j < kEach / 8; j++) {
            const bool in = high[j] >= thr && high[j] > none;
            const uint64_t b = ballot(in);
            if (b == 0) continue;
            const int p = found + (int)__popcll(b & ((1ull << lane) - 1));
            if (in && p < kGroups) groups[w][p] = (uint16_t)(tid * (kEach / 8) + j);
            found += (int)__popcll(b);
        }
        if (lane == 0) n_group[w] = found;
    }
    __syncthreads();
    s = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    t = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if constexpr (TOP) {
        // their values, one to a thread, read again
        const int g0 = n_group[0], g1 = g0 + n_group[1], g2 = g1 + n_group[2], all = g2 + n_group[3];
        bool fits = max(max(n_group[0], n_group[1]), max(n_group[2], n_group[3])) <= kGroups && all <= 4 * kGroups;
        if (fits) {
            for (int q0 = 0; q0 < 8 * all; q0 += kThreads) {
                const int q = q0 + tid, g = q >> 3;
                u64 key = 0;
                if (g < all) {
                    const int v = (g >= g0) + (g >= g1) + (g >= g2);
                    const int id = groups[v][g - (v == 0 ? 0 : v == 1 ? g0 : v == 2 ? g1 : g2)];
                    const int e = id % (kEach / 8) * 8 + (q & 7);
                    const int i = seg * kSeg + V * (id / (kEach / 8)) - shift + e / V * kThreads * V + e % V;
                    if (i >= 0 && i < J.vocab) {
                        const float y = logit<BF16>(J.x, at + i);
                        key = y >= thr ? key_of(y, i) : 0;
                    }
                }
                // (places in any order: the keys' own order decides)
                const uint64_t b = ballot(key != 0);
                int p = 0;
                if (lane == 0 && b) p = atomicAdd(&n_cand, (int)__popcll(b));
                p = __builtin_amdgcn_readfirstlane(p) + (int)__popcll(b & ((1ull << lane) - 1));
                if (key && p < kCand) cand[p] = key;
            }
            __syncthreads();
            fits = n_cand <= kCand;
        }
        if (fits) {
            rank(cand, n_cand, best, J.k, tid, kThreads);
            __syncthreads();
        } else {
            // one after the other, read again
            u64 prev = ~0ull;
            for (int r = 0; r < J.k; r++) {
                u64 mine = 0;
                for (int i = max(seg * kSeg - shift, 0) + tid; i < min((seg + 1) * kSeg - shift, J.vocab); i += kThreads) {
                    const u64 key = key_of(logit<BF16>(J.x, at + i), i);
                    mine = key < prev && key > mine ? key : mine;
                }
                mine = wave_max64(mine);
                if (lane == 0) wbest[w] = mine;
                __syncthreads();
                for (int i = 0; i < kThreads / 64; i++) mine = wbest[i] > mine ? wbest[i] : mine;
                prev = mine;
                if (tid == 0) best[r] = mine;
                __syncthreads();
            }
        }
    }
    if (J.n_seg == 1) {
        double sd = s, td = t;
        put_right(r, sd, td);
        const int token = J.lp ? J.token[row] : -1;
        const float given = token >= 0 && token < J.vocab ? logit<BF16>(J.x, at + token) : none;
        finish(J, row, from, sd, td, token, given, best, tid);
        return;
    }
    const int64_t p = row * J.n_seg + seg;
    if (tid == 0) *(v4f *)(J.part + p * 4) = v4f{m, s, t, r};
    if (tid < J.k) J.list[p * J.k + tid] = best[tid];
}

// A row's segments joined, a wave to a row.  Alternatives: a bound that k of the lists' keys reach,
// bit by bit; those that do are ranked by counting (or, where the lists are more than LDS
// holds, taken one after the other).
template <bool BF16>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LpJob J, int n_rows)
{
    __shared__ __align__(16) u64 cands[kThreads / 64][kHeld + 8];
    __shared__ u64 bests[kThreads / 64][EAKVD_TOP_MAX];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, k = J.k, n_seg = J.n_seg;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + w;
    if (row >= n_rows) return;
    u64 *cand = cands[w], *best = bests[w];
    const float none = -__builtin_inff();
    const v4f *part = (const v4f *)J.part + row * n_seg;
    // all loads at once: the lists, the segments' sums, the given token's logit
    const u64 *list = J.list + row * n_seg * k;
    const int all = n_seg * k;
    u64 key[kHeld / 64];
#pragma unroll
    for (int i = 0; i < kHeld / 64; i++) key[i] = lane + 64 * i < all ? list[lane + 64 * i] : 0;
    const int token = J.lp ? J.token[row] : -1;
    const v4f first = part[min(lane, n_seg - 1)];
    const float given = token >= 0 && token < J.vocab ? logit<BF16>(J.x, row * J.ld + token) : none;
    float m = lane < n_seg ? first[0] : none;
    for (int i = lane + 64; i < n_seg; i += 64) m = fmaxf(m, part[i][0]);
    m = wave_max(m);
    const float from = m == none ? 0.0f : m;
    double s = 0.0, t = 0.0;
    for (int i = lane; i < n_seg; i += 64) {
        const v4f x = i < 64 ? first : part[i];
        const float mine = x[0] == none ? 0.0f : x[0];
        // (a segment of -inf has S = 0, at any M)
        if (x[1] == 0.0f) continue;
        double si = x[1], ti = x[2];
        put_right(x[3], si, ti);
        const double d = ((double)mine - (double)from) * 1.4426950408889634,
                     f = (double)__builtin_amdgcn_exp2f((float)d);
        s += f * si;
        if (f != 0.0) t += f * (ti + si * d);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        t += __shfl_xor(t, o, 64);
    }
    if (k) {
        int found = kHeld + 1;
        if (all <= kHeld) {
            // a bound that k keys reach, in 16 bits of the value's order (0: there are fewer); up to 64 keys
            // are ranked without
            uint32_t t = 0;
#pragma unroll 1
            for (int bit = all > 64 ? 31 : 15; bit >= 16; bit--) {
                const uint32_t c = t | 1u << bit;
                int n = 0;
#pragma unroll
                for (int i = 0; i < kHeld / 64; i++)
                    if (64 * i < all) n += (int)__popcll(ballot((uint32_t)(key[i] >> 32) >= c));
                t = n >= k ? c : t;
            }
            found = 0;
#pragma unroll
            for (int i = 0; i < kHeld / 64; i++) {
                const bool in = key[i] != 0 && (uint32_t)(key[i] >> 32) >= t;
                const uint64_t b = ballot(in);
                const int p = found + (int)__popcll(b & ((1ull << lane) - 1));
                if (in) cand[p] = key[i];
                found += (int)__popcll(b);
            }
        }
        if (lane < k) best[lane] = 0;
        if (found <= kHeld && lane < 8) cand[found + lane] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (found <= kHeld) {
            rank(cand, found, best, k, lane, 64);
        } else {
            u64 prev = ~0ull;
            for (int r = 0; r < k; r++) {
                u64 mine = 0;
                for (int i = lane; i < all; i += 64) {
                    const u64 x = list[i];
                    mine = x < prev && x > mine ? x : mine;
                }
                prev = wave_max64(mine);
                if (lane == 0) best[r] = prev;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    finish(J, row, from, s, t, token, given, best, lane);
}

// (a row's first vector may begin up to 7 places before it)
int segments(int vocab) { return (int)(((int64_t)vocab + 7 + kSeg - 1) / kSeg); }

}  // namespace

extern "C" size_t eakvd_logprobs_work_bytes(int n_rows, int vocab, int n_top)
{
    const int n = segments(vocab);
    return n == 1 ? 0 : (size_t)n_rows * n * (16 + 8 * (size_t)n_top);
}

extern "C" int eakvd_logprobs(int n_rows, int vocab, const void *logits, int bf16, int64_t ld,
                              const int32_t *tokens, int n_top, float *logprobs, float *entropy,
                              int32_t *top_tokens, float *top_logprobs, void *work, void *stream)
{
    LpJob J;
    J.vocab = vocab;
    J.k = n_top;
    J.n_seg = segments(vocab);
    J.x = logits;
    J.ld = ld;
    J.token = tokens;
    J.lp = logprobs;
    J.entropy = entropy;
    J.top = top_tokens;
    J.top_lp = top_logprobs;
    J.part = (float *)work;
    J.list = (u64 *)((uint8_t *)work + (size_t)n_rows * J.n_seg * 16);
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)((int64_t)n_rows * J.n_seg)), nt(kThreads);
    const dim3 rows((unsigned)((n_rows + kThreads / 64 - 1) / (kThreads / 64)));
    const bool top = n_top > 0, ent = entropy != nullptr;
    auto pick = [&](auto b) {
        constexpr bool B = decltype(b)::value;
        return top ? (ent ? logprob_kernel<B, true, true> : logprob_kernel<B, true, false>)
                   : (ent ? logprob_kernel<B, false, true> : logprob_kernel<B, false, false>);
    };
    auto *kern = bf16 ? pick(std::true_type()) : pick(std::false_type());
    auto *join = bf16 ? logprob_join_kernel<true> : logprob_join_kernel<false>;
    hipLaunchKernelGGL(kern, grid, nt, 0, st, J);
    if (J.n_seg > 1) hipLaunchKernelGGL(join, rows, nt, 0, st, J, n_rows);
    return (int)hipGetLastError();
}
