// logprobs.hip — log probabilities of given tokens, the entropy of their distributions and the
// most likely alternatives, from rows of logits x:
//
//   lse = M + ln S,  S = sum_j e^(x_j - M),  M = max x
//   log p_j = (x_j - M) - ln S,   H = -sum p ln p = ln S - sum_j e^(x_j - M) (x_j - M) / S
//
// Both terms of H are positive, so that sharp distributions cancel nothing.
//
// The logits are read once.  A block takes a segment of kSeg values of a row in registers, 64
// to a lane: first the maximum, then S and the sum of H in its terms, and the segment's
// alternatives.  These are found by a bound that at least k values reach (of the lanes'
// maxima, k reach it in some wave): the few values that do go to LDS and are ranked by
// counting.  Where more reach it than LDS holds (many equal values), they are taken one
// after the other.  Order: larger first, equal ones by position, a whole number of both.
// A second launch joins the segments of a row (one segment: none).
#include <math.h>
#include <string.h>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kEach = 64;
constexpr int kSeg = kThreads * kEach;
constexpr int kCand = 1024;             // candidates that LDS holds

struct LpJob {
    int vocab, k, n_seg;
    const void *x;
    int64_t ld;
    const int32_t *token;
    float *lp, *entropy, *top_lp;
    int32_t *top;
    float *part;                        // [row][seg][4]: M, S, T
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

// A row's results from M, S, T (in units of ln 2) and its sorted alternatives.
template <bool BF16>
__device__ __forceinline__ void finish(const LpJob &J, int64_t row, float m, double s, double t,
                                       const u64 *best, int tid)
{
    const double ln_s = log(s);
    if (tid == 0) {
        if (J.lp) {
            const int x = J.token[row];
            const bool in = x >= 0 && x < J.vocab;
            J.lp[row] = in ? (float)((double)logit<BF16>(J.x, row * J.ld + x) - (double)m - ln_s)
                           : -__builtin_inff();
        }
        if (J.entropy) J.entropy[row] = (float)(ln_s - 0.6931471805599453 * (t / s));
    }
    if (tid < J.k) {
        const u64 key = best[tid];
        J.top[row * J.k + tid] = key ? index_of(key) : -1;
        J.top_lp[row * J.k + tid] = key ? (float)((double)value_of(key) - (double)m - ln_s)
                                        : -__builtin_inff();
    }
}

// best[0..k): the largest of n keys in order, 0 where there are fewer.  n <= kCand (all the
// block's threads; the keys differ).
__device__ __forceinline__ void rank(const u64 *cand, int n, u64 *best, int k, int tid)
{
    if (tid < k) best[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const u64 mine = cand[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += cand[j] > mine;
        if (r < k && mine) best[r] = mine;
    }
    __syncthreads();
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 4) void logprob_kernel(LpJob J)
{
    constexpr int V = BF16 ? 8 : 4, NV = kEach / V;
    __shared__ u64 cand[kCand], best[EAKVD_TOP_MAX], wbest[kThreads / 64];
    __shared__ float red[3][kThreads / 64];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t row = blockIdx.x / J.n_seg;
    const int seg = (int)(blockIdx.x - row * J.n_seg);
    // vectors are aligned: value i of the row is at place i + shift
    const int64_t at = row * J.ld;
    const int shift = (int)(((uintptr_t)J.x / (BF16 ? 2 : 4) + (uint64_t)at) % V);
    const int i0 = seg * kSeg + V * tid - shift;        // of the lane's first vector
    const float none = -__builtin_inff();
    float x[kEach];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = i0 + j * kThreads * V;
        if (i >= 0 && i + V <= J.vocab) {
            if constexpr (BF16) {
                typedef uint32_t v4u __attribute__((ext_vector_type(4)));
                const v4u y = __builtin_nontemporal_load((const v4u *)((const uint16_t *)J.x + at + i));
#pragma unroll
                for (int e = 0; e < 8; e++)
                    x[j * V + e] = __uint_as_float(e & 1 ? y[e >> 1] & 0xffff0000u : y[e >> 1] << 16);
            } else {
                const v4f y = __builtin_nontemporal_load((const v4f *)((const float *)J.x + at + i));
#pragma unroll
                for (int e = 0; e < 4; e++) x[j * V + e] = y[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++)
                x[j * V + e] = i + e >= 0 && i + e < J.vocab ? logit<BF16>(J.x, at + i + e) : none;
        }
    }
    if (tid == 0) n_cand = 0;
    float top = x[0];
#pragma unroll
    for (int e = 1; e < kEach; e++) top = fmaxf(top, x[e]);
    // the wave's bound: the largest top half of a float's order that k lanes reach
    float thr = none;
    if (J.k) {
        const uint32_t b = __float_as_uint(top + 0.0f);
        const uint32_t key = top > none ? b ^ (b >> 31 ? 0xffffffffu : 0x80000000u) : 0;
        uint32_t t = 0;
        for (int bit = 31; bit >= 12; bit--)
            if ((int)__popcll(__ballot(key >= (t | 1u << bit))) >= J.k) t |= 1u << bit;
        thr = t ? __uint_as_float(t >> 31 ? t ^ 0x80000000u : ~t) : none;
    }
    float m = wave_max(top);
    if (lane == 0) {
        red[0][w] = m;
        red[1][w] = thr;
    }
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    thr = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    __syncthreads();
    // (nothing but -inf: every term is 0)
    const float from = m == none ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const float z = (x[e] - from) * EAKV_LOG2E, p = __builtin_amdgcn_exp2f(z);
        s += p;
        t = fmaf(p, fmaxf(z, -1000.0f), t);     // (a term of 0, not NaN, for -inf)
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) {
        red[0][w] = s;
        red[1][w] = t;
    }
    if (J.k && top >= thr) {
#pragma unroll
        for (int j = 0; j < kEach; j += 8) {
            float most = x[j];
#pragma unroll
            for (int e = 1; e < 8; e++) most = fmaxf(most, x[j + e]);
            if (most >= thr)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (x[j + e] >= thr && x[j + e] > none) {
                        const int p = atomicAdd(&n_cand, 1);
                        const int v = (j + e) / V;
                        if (p < kCand) cand[p] = key_of(x[j + e], i0 + v * kThreads * V + (j + e) % V);
                    }
        }
    }
    __syncthreads();
    s = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    t = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (J.k) {
        if (n_cand <= kCand) {
            rank(cand, n_cand, best, J.k, tid);
        } else {
            // one after the other
            u64 prev = ~0ull;
            for (int r = 0; r < J.k; r++) {
                u64 mine = 0;
#pragma unroll
                for (int e = 0; e < kEach; e++) {
                    const u64 key = key_of(x[e], i0 + e / V * kThreads * V + e % V);
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
        finish<BF16>(J, row, from, s, t, best, tid);
        return;
    }
    const int64_t p = row * J.n_seg + seg;
    if (tid == 0) *(v4f *)(J.part + p * 4) = v4f{m, s, t, 0.0f};
    if (tid < J.k) J.list[p * J.k + tid] = best[tid];
}

// A row's segments joined, a block to a row.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LpJob J)
{
    __shared__ u64 cand[kCand], best[EAKVD_TOP_MAX];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const float *part = J.part + row * J.n_seg * 4;
    float m = -__builtin_inff();
    for (int i = 0; i < J.n_seg; i++) m = fmaxf(m, part[4 * i]);
    const float from = m == -__builtin_inff() ? 0.0f : m;
    double s = 0.0, t = 0.0;
    for (int i = 0; i < J.n_seg; i++) {
        const v4f x = *(const v4f *)(part + 4 * i);
        const float mine = x[0] == -__builtin_inff() ? 0.0f : x[0];
        // (a segment of -inf has S = 0, at any M)
        const double d = ((double)mine - (double)from) * 1.4426950408889634, f = exp2(d);
        if (x[1] == 0.0f) continue;
        s += f * (double)x[1];
        if (f != 0.0) t += f * ((double)x[2] + (double)x[1] * d);
    }
    if (J.k) {
        // the lists' keys, kCand at a time, beside the best so far
        const int all = J.n_seg * J.k;
        int n = 0;
        for (int a = 0; a < all;) {
            const int more = min(kCand - n, all - a);
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) cand[i] = best[i];
            for (int i = tid; i < more; i += kThreads) cand[n + i] = J.list[row * all + a + i];
            __syncthreads();
            rank(cand, n + more, best, J.k, tid);
            a += more;
            n = J.k;
        }
    }
    finish<BF16>(J, row, from, s, t, best, tid);
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
    const dim3 grid((unsigned)((int64_t)n_rows * J.n_seg)), rows((unsigned)n_rows), nt(kThreads);
    auto *kern = bf16 ? logprob_kernel<true> : logprob_kernel<false>;
    auto *join = bf16 ? logprob_join_kernel<true> : logprob_join_kernel<false>;
    hipLaunchKernelGGL(kern, grid, nt, 0, st, J);
    if (J.n_seg > 1) hipLaunchKernelGGL(join, rows, nt, 0, st, J);
    return (int)hipGetLastError();
}
