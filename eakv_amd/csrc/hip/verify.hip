// verify.hip — which drafted tokens the target model keeps, and the token after
// them (speculative sampling), for a padded batch of drafts.
//
// Draft i with token x is kept while u_i * q_i(x) < p_i(x) (u in [0, 1), so kept
// with probability min(1, p/q)).  a = the number kept.  The next token is drawn
// from r = max(p_a - q_a, 0) after a rejection, from r = p_a when all were kept:
// the least j whose sum r[0..j] exceeds u * sum(r).
//
// Every comparison is of exact products and differences of f32 values in f64, and
// the sums are f64: the result does not depend on the order of a sum unless the
// drawn number lies within 1e-15 of a step.
//
// Work: one row of p and one of q per sequence, bound by HBM for large batches and
// by latency for small ones.  Small vocabularies: one launch, a block of 16 waves per
// sequence.  Else two: each wave sums one segment of its
// sequence's row; one block per sequence then finds the segment and scans it, in one
// step up to 2^18 tokens.  7 drafts of 64 sequences, 151665 tokens (77.7 MB): 14.0 us of
// sums (5.5 TB/s) and 4.6 of scan; with a segment of 4096 values to a block, scanned in
// four steps, 13.9 and 11.8.  One sequence: two launches' latency, 7.4 us.
#include "common.h"

namespace {

constexpr int kVerThreads = 256;
// Vocabularies up to this take one launch (the block's f64 sums take the time of the second
// launch there): one / two for 32 sequences, us: 2000 5.6 / 9.4, 8000 7.0 / 9.2, 12000 8.0 / 8.9,
// 16000 8.9 / 8.8, 32000 12.8 / 8.1.
constexpr int kVerOne = 12288;
constexpr int kVerStep = 1024;          // values of a wave's step, a multiple of 256

typedef float v4f4 __attribute__((ext_vector_type(4), aligned(4)));

struct VerJob {
    int k, vocab, n_seg, seg;   // seg: values of a wave's segment
    const int32_t *count, *token;
    const float *draft, *target, *uniform;
    int64_t ld_draft, ld_target;
    int32_t *kept, *next;
    double *part;               // [n_seqs][n_seg][2]: sums of r and of p
};

__device__ __forceinline__ int count_of(const VerJob &J, int s)
{
    const int n = J.count ? J.count[s] : J.k;
    return n < 0 ? 0 : n > J.k ? J.k : n;
}

// Negative values and NaN as 0, in one instruction (the median takes NaN for the least).
__device__ __forceinline__ float some(float x)
{
    return __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff());
}

// The drafts of sequence s that are kept (every lane of a wave gets it).
__device__ __forceinline__ int kept_of(const VerJob &J, int s, int n, int lane)
{
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        bool ok = false;
        if (i < n) {
            const int64_t at = (int64_t)s * J.k + i;
            const int x = J.token[at];
            if (x >= 0 && x < J.vocab) {
                const float p = J.target[((int64_t)s * (J.k + 1) + i) * J.ld_target + x];
                const float q = J.draft ? some(J.draft[at * J.ld_draft + x]) : 1.0f;
                ok = (double)J.uniform[(int64_t)s * (J.k + 1) + i] * (double)q < (double)p;
            }
        }
        const uint64_t bad = __ballot(i < n && !ok);
        if (bad) return i0 + __ffsll((unsigned long long)bad) - 1;
    }
    return n;
}

// The row that the next token is drawn from.
struct Row {
    const float *p, *q;         // q NULL: no draft row
    int less;                   // a token whose weight is 0 (one-hot draft), or -1
    // (negative values and NaN are 0 in both)
    __device__ __forceinline__ double at(float p_, float q_, int j) const
    {
        const double r = q ? (double)p_ - (double)some(q_) : (double)p_;
        return j != less && r > 0.0 ? r : 0.0;
    }
};

__device__ __forceinline__ Row row_of(const VerJob &J, int s, int n, int kept)
{
    Row r;
    r.p = J.target + ((int64_t)s * (J.k + 1) + kept) * J.ld_target;
    const int64_t at = (int64_t)s * J.k + kept;
    r.q = kept < n && J.draft ? J.draft + at * J.ld_draft : nullptr;
    r.less = kept < n && !J.draft ? J.token[at] : -1;
    return r;
}

__device__ __forceinline__ double wave_sum_d(double v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__global__ __launch_bounds__(kVerThreads) void verify_sum_kernel(VerJob J)
{
    const int s = blockIdx.y, lane = threadIdx.x & 63;
    const int b = (int)blockIdx.x * (kVerThreads / 64) + (threadIdx.x >> 6);
    if (b >= J.n_seg) return;
    const int n = count_of(J, s);
    const int kept = kept_of(J, s, n, lane);
    if (b == 0 && lane == 0) J.kept[s] = kept;
    const Row R = row_of(J, s, n, kept);
    const int lo = b * J.seg, hi = min(J.vocab, lo + J.seg);
    double sr = 0.0, sp = 0.0;
    auto add = [&](float p, float q, int j) {
        sr += R.at(p, q, j);
        sp += p > 0.0f ? (double)p : 0.0;
    };
    int j = lo + 4 * lane;
    // a whole step: all loads in flight before the first sum
    for (; j - 4 * lane + kVerStep <= hi; j += kVerStep) {
        v4f4 p[kVerStep / 256], q[kVerStep / 256];
#pragma unroll
        for (int i = 0; i < kVerStep / 256; i++) p[i] = *(const v4f4 *)(R.p + j + 256 * i);
#pragma unroll
        for (int i = 0; i < kVerStep / 256; i++)
            q[i] = R.q ? *(const v4f4 *)(R.q + j + 256 * i) : v4f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kVerStep / 256; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) add(p[i][e], q[i][e], j + 256 * i + e);
    }
    for (; j < hi; j += 256)
        for (int e = 0; e < 4 && j + e < hi; e++) add(R.p[j + e], R.q ? R.q[j + e] : 0.0f, j + e);
    sr = wave_sum_d(sr);
    sp = wave_sum_d(sp);
    if (lane == 0) {
        double *o = J.part + ((int64_t)s * J.n_seg + b) * 2;
        o[0] = sr;
        o[1] = sp;
    }
}

// Inclusive sum over the block's threads; *total gets the block's.
__device__ __forceinline__ double block_scan(double v, double *sh, int tid, double *total)
{
    const int lane = tid & 63, w = tid >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) sh[w] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kVerThreads / 64; i++) {
        if (i < w) before += sh[i];
        all += sh[i];
    }
    *total = all;
    return before + v;
}

// The least `first` and the greatest `last` of a block's threads, both rising with the
// thread where they are not INT32_MAX or -1: one atomic of a wave.
__device__ __forceinline__ void least_and_most(int *least, int *most, int first, int last)
{
    const uint64_t a = __ballot(first != INT32_MAX), b = __ballot(last >= 0);
    const int lane = threadIdx.x & 63;
    if (a && lane == __ffsll((unsigned long long)a) - 1) atomicMin(least, first);
    if (b && lane == 63 - __clzll((long long)b)) atomicMax(most, last);
}

__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerJob J)
{
    __shared__ double sh[kVerThreads / 64];
    __shared__ double s_before;
    __shared__ int s_first, s_last;
    const int s = blockIdx.x, tid = threadIdx.x;
    const int n = count_of(J, s);
    const int kept = J.kept[s];
    Row R = row_of(J, s, n, kept);
    // n_seg <= kVerThreads
    const double *o = J.part + ((int64_t)s * J.n_seg + tid) * 2;
    const double pr = tid < J.n_seg ? o[0] : 0.0, pp = tid < J.n_seg ? o[1] : 0.0;
    if (tid == 0) {
        s_first = INT32_MAX;
        s_last = -1;
        s_before = 0.0;
    }
    double total, cum = block_scan(pr, sh, tid, &total);
    double mine = pr;
    if (!(total > 0.0)) {
        // nothing left of p - q: the target's own row
        R.q = nullptr;
        R.less = -1;
        mine = pp;
        cum = block_scan(pp, sh, tid, &total);
    }
    if (!(total > 0.0)) {
        if (tid == 0) J.next[s] = -1;
        return;
    }
    const double want = (double)J.uniform[(int64_t)s * (J.k + 1) + J.k] * total;
    const bool some = tid < J.n_seg && mine > 0.0;
    least_and_most(&s_first, &s_last, some && cum > want ? tid : INT32_MAX, some ? tid : -1);
    __syncthreads();
    const int b = s_first == INT32_MAX ? s_last : s_first;
    if (tid == b) s_before = cum - mine;
    __syncthreads();
    double before = s_before;
    __syncthreads();
    if (tid == 0) {
        s_first = INT32_MAX;
        s_last = -1;
    }
    const int lo = b * J.seg, hi = min(J.vocab, lo + J.seg);
    for (int j0 = lo; j0 < hi; j0 += 4 * kVerThreads) {
        const int j = j0 + 4 * tid;
        double r[4], sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            r[e] = j + e < hi ? R.at(R.p[j + e], R.q ? R.q[j + e] : 0.0f, j + e) : 0.0;
            sum += r[e];
        }
        double all;
        double upto = before + (block_scan(sum, sh, tid, &all) - sum);
        int first = INT32_MAX, last = -1;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            upto += r[e];
            if (r[e] > 0.0) {
                last = j + e;
                if (upto > want && first == INT32_MAX) first = j + e;
            }
        }
        least_and_most(&s_first, &s_last, first, last);
        __syncthreads();
        if (s_first != INT32_MAX) break;
        before += all;
    }
    if (tid == 0) J.next[s] = s_first != INT32_MAX ? s_first : s_last;
}

// Small vocabularies in one launch: a block of 16 waves per sequence, each with a part of
// the row; the wave whose part the number falls in scans it, out of the caches.
__global__ __launch_bounds__(1024) void verify_one_kernel(VerJob J)
{
    __shared__ double sh[2][16];
    const int s = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = count_of(J, s);
    const int kept = kept_of(J, s, n, lane);
    Row R = row_of(J, s, n, kept);
    const int steps = (J.vocab + 16 * 256 - 1) / (16 * 256);     // of a wave, 256 values each
    const int j0 = w * steps * 256 + 4 * lane;
    auto four = [&](const float *x, int j) {
        if (j + 4 <= J.vocab) return *(const v4f4 *)(x + j);
        v4f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int e = 0; e < 4; e++)
            if (j + e < J.vocab) v[e] = x[j + e];
        return v;
    };
    const v4f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    double sr = 0.0, sp = 0.0;
#pragma unroll 4
    for (int i = 0; i < steps; i++) {
        const int j = j0 + 256 * i;
        const v4f4 p = four(R.p, j), q = R.q ? four(R.q, j) : none;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sr += R.at(p[e], q[e], j + e);
            sp += p[e] > 0.0f ? (double)p[e] : 0.0;
        }
    }
    sr = wave_sum_d(sr);
    sp = wave_sum_d(sp);
    if (lane == 0) {
        sh[0][w] = sr;
        sh[1][w] = sp;
    }
    __syncthreads();
    // every wave: the sums before each wave's part, and the part that the number falls in
    auto whole = [&](int k) {
        double t = 0.0;
        for (int i = 0; i < 16; i++) t += sh[k][i];
        return t;
    };
    int k = 0;
    double total = whole(0);
    if (!(total > 0.0)) {
        // nothing left of p - q: the target's own row
        R.q = nullptr;
        R.less = -1;
        k = 1;
        total = whole(1);
    }
    if (threadIdx.x == 0) J.kept[s] = kept;
    if (!(total > 0.0)) {
        if (threadIdx.x == 0) J.next[s] = -1;
        return;
    }
    const double want = (double)J.uniform[(int64_t)s * (J.k + 1) + J.k] * total;
    int b = -1;
    double before = 0.0, cum = 0.0;
    for (int i = 0; i < 16; i++) {
        const double mine = sh[k][i];
        if (mine > 0.0) {
            b = i;
            before = cum;
            if (cum + mine > want) break;
        }
        cum += mine;
    }
    if (w != b) return;
    int first = -1, last = -1;
    for (int i = 0; i < steps && first < 0; i++) {
        const int j = j0 + 256 * i;
        const v4f4 p = four(R.p, j), q = R.q ? four(R.q, j) : none;
        double r[4], sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            r[e] = R.at(p[e], q[e], j + e);
            sum += r[e];
        }
        double v = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double u = __shfl_up(v, o, 64);
            if (lane >= o) v += u;
        }
        double upto = before + (v - sum);
        int f = -1, l = -1;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            upto += r[e];
            if (r[e] > 0.0) {
                l = j + e;
                if (upto > want && f < 0) f = l;
            }
        }
        const uint64_t hit = __ballot(f >= 0), some = __ballot(l >= 0);
        if (some) last = __shfl(l, 63 - __clzll((long long)some), 64);
        if (hit) first = __shfl(f, __ffsll((unsigned long long)hit) - 1, 64);
        before += __shfl(v, 63, 64);
    }
    if (lane == 0) J.next[s] = first >= 0 ? first : last;
}

// One step of a wave, so that the second launch scans a segment in one step; at most
// one segment per thread of that launch.
int seg_of(int vocab)
{
    int64_t seg = kVerStep;
    while ((vocab + seg - 1) / seg > kVerThreads) seg *= 2;
    return (int)seg;
}

}  // namespace

extern "C" size_t eakvd_verify_work_bytes(int n_seqs, int vocab)
{
    const int seg = seg_of(vocab);
    return (size_t)n_seqs * ((vocab + (int64_t)seg - 1) / seg) * 2 * sizeof(double);
}

extern "C" int eakvd_verify(int n_seqs, int k, int vocab, const int32_t *count, const int32_t *token,
                            const float *draft, int64_t ld_draft, const float *target,
                            int64_t ld_target, const float *uniform, int32_t *kept, int32_t *next,
                            void *work, void *stream)
{
    VerJob J;
    J.k = k;
    J.vocab = vocab;
    J.seg = seg_of(vocab);
    J.n_seg = (int)((vocab + (int64_t)J.seg - 1) / J.seg);
    J.count = count;
    J.token = token;
    J.draft = draft;
    J.target = target;
    J.uniform = uniform;
    J.ld_draft = ld_draft;
    J.ld_target = ld_target;
    J.kept = kept;
    J.next = next;
    J.part = (double *)work;
    const hipStream_t st = (hipStream_t)stream;
    if (vocab <= kVerOne) {
        hipLaunchKernelGGL(verify_one_kernel, dim3((unsigned)n_seqs), dim3(1024), 0, st, J);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL(verify_sum_kernel,
                       dim3((unsigned)((J.n_seg + kVerThreads / 64 - 1) / (kVerThreads / 64)), (unsigned)n_seqs),
                       dim3(kVerThreads), 0, st, J);
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)n_seqs), dim3(kVerThreads), 0, st, J);
    return (int)hipGetLastError();
}
