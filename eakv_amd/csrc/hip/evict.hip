// evict.hip — which tokens of a full cache stay: the first and the most recent ones, and of
// the others those of largest score, ties to the lower position; positions ascending, as a
// gather takes them.  score[t] = the heads' weights, summed in f64 and rounded to f32.
//
// Scores become whole numbers in their order (u32); the keep-th largest is found bit by
// bit, then every token knows its place from counts of the tokens before it.  Counts alone are
// shared between blocks: the same list on every call.
//
// Up to kOneMost tokens: one launch, a block to a sequence, the numbers in registers.
// More: blocks of kPart tokens write the numbers and a histogram of their top bits, two more
// launches narrow it down (11, 11 and 10 bits), one counts, the last writes.
#include <string.h>

#include "common.h"

namespace {

constexpr int kOneThreads = 1024;
constexpr int kOneEach = 16;
constexpr int kOneMost = kOneThreads * kOneEach;
constexpr int kPartThreads = 256;
constexpr int kPartEach = 16;
constexpr int kPart = kPartThreads * kPartEach;

struct EvictJob {
    eakvd_evict e;
    const float *weights;
    int64_t ld, ld_kept;
    int32_t *index;
    float *kept;
    int most;               // the longest sequence's tokens
    uint32_t *key;          // [n_seq][most]
    uint32_t *hist;         // [n_seq][3][2048]
    uint32_t *count;        // [n_seq][parts][2]: larger than the threshold, equal to it
    int parts;
};

// Positions in the order of their scores; NaN below everything, the tokens that stay anyway
// above.
__device__ __forceinline__ uint32_t key_of(const EvictJob &J, int s, int t, int n)
{
    if (t < J.e.n_first || t >= n - J.e.n_recent) return 0xffffffffu;
    const float *w = J.weights + (int64_t)s * J.e.n_heads * J.ld + t;
    double sum = 0.0;
    for (int h = 0; h < J.e.n_heads; h++) sum += (double)w[h * J.ld];
    const float x = (float)sum + 0.0f;          // (-0 as 0)
    const uint32_t b = __float_as_uint(x);
    return x != x ? 0u : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

// Token t of sequence s stays, as the rank-th.
__device__ __forceinline__ void put(const EvictJob &J, int s, int t, int rank)
{
    J.index[J.e.first[s] + rank] = t;
    if (J.kept) {
        const float *w = J.weights + (int64_t)s * J.e.n_heads * J.ld + t;
        float *k = J.kept + (int64_t)s * J.e.n_heads * J.ld_kept + rank;
        for (int h = 0; h < J.e.n_heads; h++) k[h * J.ld_kept] = w[h * J.ld];
    }
}

// The kept weights' places behind the last are 0 (tokens to come have no weight yet): thread i
// of n threads.
__device__ __forceinline__ void clear_rest(const EvictJob &J, int s, int i, int n)
{
    if (!J.kept) return;
    for (int h = 0; h < J.e.n_heads; h++) {
        float *k = J.kept + ((int64_t)s * J.e.n_heads + h) * J.ld_kept;
        for (int64_t r = J.e.n_keep[s] + i; r < J.ld_kept; r += n) k[r] = 0.0f;
    }
}

__global__ __launch_bounds__(kOneThreads) void evict_one_kernel(EvictJob J)
{
    __shared__ int sums[2][16][3];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int n = J.e.n_tokens[s], keep = J.e.n_keep[s];
    clear_rest(J, s, tid, kOneThreads);
    if (keep == 0) return;
    // token (w * each + i) * 64 + lane
    const int each = (n + kOneThreads - 1) / kOneThreads;
    const int t0 = w * each * 64 + lane;
    uint32_t key[kOneEach];
#pragma unroll
    for (int i = 0; i < kOneEach; i++) {
        const int t = t0 + 64 * i;
        key[i] = i < each && t < n ? key_of(J, s, t, n) : 0u;
    }
    // the largest threshold that at least `keep` keys reach, two bits at a time.  (Tokens behind
    // the last have key 0, as the lowest have: they count for threshold 0 alone.)
    uint32_t thr = 0;
    int reach = INT32_MAX, it = 0;              // keys that reach thr, where known
    for (int bit = 30; bit >= 0; bit -= 2, it ^= 1) {
        int c[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < kOneEach; i++) {
            if (i < each)
#pragma unroll
                for (int k = 0; k < 3; k++)
                    c[k] += (int)__popcll(__ballot(key[i] >= thr + ((uint32_t)(k + 1) << bit)));
        }
        if (lane < 3) sums[it][w][lane] = lane == 0 ? c[0] : lane == 1 ? c[1] : c[2];
        __syncthreads();
        int all[3] = {0, 0, 0};
        for (int i = 0; i < 16; i++)
#pragma unroll
            for (int k = 0; k < 3; k++) all[k] += sums[it][i][k];
#pragma unroll
        for (int k = 2; k >= 0; k--)
            if (all[k] >= keep) {
                thr += (uint32_t)(k + 1) << bit;
                reach = all[k];
                break;
            }
        if (reach == keep) break;
    }
    // larger than thr: all; equal: the first `ties`
    __syncthreads();
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < kOneEach; i++) {
        const bool in = i < each && t0 + 64 * i < n;
        gt += (int)__popcll(__ballot(in && key[i] > thr));
        eq += (int)__popcll(__ballot(in && key[i] == thr));
    }
    if (lane == 0) {
        sums[0][w][0] = gt;
        sums[0][w][1] = eq;
    }
    __syncthreads();
    int gt_all = 0, gt_before = 0, eq_before = 0;
    for (int i = 0; i < 16; i++) {
        gt_all += sums[0][i][0];
        gt_before += i < w ? sums[0][i][0] : 0;
        eq_before += i < w ? sums[0][i][1] : 0;
    }
    const int ties = keep - gt_all;
#pragma unroll
    for (int i = 0; i < kOneEach; i++) {
        const int t = t0 + 64 * i;
        const bool in = i < each && t < n;
        const uint64_t below = (1ull << lane) - 1;
        const uint64_t g = __ballot(in && key[i] > thr), e = __ballot(in && key[i] == thr);
        const int eq_at = eq_before + (int)__popcll(e & below);
        const bool mine = (g >> lane & 1) || ((e >> lane & 1) && eq_at < ties);
        if (mine) put(J, s, t, gt_before + (int)__popcll(g & below) + min(eq_at, ties));
        gt_before += (int)__popcll(g);
        eq_before += (int)__popcll(e);
    }
}

__global__ __launch_bounds__(256) void evict_clear_kernel(uint32_t *p, int n)
{
    const int i = (int)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

// The digit that the keep-th largest key has, of `bins` (a multiple of kPartThreads): hist[d] keys have
// digit d; *above gets the keys with larger ones.  All threads of the block.
__device__ __forceinline__ int digit_of(const uint32_t *hist, int bins, int keep, int *above, int *sh, int tid)
{
    const int lane = tid & 63, w = tid >> 6, per = bins / kPartThreads;
    // thread 0 has the largest digits
    int sum = 0;
    for (int i = 0; i < per; i++) sum += (int)hist[bins - 1 - (tid * per + i)];
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(upto, o, 64);
        if (lane >= o) upto += u;
    }
    __syncthreads();
    if (lane == 63) sh[w] = upto;
    __syncthreads();
    int before = upto - sum;
    for (int i = 0; i < w; i++) before += sh[i];
    if (before < keep && keep <= before + sum)
        for (int i = 0; i < per; i++) {
            const int d = bins - 1 - (tid * per + i), c = (int)hist[d];
            if (keep <= before + c) {
                sh[4] = d;
                sh[5] = before;
                break;
            }
            before += c;
        }
    __syncthreads();
    *above = sh[5];
    const int d = sh[4];
    __syncthreads();
    return d;
}

// What is known of the threshold after `level` histograms: its top bits, and how many keys
// with them stay.
struct Known {
    uint32_t top;
    int keep;
};
__device__ __forceinline__ Known known(const EvictJob &J, int s, int level, int *sh, int tid)
{
    Known k = {0, J.e.n_keep[s]};
    for (int l = 0; l < level; l++) {
        int above;
        const int bins = l < 2 ? 2048 : 1024;
        const int d = digit_of(J.hist + ((int64_t)s * 3 + l) * 2048, bins, k.keep, &above, sh, tid);
        k.top = k.top * (uint32_t)bins + (uint32_t)d;
        k.keep -= above;
    }
    return k;
}

// LEVEL 0: keys and the histogram of their top 11 bits; 1, 2: that of the next 11 and 10 bits
// of the keys that have the bits known; 3: the part's keys above and at the threshold.
template <int LEVEL>
__global__ __launch_bounds__(kPartThreads) void evict_part_kernel(EvictJob J)
{
    __shared__ uint32_t bins[2048];
    __shared__ int sh[8];
    const int s = blockIdx.y, tid = threadIdx.x, t0 = (int)blockIdx.x * kPart;
    const int n = J.e.n_tokens[s];
    if (t0 >= n || J.e.n_keep[s] == 0) return;
    const Known k = known(J, s, LEVEL, sh, tid);
    uint32_t *keys = J.key + (int64_t)s * J.most;
    if constexpr (LEVEL < 3) {
        for (int i = tid; i < 2048; i += kPartThreads) bins[i] = 0;
        __syncthreads();
    }
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < kPartEach; i++) {
        const int t = t0 + i * kPartThreads + tid;
        if (t >= n) break;
        uint32_t x;
        if constexpr (LEVEL == 0) {
            x = key_of(J, s, t, n);
            keys[t] = x;
        } else {
            x = keys[t];
        }
        if constexpr (LEVEL == 0) atomicAdd(&bins[x >> 21], 1u);
        if constexpr (LEVEL == 1) {
            if (x >> 21 == k.top) atomicAdd(&bins[x >> 10 & 2047], 1u);
        }
        if constexpr (LEVEL == 2) {
            if (x >> 10 == k.top) atomicAdd(&bins[x & 1023], 1u);
        }
        if constexpr (LEVEL == 3) {
            gt += x > k.top;
            eq += x == k.top;
        }
    }
    __syncthreads();
    if constexpr (LEVEL < 3) {
        uint32_t *h = J.hist + ((int64_t)s * 3 + LEVEL) * 2048;
        for (int i = tid; i < 2048; i += kPartThreads)
            if (bins[i]) atomicAdd(h + i, bins[i]);
    } else {
        if (tid < 2) sh[tid] = 0;
        __syncthreads();
        atomicAdd(&sh[0], gt);
        atomicAdd(&sh[1], eq);
        __syncthreads();
        if (tid < 2) J.count[((int64_t)s * J.parts + blockIdx.x) * 2 + tid] = (uint32_t)sh[tid];
    }
}

__global__ __launch_bounds__(kPartThreads) void evict_write_kernel(EvictJob J)
{
    __shared__ int sh[8], sums[2][kPartThreads / 64][2];
    const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, t0 = (int)blockIdx.x * kPart;
    const int n = J.e.n_tokens[s];
    clear_rest(J, s, (int)blockIdx.x * kPartThreads + tid, (int)gridDim.x * kPartThreads);
    if (t0 >= n || J.e.n_keep[s] == 0) return;
    const Known k = known(J, s, 3, sh, tid);
    // (k.keep of the keys at the threshold stay)
    if (tid < 2) sh[tid] = 0;
    __syncthreads();
    {
        int g = 0, e = 0;
        for (int p = tid; p < (int)blockIdx.x; p += kPartThreads) {
            const uint32_t *c = J.count + ((int64_t)s * J.parts + p) * 2;
            g += (int)c[0];
            e += (int)c[1];
        }
        if (g) atomicAdd(&sh[0], g);
        if (e) atomicAdd(&sh[1], e);
    }
    __syncthreads();
    int gt_before = sh[0], eq_before = sh[1];
    const uint32_t *keys = J.key + (int64_t)s * J.most;
    const uint64_t below = (1ull << lane) - 1;
    for (int i = 0; i < kPartEach; i++) {
        const int t = t0 + i * kPartThreads + tid;
        const uint32_t x = t < n ? keys[t] : 0;
        const uint64_t g = __ballot(t < n && x > k.top), e = __ballot(t < n && x == k.top);
        if (lane == 0) {
            sums[i & 1][w][0] = (int)__popcll(g);
            sums[i & 1][w][1] = (int)__popcll(e);
        }
        __syncthreads();
        int g_at = gt_before + (int)__popcll(g & below), e_at = eq_before + (int)__popcll(e & below);
#pragma unroll
        for (int j = 0; j < kPartThreads / 64; j++) {
            const int a = sums[i & 1][j][0], b = sums[i & 1][j][1];
            g_at += j < w ? a : 0;
            e_at += j < w ? b : 0;
            gt_before += a;
            eq_before += b;
        }
        if ((g >> lane & 1) || ((e >> lane & 1) && e_at < k.keep)) put(J, s, t, g_at + min(e_at, k.keep));
    }
}

int most_of(int n_seq, const int32_t *n)
{
    int most = 0;
    for (int i = 0; i < n_seq; i++) most = n[i] > most ? n[i] : most;
    return most;
}

}  // namespace

extern "C" size_t eakvd_evict_work_bytes(int n_seq, const int32_t *n_tokens)
{
    const int most = most_of(n_seq, n_tokens);
    if (most <= kOneMost) return 0;
    const size_t parts = ((size_t)most + kPart - 1) / kPart;
    return (size_t)n_seq * ((size_t)most + 3 * 2048 + 2 * parts) * 4;
}

extern "C" int eakvd_evict_select(const eakvd_evict *job, const float *weights, int64_t ld, int32_t *index,
                                  float *kept, int64_t ld_kept, void *work, void *stream)
{
    EvictJob J;
    memset(&J, 0, sizeof(J));
    J.e = *job;
    J.weights = weights;
    J.ld = ld;
    J.ld_kept = ld_kept;
    J.index = index;
    J.kept = kept;
    J.most = most_of(job->n_seq, job->n_tokens);
    const hipStream_t st = (hipStream_t)stream;
    const unsigned n = (unsigned)job->n_seq;
    if (J.most <= kOneMost) {
        hipLaunchKernelGGL(evict_one_kernel, dim3(n), dim3(kOneThreads), 0, st, J);
        return (int)hipGetLastError();
    }
    J.parts = (J.most + kPart - 1) / kPart;
    J.hist = (uint32_t *)work;
    J.count = J.hist + (size_t)n * 3 * 2048;
    J.key = J.count + (size_t)n * J.parts * 2;
    const int zero = (int)n * 3 * 2048;
    const dim3 grid((unsigned)J.parts, n), nt(kPartThreads);
    hipLaunchKernelGGL(evict_clear_kernel, dim3((unsigned)(zero + 255) / 256), dim3(256), 0, st, J.hist, zero);
    hipLaunchKernelGGL(evict_part_kernel<0>, grid, nt, 0, st, J);
    hipLaunchKernelGGL(evict_part_kernel<1>, grid, nt, 0, st, J);
    hipLaunchKernelGGL(evict_part_kernel<2>, grid, nt, 0, st, J);
    hipLaunchKernelGGL(evict_part_kernel<3>, grid, nt, 0, st, J);
    hipLaunchKernelGGL(evict_write_kernel, grid, nt, 0, st, J);
    return (int)hipGetLastError();
}
