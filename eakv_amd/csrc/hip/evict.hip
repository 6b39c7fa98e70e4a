// evict.hip — which tokens of a full cache stay: the first and the most recent ones, and of
// the others those of largest score, ties to the lower position; positions ascending, as a
// gather takes them.  score[t] = the heads' weights, summed in f64 and rounded to f32.
//
// Scores become whole numbers in their order (u32); the keep-th largest is found by
// histograms of 8 to 11 of its bits at a time, then every token knows its place from counts of
// the tokens before it.  Counts alone are shared between blocks: the same list on every call.
//
// Up to kOneMost tokens: one launch, a block to a sequence, the numbers in registers, four
// histograms of 8 bits in LDS.  (2048 of 2100 x 8 sequences, 8 heads: 10.3 us, latency of a chain of
// barriers.  Many heads are one CU's to read: 256 of 8192 tokens 215 us, more than 8193 tokens' 67.)
// More: blocks of kPart tokens write the numbers and a histogram of their top bits, two more
// launches narrow it down (11, 11 and 10 bits), one counts, the last writes; each leaves what is
// known of the threshold to the next.  (20000 of 131072 x 2, 8 heads: 26 us, six launches of 2 to 8;
// of 500000: 32.6.)
#include <string.h>

#include "common.h"

namespace {

constexpr int kOneThreads = 1024;
constexpr int kOneMost = kOneThreads * 8;
constexpr int kPartThreads = 256;
constexpr int kPartEach = 8;
constexpr int kPart = kPartThreads * kPartEach;

struct Known {
    uint32_t top;
    int keep;
};

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
    Known *known;           // [n_seq][3]: what 1, 2 and 3 histograms say
    int parts;
};

// Scores in their order: NaN below everything, the tokens that stay anyway above.
__device__ __forceinline__ uint32_t key_of(const EvictJob &J, int t, int n, double sum)
{
    if (t < J.e.n_first || t >= n - J.e.n_recent) return 0xffffffffu;
    const float x = (float)sum + 0.0f;          // (-0 as 0)
    const uint32_t b = __float_as_uint(x);
    return x != x ? 0u : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

// Keys of E tokens `step` apart from t0 on (0 from `end` on) of a sequence of n: heads H at a time,
// all their loads in flight.  A head's sum is in its order, whatever H.  x: the last H heads' weights.
template <int E>
constexpr int kHeadsOf = E > 8 ? 2 : 32 / E > 8 ? 8 : 32 / E;
template <int E>
__device__ __forceinline__ void load_heads(const EvictJob &J, int s, int t0, int step, int n, int h0,
                                           float (&x)[E][kHeadsOf<E>])
{
    const float *w = J.weights + (int64_t)s * J.e.n_heads * J.ld;
#pragma unroll
    for (int h = 0; h < kHeadsOf<E>; h++)
#pragma unroll
        for (int i = 0; i < E; i++)
            x[i][h] = w[(int64_t)min(h0 + h, J.e.n_heads - 1) * J.ld + min(t0 + i * step, n - 1)];
}
template <int E>
__device__ __forceinline__ void keys_of(const EvictJob &J, int s, int t0, int step, int end, int n, uint32_t *key,
                                        float (&x)[E][kHeadsOf<E>])
{
    constexpr int H = kHeadsOf<E>;
    double sum[E];
#pragma unroll
    for (int i = 0; i < E; i++) sum[i] = 0.0;
    for (int h0 = 0; h0 < J.e.n_heads; h0 += H) {
        load_heads<E>(J, s, t0, step, n, h0, x);
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int i = 0; i < E; i++)
                if (h0 + h < J.e.n_heads) sum[i] += (double)x[i][h];
    }
#pragma unroll
    for (int i = 0; i < E; i++) key[i] = t0 + i * step < end ? key_of(J, t0 + i * step, n, sum[i]) : 0u;
}

// Tokens t0 + i * step of sequence s stay, as the rank[i]-th (-1: do not): x holds their weights of
// the first kHeadsOf heads (have), the others' are read, all tokens' loads of some heads in flight.
template <int E>
__device__ __forceinline__ void put_all(const EvictJob &J, int s, int t0, int step, int n, const int *rank,
                                        float (&x)[E][kHeadsOf<E>], bool have)
{
    constexpr int H = kHeadsOf<E>;
    int32_t *index = J.index + J.e.first[s];
#pragma unroll
    for (int i = 0; i < E; i++)
        if (rank[i] >= 0) index[rank[i]] = t0 + i * step;
    if (!J.kept) return;
    float *k = J.kept + (int64_t)s * J.e.n_heads * J.ld_kept;
    for (int h0 = 0; h0 < J.e.n_heads; h0 += H) {
        if (h0 > 0 || !have) load_heads<E>(J, s, t0, step, n, h0, x);
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int i = 0; i < E; i++)
                if (rank[i] >= 0 && h0 + h < J.e.n_heads) k[(h0 + h) * J.ld_kept + rank[i]] = x[i][h];
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

// The sum of the lanes 4 apart: two rotations in a row of 16, two exchanges between rows.
__device__ __forceinline__ int over_waves(int v)
{
    v += __builtin_amdgcn_mov_dpp(v, 0x124, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = (int)(r[0] + r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (int)(r[0] + r[1]);
}

template <int E>
__global__ __launch_bounds__(kOneThreads) void evict_one_kernel(EvictJob J)
{
    __shared__ int sums[64];                    // [wave][4]
    __shared__ __align__(16) uint32_t hist[4][1024];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int n = J.e.n_tokens[s], keep = J.e.n_keep[s];
    clear_rest(J, s, tid, kOneThreads);
    if (keep == 0) return;
    // token (w * each + i) * 64 + lane
    const int each = (n + kOneThreads - 1) / kOneThreads;
    const int t0 = w * each * 64 + lane;
    uint32_t key[E];
    float x[E][kHeadsOf<E>];
    *(uint4 *)&hist[tid >> 8][(tid & 255) * 4] = uint4{0, 0, 0, 0};
    __syncthreads();
    keys_of<E>(J, s, t0, 64, min(n, (w + 1) * each * 64), n, key, x);
    // the keep-th largest key, 8 bits at a time: a histogram in LDS (four copies, as neighbouring lanes
    // often meet in one bin), which every wave searches for itself
    uint32_t thr = 0;
    int ties = keep;                            // of the keys that have the bits known
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int shift = 24 - 8 * p;
#pragma unroll
        for (int i = 0; i < E; i++)
            if (i < each && t0 + 64 * i < n && (p == 0 || key[i] >> (32 - 8 * p) == thr))
                atomicAdd(&hist[p][(key[i] >> shift & 255) * 4 + (lane & 3)], 1u);
        __syncthreads();
        // lane l: digits 255 - 4 l down to 252 - 4 l
        int c[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint4 x = *(const uint4 *)&hist[p][(255 - 4 * lane - k) * 4];
            c[k] = (int)(x.x + x.y + x.z + x.w);
            sum += c[k];
        }
        const int upto = wave_scan_i(sum);
        const int at = __ffsll((unsigned long long)__ballot(upto >= ties)) - 1;
        int before = __builtin_amdgcn_readlane(upto - sum, at), d = 255 - 4 * at;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int n_k = __builtin_amdgcn_readlane(c[k], at);
            if (d == 255 - 4 * at - k && before + n_k < ties) {
                before += n_k;
                d--;
            }
        }
        ties -= before;
        thr = thr << 8 | (uint32_t)d;
    }
    // larger than thr: all; equal: the first `ties`
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const bool in = i < each && t0 + 64 * i < n;
        gt += (int)__popcll(__builtin_amdgcn_ballot_w64(in && key[i] > thr));
        eq += (int)__popcll(__builtin_amdgcn_ballot_w64(in && key[i] == thr));
    }
    if (lane < 2) sums[4 * w + lane] = lane ? eq : gt;
    __syncthreads();
    const int mine4 = sums[lane];
    const int before = over_waves(lane >> 2 < w ? mine4 : 0);
    int gt_before = __builtin_amdgcn_readlane(before, 0), eq_before = __builtin_amdgcn_readlane(before, 1);
    int rank[E];
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int t = t0 + 64 * i;
        const bool in = i < each && t < n;
        const uint64_t below = (1ull << lane) - 1;
        const uint64_t g = __builtin_amdgcn_ballot_w64(in && key[i] > thr),
                       e = __builtin_amdgcn_ballot_w64(in && key[i] == thr);
        const int eq_at = eq_before + (int)__popcll(e & below);
        const bool mine = (g >> lane & 1) || ((e >> lane & 1) && eq_at < ties);
        rank[i] = mine ? gt_before + (int)__popcll(g & below) + min(eq_at, ties) : -1;
        gt_before += (int)__popcll(g);
        eq_before += (int)__popcll(e);
    }
    put_all<E>(J, s, t0, 64, n, rank, x, J.e.n_heads <= kHeadsOf<E>);
}

__global__ __launch_bounds__(256) void evict_clear_kernel(uint32_t *p, int n)
{
    const int i = (int)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

// The digit that the keep-th largest key has, of BINS: hist[d] keys have
// digit d; *above gets the keys with larger ones.  All threads of the block.
template <int BINS>
__device__ __forceinline__ int digit_of(const uint32_t *hist, int keep, int *above, int *sh, int tid)
{
    constexpr int per = BINS / kPartThreads;
    const int lane = tid & 63, w = tid >> 6;
    // thread 0 has the largest digits
    int c[BINS / kPartThreads], sum = 0;
#pragma unroll
    for (int i = 0; i < per; i++) c[i] = (int)hist[BINS - 1 - (tid * per + i)];
#pragma unroll
    for (int i = 0; i < per; i++) sum += c[i];
    const int upto = wave_scan_i(sum);
    __syncthreads();
    if (lane == 63) sh[w] = upto;
    __syncthreads();
    int before = upto - sum;
    for (int i = 0; i < w; i++) before += sh[i];
    if (before < keep && keep <= before + sum)
#pragma unroll
        for (int i = 0; i < per; i++) {
            if (before < keep && keep <= before + c[i]) {
                sh[4] = BINS - 1 - (tid * per + i);
                sh[5] = before;
            }
            before += c[i];
        }
    __syncthreads();
    *above = sh[5];
    const int d = sh[4];
    __syncthreads();
    return d;
}

// What is known of the threshold after LEVEL histograms: its top bits, and how many keys
// with them stay.  The launch before left it after LEVEL - 1 of them.
template <int LEVEL>
__device__ __forceinline__ Known known(const EvictJob &J, int s, int *sh, int tid)
{
    if constexpr (LEVEL == 0) return Known{0, J.e.n_keep[s]};
    Known k = LEVEL == 1 ? Known{0, J.e.n_keep[s]} : J.known[3 * s + LEVEL - 2];
    int above;
    const uint32_t *hist = J.hist + ((int64_t)s * 3 + LEVEL - 1) * 2048;
    const int d = LEVEL < 3 ? digit_of<2048>(hist, k.keep, &above, sh, tid) : digit_of<1024>(hist, k.keep, &above, sh, tid);
    k.top = k.top * (LEVEL < 3 ? 2048u : 1024u) + (uint32_t)d;
    k.keep -= above;
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
    uint32_t *keys = J.key + (int64_t)s * J.most, key[kPartEach];
    if constexpr (LEVEL > 0)
#pragma unroll
        for (int i = 0; i < kPartEach; i++) key[i] = keys[min(t0 + i * kPartThreads + tid, n - 1)];
    const Known k = known<LEVEL>(J, s, sh, tid);
    if (LEVEL > 0 && blockIdx.x == 0 && tid == 0) J.known[3 * s + LEVEL - 1] = k;
    if constexpr (LEVEL < 3) {
        for (int i = tid; i < 2048; i += kPartThreads) bins[i] = 0;
        __syncthreads();
    }
    int gt = 0, eq = 0;
    if constexpr (LEVEL == 0) {
        float x[kPartEach][kHeadsOf<kPartEach>];
        keys_of<kPartEach>(J, s, t0 + tid, kPartThreads, n, n, key, x);
    }
#pragma unroll
    for (int i = 0; i < kPartEach; i++) {
        const int t = t0 + i * kPartThreads + tid;
        if (t >= n) continue;
        const uint32_t x = key[i];
        if constexpr (LEVEL == 0) keys[t] = x;
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
    __shared__ int before[kPartThreads / 64][2], sums[kPartEach][kPartThreads / 64][2];
    const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, t0 = (int)blockIdx.x * kPart;
    const int n = J.e.n_tokens[s];
    clear_rest(J, s, (int)blockIdx.x * kPartThreads + tid, (int)gridDim.x * kPartThreads);
    if (t0 >= n || J.e.n_keep[s] == 0) return;
    const uint32_t *keys = J.key + (int64_t)s * J.most;
    uint32_t key[kPartEach];
#pragma unroll
    for (int i = 0; i < kPartEach; i++) key[i] = keys[min(t0 + i * kPartThreads + tid, n - 1)];
    const Known k = J.known[3 * s + 2];         // (k.keep of the keys at the threshold stay)
    int g0 = 0, e0 = 0;                         // of the parts before
    for (int p = tid; p < (int)blockIdx.x; p += kPartThreads) {
        const uint32_t *c = J.count + ((int64_t)s * J.parts + p) * 2;
        g0 += (int)c[0];
        e0 += (int)c[1];
    }
    float w4[kPartEach][kHeadsOf<kPartEach>];
    if (J.kept) load_heads<kPartEach>(J, s, t0 + tid, kPartThreads, n, 0, w4);
    g0 = __builtin_amdgcn_readlane(wave_scan_i(g0), 63);
    e0 = __builtin_amdgcn_readlane(wave_scan_i(e0), 63);
    if (lane == 0) before[w][0] = g0, before[w][1] = e0;
    const uint64_t below = (1ull << lane) - 1;
    uint64_t gs[kPartEach], es[kPartEach];
#pragma unroll
    for (int i = 0; i < kPartEach; i++) {
        const int t = t0 + i * kPartThreads + tid;
        gs[i] = __builtin_amdgcn_ballot_w64(t < n && key[i] > k.top);
        es[i] = __builtin_amdgcn_ballot_w64(t < n && key[i] == k.top);
        if (lane == 0) {
            sums[i][w][0] = (int)__popcll(gs[i]);
            sums[i][w][1] = (int)__popcll(es[i]);
        }
    }
    __syncthreads();
    int gt_before = 0, eq_before = 0;
#pragma unroll
    for (int j = 0; j < kPartThreads / 64; j++) {
        gt_before += before[j][0];
        eq_before += before[j][1];
    }
    int rank[kPartEach];
#pragma unroll
    for (int i = 0; i < kPartEach; i++) {
        int g_at = gt_before + (int)__popcll(gs[i] & below), e_at = eq_before + (int)__popcll(es[i] & below);
#pragma unroll
        for (int j = 0; j < kPartThreads / 64; j++) {
            const int a = sums[i][j][0], b = sums[i][j][1];
            g_at += j < w ? a : 0;
            e_at += j < w ? b : 0;
            gt_before += a;
            eq_before += b;
        }
        rank[i] = (gs[i] >> lane & 1) || ((es[i] >> lane & 1) && e_at < k.keep) ? g_at + min(e_at, k.keep) : -1;
    }
    put_all<kPartEach>(J, s, t0 + tid, kPartThreads, n, rank, w4, true);
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
    return (size_t)n_seq * ((size_t)most + 3 * 2048 + 3 * 2 + 2 * parts) * 4;
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
        auto *kern = J.most <= 4 * kOneThreads ? evict_one_kernel<4> : evict_one_kernel<8>;
        hipLaunchKernelGGL(kern, dim3(n), dim3(kOneThreads), 0, st, J);
        return (int)hipGetLastError();
    }
    J.parts = (J.most + kPart - 1) / kPart;
    J.hist = (uint32_t *)work;
    J.known = (Known *)(J.hist + (size_t)n * 3 * 2048);
    J.count = (uint32_t *)(J.known + (size_t)n * 3);
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
