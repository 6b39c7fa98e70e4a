// move.hip — tokens of a cache moved between and within caches, planes as they
// stand: a range into several caches (copy) and a list of tokens into another
// cache or to the front of the same one (gather).  Every byte of a token is read once
// and written once (copy: once per destination); copies and gathers to another cache are
// bound by HBM, gathers in place by the passes of a row, which wait for one another.
//
// A row is one kv head of one (layer, kv) block: its tokens' packed bytes, scales
// and biases, each contiguous.  A block of the copy moves 1024 groups of a row (40 KB),
// all its loads in flight before the first store: 32768 tokens of 4 layers x 8 heads,
// d = 128, into 4 caches take 159 us (839 MB, 5.3 TB/s, what a large copy reaches).
#include "common.h"

namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveGroups = 1024;                               // of one block's pass
constexpr int kMoveW = kMoveGroups * 2 / kMoveThreads;          // 16-byte pieces of a thread
constexpr int kMoveS = kMoveGroups / kMoveThreads;              // scales (and biases)

struct CopyJob {
    const uint8_t *src;
    uint8_t *dst[EAKVD_MAX_BATCH];
    int n_dst;
    int64_t src_pos, dst_pos, n_tokens;
};

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kMoveThreads) void copy_kernel(eakvd_geom gs, eakvd_geom gd, CopyJob job,
                                                            int n_rows)
{
    const int64_t n = job.n_tokens * gs.gpd;
    const int64_t g0 = (int64_t)blockIdx.x * kMoveGroups;
    const int cnt = (int)(n - g0 < kMoveGroups ? n - g0 : kMoveGroups);
    const int tid = threadIdx.x;
    for (int row = blockIdx.y; row < n_rows; row += gridDim.y) {
        const int blk = row / gs.n_kv_heads, hd = row - blk * gs.n_kv_heads;
        const uint8_t *sb = job.src + (int64_t)blk * gs.block_bytes;
        const int64_t si = hd * gs.gph + job.src_pos * gs.gpd + g0;
        const v4u *sw = (const v4u *)(sb + si * 32);
        const float *ss = (const float *)(sb + gs.s_off) + si;
        const float *sc = (const float *)(sb + gs.b_off) + si;
        v4u x[kMoveW];
        float a[kMoveS], b[kMoveS];
#pragma unroll
        for (int k = 0; k < kMoveW; k++) {
            const int i = tid + k * kMoveThreads;
            if (i < 2 * cnt) x[k] = __builtin_nontemporal_load(sw + i);
        }
#pragma unroll
        for (int k = 0; k < kMoveS; k++) {
            const int i = tid + k * kMoveThreads;
            if (i < cnt) {
                a[k] = __builtin_nontemporal_load(ss + i);
                b[k] = __builtin_nontemporal_load(sc + i);
            }
        }
        const int64_t di = hd * gd.gph + job.dst_pos * gd.gpd + g0;
        for (int d = 0; d < job.n_dst; d++) {
            uint8_t *db = job.dst[d] + (int64_t)blk * gd.block_bytes;
            v4u *dw = (v4u *)(db + di * 32);
            float *ds = (float *)(db + gd.s_off) + di;
            float *dc = (float *)(db + gd.b_off) + di;
#pragma unroll
            for (int k = 0; k < kMoveW; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < 2 * cnt) __builtin_nontemporal_store(x[k], dw + i);
            }
#pragma unroll
            for (int k = 0; k < kMoveS; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < cnt) {
                    __builtin_nontemporal_store(a[k], ds + i);
                    __builtin_nontemporal_store(b[k], dc + i);
                }
            }
        }
    }
}

// dst token dst_pos + i = src token index[i].  Into another cache the passes of
// a row are separate blocks.  In place (SERIAL) one block takes a row's passes
// in order: with index ascending and index[i] >= dst_pos + i, the tokens that a
// pass writes lie before every token that a later pass reads, and within a pass
// all loads are done (the barrier) before the first store.  Positions are
// clamped to the cache's room (in place: from dst_pos + i on), so that any list
// stays within the planes.
//
// 13001 of 30011 tokens, 8 layers of 8 heads, d = 128: 80 us a call in a row of them
// (3.35 TB/s of 266 MB; contiguous tokens 66 us): tokens of 64 packed bytes fill half of
// a 128-byte line, and a list that skips tokens fetches lines for one of the two.
// Passes of 256 groups against 1024: 80 against 86 us; with loads past the caches,
// 83 and 93; with stores through them, 93 and more.  In place the passes wait for one
// another, and the longer ones are kept: one block to a row, 107 us for 16384 tokens of
// 32768 at one layer of 8 heads (16 blocks; 42 MB), 207 to 270 at 8 layers; a pair in
// place takes the call's other pairs along.
template <bool SERIAL>
constexpr int kGatherGroups = SERIAL ? kMoveGroups : 256;

template <int GPD, bool SERIAL>
__global__ __launch_bounds__(kMoveThreads) void gather_kernel(eakvd_geom gs, eakvd_geom gd,
                                                              eakvd_gather job, int rows_per,
                                                              int n_rows)
{
    constexpr int G = kGatherGroups<SERIAL>, T = G / GPD;        // groups, tokens of a pass
    constexpr int W = G * 2 / kMoveThreads, S = G / kMoveThreads;
    const int tid = threadIdx.x;
    for (int row = blockIdx.y; row < n_rows; row += gridDim.y) {
        const int c = row / rows_per, r = row - c * rows_per;
        const int blk = r / gs.n_kv_heads, hd = r - blk * gs.n_kv_heads;
        const uint8_t *sb = job.src[c] + (int64_t)blk * gs.block_bytes;
        uint8_t *db = job.dst[c] + (int64_t)blk * gd.block_bytes;
        const int64_t s0 = hd * gs.gph, d0 = hd * gd.gph + (int64_t)job.dst_pos[c] * GPD;
        const int32_t *index = job.index + job.first[c];
        const int n = job.n_tokens[c], top = gs.max_seq_len - 1;
        const bool same = job.src[c] == job.dst[c];
        for (int t0 = (int)blockIdx.x * T; t0 < n; t0 += (int)gridDim.x * T) {
            const int cnt = (n - t0 < T ? n - t0 : T) * GPD;      // groups
            auto from = [&](int g) {
                const int i = t0 + g / GPD;
                const int low = same ? job.dst_pos[c] + i : 0;
                int t = index[i];
                t = t < low ? low : t > top ? top : t;
                return s0 + (int64_t)t * GPD + g % GPD;
            };
            v4u x[W];
            float a[S], b[S];
#pragma unroll
            for (int k = 0; k < W; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < 2 * cnt)
                    x[k] = ((const v4u *)(sb + from(i >> 1) * 32))[i & 1];
            }
#pragma unroll
            for (int k = 0; k < S; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < cnt) {
                    const int64_t g = from(i);
                    a[k] = ((const float *)(sb + gs.s_off))[g];
                    b[k] = ((const float *)(sb + gs.b_off))[g];
                }
            }
            if constexpr (SERIAL) {
                // every load of this pass is in registers before any store
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
            const int64_t d = d0 + (int64_t)t0 * GPD;
            v4u *dw = (v4u *)(db + d * 32);
            float *ds = (float *)(db + gd.s_off) + d;
            float *dc = (float *)(db + gd.b_off) + d;
#pragma unroll
            for (int k = 0; k < W; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < 2 * cnt) __builtin_nontemporal_store(x[k], dw + i);
            }
#pragma unroll
            for (int k = 0; k < S; k++) {
                const int i = tid + k * kMoveThreads;
                if (i < cnt) {
                    __builtin_nontemporal_store(a[k], ds + i);
                    __builtin_nontemporal_store(b[k], dc + i);
                }
            }
        }
    }
}

unsigned grid_y(int64_t rows) { return (unsigned)(rows < 65535 ? rows : 65535); }

}  // namespace

extern "C" int eakvd_copy_tokens(const eakvd_geom *gs, const eakvd_geom *gd, const uint8_t *src,
                                 int src_pos, uint8_t *const *dst, int n_dst, int dst_pos,
                                 int n_tokens, void *stream)
{
    if (n_tokens <= 0 || n_dst <= 0) return 0;
    CopyJob job{};
    job.src = src;
    job.n_dst = n_dst;
    for (int i = 0; i < n_dst; i++) job.dst[i] = dst[i];
    job.src_pos = src_pos;
    job.dst_pos = dst_pos;
    job.n_tokens = n_tokens;
    const int64_t rows = (int64_t)2 * gs->n_layers * gs->n_kv_heads;
    if (rows > INT32_MAX) return (int)hipErrorInvalidValue;
    const int64_t n = (int64_t)n_tokens * gs->gpd;
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)((n + kMoveGroups - 1) / kMoveGroups), grid_y(rows)),
                       dim3(kMoveThreads), 0, (hipStream_t)stream, *gs, *gd, job, (int)rows);
    return (int)hipGetLastError();
}

extern "C" int eakvd_gather_tokens(const eakvd_geom *gs, const eakvd_geom *gd,
                                   const eakvd_gather *job, void *stream)
{
    int most = 0;
    bool serial = false;
    for (int i = 0; i < job->n_seq; i++) {
        most = job->n_tokens[i] > most ? job->n_tokens[i] : most;
        serial = serial || job->src[i] == job->dst[i];
    }
    if (most <= 0) return 0;
    const int per = 2 * gs->n_layers * gs->n_kv_heads;
    const int64_t rows = (int64_t)per * job->n_seq;
    if (rows > INT32_MAX) return (int)hipErrorInvalidValue;
    const int t = kGatherGroups<false> / (int)gs->gpd;
    const dim3 grid(serial ? 1u : (unsigned)((most + t - 1) / t), grid_y(rows));
    auto *kern = gs->gpd == 2 ? (serial ? gather_kernel<2, true> : gather_kernel<2, false>)
                              : (serial ? gather_kernel<1, true> : gather_kernel<1, false>);
    hipLaunchKernelGGL(kern, grid, dim3(kMoveThreads), 0, (hipStream_t)stream, *gs, *gd, *job, per,
                       (int)rows);
    return (int)hipGetLastError();
}
