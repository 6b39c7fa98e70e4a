// weights.hip — the attention weight that each cached token gets from a window's queries,
// summed over the queries and the q heads of a kv head and added to what it had:
//
//   w[h][t] = keep * w[h][t] + sum_{i, q heads of h} exp(s_i[t] - M_i) / L_i,
//   s_i[t] = q_i.K[t] / sqrt(d) where query i sees t, M_i = max_t s_i, L_i = sum_t exp(s_i - M_i).
//
// The scores are made on the matrix cores (rows16.h; the arithmetic of window.hip, K's operands
// exact for both types).  A first pass over K leaves each row's (M, L) of a chunk of tokens.
// Few rows (up to kStore to a kv head, a decode step): it also leaves the scores, and the
// second launch adds their weights up: 8 bytes a row and token more against K's 80, and no
// products.  More: the second pass makes the scores again, with tokens across the lanes so that
// rows add up in a lane's registers.  Rows (window tokens x q heads) are taken several row tiles
// at a time, their operands in LDS; a wave holds 32 tokens' operands of K in registers and goes
// through the rows.  The first pass gives groups of row tiles to blocks of their own; the
// second, which sums over all rows, has them one after the other.  A token's sum is one
// thread's or one wave's: no atomics, the same bits on every call.
//
// Few rows are bound by memory (one f32 token x 8 at 32768, 32 q / 8 kv: 65 us; K and the scores
// both ways at a copy's 5.17 TB/s 49); many by instructions issued (32 bf16 tokens x 4 to 20011, 64 q /
// 8 kv: 85-97 us, the passes alike; vector ALUs 72 % and all kinds 93 to 96 % of the cycles,
// matrix cores 29 to 35 %; 90 and 73 vector instructions for 16 rows x 32 tokens).
#include <string.h>

#include "rows16.h"

namespace {

constexpr int kTile = 256;
constexpr int kRowTiles = 8;                    // of a block of the first pass, at most
constexpr int kSumTiles = 16;                   // of a pass over a chunk's tokens in the second
constexpr int kStore = 8;

struct WeightsJob {
    int n_seq, n_q, n_kv, qpk, layer;
    const uint8_t *base[EAKVD_MAX_BATCH];
    int start[EAKVD_MAX_BATCH], ntok[EAKVD_MAX_BATCH], tok0[EAKVD_MAX_BATCH];
    int seq[EAKVD_MAX_BATCH];                   // its number in the call
    int mc[EAKVD_MAX_BATCH];                    // chunks of the first pass
    int clen[2][EAKVD_MAX_BATCH];               // a chunk's tokens, either pass
    int pre[2][EAKVD_MAX_BATCH + 1];            // blocks before this sequence's
    int add[EAKVD_MAX_BATCH + 1];               // weights_add_kernel: likewise
    int64_t stat[EAKVD_MAX_BATCH];              // its rows' first (M, L)
    int64_t score[EAKVD_MAX_BATCH], ld_s[EAKVD_MAX_BATCH];      // its scores, and from row to row
};

// LDS: the waves' scales, a Tile for each row tile of a pass, then (first pass) the waves' running
// M and L, a lane's each, [tile][wave][64].
struct Scales {
    float ks[2][32], zk[2][32];
};
template <int D, bool F32>
struct __align__(16) Tile {
    static constexpr int NQ = D / 32 * (F32 ? 2 : 1) + 1;       // operands
    uint4 q[NQ][64];
    float rf[16];
    int vis[16];                                // positions that the row sees
    int all, pad[3];                            // that all of them see
    float off[16];                              // second pass: M + log2 L
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, int64_t bytes)
{
    // dword3 0x00020000: raw 32-bit buffer; reads beyond `bytes` return 0
    const int64_t most = 0xfffffff0ll;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0,
                                             (int)(uint32_t)(bytes < most ? bytes : most), 0x00020000);
}

// The chunks' (M, L) of a row joined, 4 lanes to a row (sub): M + log2 L, whose power is taken off a
// score's: one exponential is the weight.  (Its rounding is half a step of M's, which M's own has
// as well; the logarithm is off by 2 steps at most.)
// (Eight loads in flight: a chunk at a time this was most of a small launch.)
__device__ __forceinline__ float join_row(const float2 *st, int mc, int sub, bool live)
{
    float mm = kMInit, l = 0.0f;
    for (int k0 = sub; live && k0 < mc; k0 += 32) {
        float2 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = st[min(k0 + 4 * k, mc - 1)];
        float top = mm;
#pragma unroll
        for (int k = 0; k < 8; k++) top = x[k].y != 0.0f ? fmaxf(top, x[k].x) : top;
        l *= __builtin_amdgcn_exp2f(mm - top);
#pragma unroll
        for (int k = 0; k < 8; k++)
            l = k0 + 4 * k < mc && x[k].y != 0.0f ? fmaf(__builtin_amdgcn_exp2f(x[k].x - top), x[k].y, l) : l;
        mm = top;
    }
    float top = fmaxf(mm, __shfl_xor(mm, 1, 64));
    top = fmaxf(top, __shfl_xor(top, 2, 64));
    l *= __builtin_amdgcn_exp2f(mm - top);
    l += __shfl_xor(l, 1, 64);
    l += __shfl_xor(l, 2, 64);
    return top + __builtin_amdgcn_logf(l);
}

// A row tile's operands from LDS; the bias's is the result.
template <int D, bool F32>
__device__ __forceinline__ b8 load_query(const uint4 (*q)[64], int lane, Query<D, F32, false> &Q)
{
#pragma unroll
    for (int f = 0; f < D / 32; f++) {
        Q.a[f] = __builtin_bit_cast(h8, q[f][lane]);
        if constexpr (F32) Q.b[F32 ? f : 0] = __builtin_bit_cast(h8, q[D / 32 + (F32 ? f : 0)][lane]);
    }
    return __builtin_bit_cast(b8, q[D / 32 * (F32 ? 2 : 1)][lane]);
}

// group_dots with tokens across: a lane has one token's of four rows.
template <int D, bool F32>
__device__ __forceinline__ v4f row_dots(const h8 &lo, const h8 &hi, const Query<D, F32, false> &Q, int g)
{
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (F32) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(Q.b[F32 ? 2 * g : 0], lo, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(Q.b[F32 ? 2 * g + 1 : 0], hi, acc, 0, 0, 0);
    }
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(Q.a[2 * g], lo, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(Q.a[2 * g + 1], hi, acc, 0, 0, 0);
}

// W waves.  SUM: the second pass; STORE: the first pass leaves the scores, log2, [kv head][row][ld_s].
template <int D, bool F32, int W, bool SUM, bool STORE>
__global__ __launch_bounds__(64 * W, W == 4 ? 3 : W == 8 && F32 ? 2 : 4) void weights_kernel(
    eakvd_geom geo, WeightsJob job, const void *q, float2 *stat, float *score, float *out, int64_t ld,
    float keep, float ksc, int vec, int tiles)
{
    constexpr int GPD = D / 64, RB = 32 * GPD;
    typedef Tile<D, F32> Tl;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    Scales &S = ((Scales *)lds)[w];
    Tl *T = (Tl *)(lds + W * sizeof(Scales));
    float2 (*run)[W][64] = (float2 (*)[W][64])(T + tiles);
    const int n16 = lane & 15, blk = lane >> 4, n32 = lane & 31, h = lane >> 5;
    const bool owner = GPD == 2 || h == 0;
    const int gh = GPD == 2 ? h : 0;

    const int c = seq_of(job.pre[SUM], job.n_seq, (int)blockIdx.x, lane);
    const int rem = (int)blockIdx.x - job.pre[SUM][c];
    const int m = job.ntok[c], start = job.start[c], qpk = job.qpk, mc = job.mc[c], clen = job.clen[SUM][c];
    const int kvh = rem % job.n_kv;
    const int chunk = SUM ? rem / job.n_kv : rem / job.n_kv % mc;
    // the block's rows: tiles of them in the first pass, all in the second
    const int row0 = SUM ? 0 : rem / job.n_kv / mc * 16 * tiles;
    const int rows = m * qpk, row1 = SUM ? rows : min(rows, row0 + 16 * tiles), t_end = start + m;
    const int lo = chunk * clen;
    const int hi = t_end - lo > clen ? lo + clen : t_end;
    const int n_sub = hi > lo ? (hi - lo + 31) / 32 : 0;
    const int n_i = n_sub > w ? (n_sub - w + W - 1) / W : 0;
    float2 *st = stat + job.stat[c] + (int64_t)kvh * rows * mc;          // [row][chunk]

    // (offsets from the chunk's first token are 32 bits; behind the plane's end loads give 0)
    const Planes K = planes_of(geo, job.base[c], job.layer, 0);
    const int64_t g0 = (int64_t)kvh * geo.gph + (int64_t)lo * GPD;
    const int64_t room = (int64_t)(geo.max_seq_len - lo) * GPD;
    const auto rk = rsrc(K.w + g0 * 32, room * 32), rks = rsrc(K.s + g0, room * 4), rkb = rsrc(K.b + g0, room * 4);
    NibConst nc;
    nc.hold();

    for (int r0 = row0; r0 < row1; r0 += 16 * tiles) {
        const int nu = min(tiles, (rows - r0 + 15) / 16);
        __syncthreads();
        for (int u = w; u < nu; u += W) {
            const int at = r0 + 16 * u + n16, row = min(at, rows - 1), tok = row / qpk;
            Query<D, F32, false> Q;
            Q.load(q, ((int64_t)(job.tok0[c] + tok) * job.n_q + kvh * qpk + row - tok * qpk) * D, vec, blk);
#pragma unroll
            for (int f = 0; f < D / 32; f++) {
                T[u].q[f][lane] = __builtin_bit_cast(uint4, Q.a[f]);
                if constexpr (F32) T[u].q[D / 32 + (F32 ? f : 0)][lane] = __builtin_bit_cast(uint4, Q.b[F32 ? f : 0]);
            }
            T[u].q[Tl::NQ - 1][lane] = __builtin_bit_cast(uint4, Q.bias);
            if (blk == 0) {
                T[u].rf[n16] = Q.rf;
                T[u].vis[n16] = at < rows ? start + tok + 1 : 0;
                if (n16 == 0) T[u].all = r0 + 16 * u + 15 < rows ? start + tok + 1 : 0;
            }
            if constexpr (!SUM)
                for (int k = 0; k < W; k++) run[u][k][lane] = float2{kMInit, 0.0f};
        }
        if constexpr (SUM)
            for (int r = tid >> 2; r < 16 * nu; r += 16 * W) {
                const float x = join_row(st + (int64_t)(r0 + r) * mc, mc, tid & 3, r0 + r < rows);
                if ((tid & 3) == 0) T[r >> 4].off[r & 15] = x;
            }
        __syncthreads();

        uint2 kx[2][GPD];
        float s0 = 0.0f, b0 = 0.0f;
        auto load = [&](int i) __attribute__((always_inline)) {
            const int t = 32 * (w + W * i);
            constexpr int aux = W == 4 && !SUM ? 2 : 0;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int g = 0; g < GPD; g++) {
                    const auto y = __builtin_amdgcn_raw_buffer_load_b64(rk, n16 * RB + 8 * blk, (t + 16 * k) * RB + 32 * g,
                                                                        aux);
                    kx[k][g] = uint2{y[0], y[1]};
                }
            const int at = (n32 * GPD + gh) * 4;
            s0 = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rks, at, t * GPD * 4, aux));
            b0 = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rkb, at, t * GPD * 4, aux));
        };
        if (n_i > 0) load(0);
        for (int i = 0; i < n_i; i++) {
            const int t0 = lo + 32 * (w + W * i);
            const float zk = zero_nibble(s0, b0), ck = fmaf(zk, s0, b0) * ksc;
            if (owner) {
                S.ks[gh][n32] = s0 * ksc;
                S.zk[gh][n32] = zk;
            }
            b8 bias[2];
            bias_operands(owner ? ck : 0.0f, 0.0f, false, bias, n32);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            h8 kl[2][GPD], kh[2][GPD];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int g = 0; g < GPD; g++)
                    k_operands<false>(kx[k][g], S.zk[g][16 * k + n16], nc, kl[k][g], kh[k][g]);
            if (i + 1 < n_i) load(i + 1);
            if constexpr (SUM) {
                // a lane: token n16 of each half, rows 4 blk to 4 blk + 3, so that the rows add up in
                // its own registers
                float acc[2] = {0.0f, 0.0f}, ks[2][GPD];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int g = 0; g < GPD; g++) ks[k][g] = S.ks[g][16 * k + n16];
#pragma unroll 1
                for (int u = 0; u < nu; u++) {
                    Query<D, F32, false> Q;
                    const b8 qb = load_query<D, F32>(T[u].q, lane, Q);
                    const v4f rf = *(const v4f *)&T[u].rf[4 * blk], off = *(const v4f *)&T[u].off[4 * blk];
                    float y[2][4];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        v4f s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qb, bias[k], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                        for (int g = 0; g < GPD; g++) {
                            const v4f dot = row_dots(kl[k][g], kh[k][g], Q, g);
#pragma unroll
                            for (int e = 0; e < 4; e++) s[e] = fmaf(ks[k][g], dot[e], s[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) y[k][e] = __builtin_amdgcn_exp2f(fmaf(s[e], rf[e], -off[e]));
                    }
                    if (t0 + 32 > T[u].all) {
                        const int4 vis = *(const int4 *)&T[u].vis[4 * blk];
                        const int seen[4] = {vis.x, vis.y, vis.z, vis.w};
#pragma unroll
                        for (int k = 0; k < 2; k++)
#pragma unroll
                            for (int e = 0; e < 4; e++) y[k][e] = t0 + 16 * k + n16 < seen[e] ? y[k][e] : 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) acc[k] += (y[k][0] + y[k][1]) + (y[k][2] + y[k][3]);
                }
                // over the lanes of one token: one half's sums to lanes 0-15, the other's to 16-31
                float v = row_sum(acc[0]);
                const float v1 = row_sum(acc[1]);
                v = blk == 1 ? v1 : v;
                const int t = t0 + n32;
                if (h == 0 && t < hi) {
                    float *o = out + ((int64_t)job.seq[c] * job.n_kv + kvh) * ld + t;
                    const float by = r0 == 0 ? keep : 1.0f;
                    *o = by == 0.0f ? v : fmaf(by, *o, v);
                }
            } else {
                v4f sc[2][GPD];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int g = 0; g < GPD; g++) sc[k][g] = *(const v4f *)&S.ks[g][16 * k + 4 * blk];
#pragma unroll 1
                for (int u = 0; u < nu; u++) {
                    Query<D, F32, false> Q;
                    const b8 qb = load_query<D, F32>(T[u].q, lane, Q);
                    const float rf = T[u].rf[n16];
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        v4f s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias[k], qb, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                        for (int g = 0; g < GPD; g++) {
                            const v4f dot = group_dots(kl[k][g], kh[k][g], Q, g);
#pragma unroll
                            for (int e = 0; e < 4; e++) s[e] = fmaf(sc[k][g][e], dot[e], s[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) x[4 * k + e] = s[e];
                    }
                    if (t0 + 32 > T[u].all) {
                        const int seen = T[u].vis[n16] - t0 - 4 * blk;          // of the lane's first half on
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            x[j] = 16 * (j >> 2) + (j & 3) < seen ? x[j] : -__builtin_inff();
                    }
                    if constexpr (STORE) {
                        if (r0 + 16 * u + n16 < rows) {
                            float *o = score + job.score[c] + ((int64_t)kvh * rows + r0 + 16 * u + n16) * job.ld_s[c] + t0 +
                                       4 * blk;
                            *(v4f *)o = v4f{x[0] * rf, x[1] * rf, x[2] * rf, x[3] * rf};
                            *(v4f *)(o + 16) = v4f{x[4] * rf, x[5] * rf, x[6] * rf, x[7] * rf};
                        }
                    }
                    const float2 old = run[u][w][lane];
                    const float top = max3(max3(max3(x[0], x[1], x[2]), x[3], x[4]), max3(x[5], x[6], x[7]), x[7]);
                    const float mn = fmaxf(old.x, top * rf);
                    float l = old.y * __builtin_amdgcn_exp2f(old.x - mn);
#pragma unroll
                    for (int j = 0; j < 8; j++) l += __builtin_amdgcn_exp2f(fmaf(x[j], rf, -mn));
                    run[u][w][lane] = float2{mn, l};
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if constexpr (!SUM) {
            // rows' (M, L) of the chunk: over the lanes of a row and the waves
            __syncthreads();
            for (int r = tid >> 2; r < 16 * nu; r += 16 * W) {
                const int row = r0 + r;
                float mm = kMInit;
                for (int k = 0; k < W; k++) mm = fmaxf(mm, run[r >> 4][k][(r & 15) + 16 * (tid & 3)].x);
                mm = fmaxf(mm, __shfl_xor(mm, 1, 64));
                mm = fmaxf(mm, __shfl_xor(mm, 2, 64));
                float l = 0.0f;
                for (int k = 0; k < W; k++) {
                    const float2 x = run[r >> 4][k][(r & 15) + 16 * (tid & 3)];
                    l = x.y == 0.0f ? l : fmaf(__builtin_amdgcn_exp2f(x.x - mm), x.y, l);
                }
                l += __shfl_xor(l, 1, 64);
                l += __shfl_xor(l, 2, 64);
                if ((tid & 3) == 0 && row < rows) st[(int64_t)row * mc + chunk] = float2{mm, l};
            }
        }
    }
}

// The scores that the first pass left, as weights: 4 tokens to a thread, the unit's rows one
// after the other.
constexpr int kAddThreads = 256;
__global__ __launch_bounds__(kAddThreads) void weights_add_kernel(WeightsJob job, const float2 *stat,
                                                                  const float *score, float *out, int64_t ld,
                                                                  float keep)
{
    __shared__ float off[kStore];
    const int tid = threadIdx.x, lane = tid & 63;
    const int c = seq_of(job.add, job.n_seq, (int)blockIdx.x, lane);
    const int rem = (int)blockIdx.x - job.add[c];
    const int kvh = rem % job.n_kv, t0 = (rem / job.n_kv) * 4 * kAddThreads + 4 * tid;
    const int rows = job.ntok[c] * job.qpk, mc = job.mc[c], hi = job.start[c] + job.ntok[c];
    if (tid < 4 * kStore) {
        const int r = tid >> 2;
        const float x = join_row(stat + job.stat[c] + ((int64_t)kvh * rows + min(r, rows - 1)) * mc, mc, tid & 3,
                                 r < rows);
        if ((tid & 3) == 0) off[r] = x;
    }
    __syncthreads();
    if (t0 >= hi) return;
    // (rows of scores are whole tiles; those that a row does not see are -inf, and what is
    // there has no part in the sum where the row's is NaN)
    const float *s = score + job.score[c] + (int64_t)kvh * rows * job.ld_s[c] + t0;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = 0; r < rows; r++) {
        const v4f x = __builtin_nontemporal_load((const v4f *)(s + (int64_t)r * job.ld_s[c]));
        const float y = off[r];
        const int vis = job.start[c] + r / job.qpk + 1;
#pragma unroll
        for (int e = 0; e < 4; e++)
            acc[e] += t0 + e < vis ? __builtin_amdgcn_exp2f(x[e] - y) : 0.0f;
    }
    float *o = out + ((int64_t)job.seq[c] * job.n_kv + kvh) * ld + t0;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (t0 + e < hi) o[e] = keep == 0.0f ? acc[e] : fmaf(keep, o[e], acc[e]);
}

struct WeightsPlan {
    WeightsJob job;
    int waves, tiles[2];
    bool store;
    size_t stat_bytes, bytes;
};

// Chunks of an even share of the tiles: 3 blocks of 4 waves to a CU for up to two row tiles.  More:
// blocks of 8 waves and up to kRowTiles row tiles in the first pass (bf16: two to a CU); in
// the second one of 16 waves, all rows after one another.
void weights_plan(const eakvd_window *b, int n_q, int n_kv, bool bf16, WeightsPlan *p)
{
    memset(p, 0, sizeof(*p));
    WeightsJob &j = p->job;
    j.n_q = n_q;
    j.n_kv = n_kv;
    j.qpk = n_q / n_kv;
    int64_t tiles[2] = {0, 0}, stat = 0, score = 0, rows = 0;
    int tok0 = 0;
    for (int i = 0; i < b->n_seq; i++) {
        if (b->ntok[i]) {
            const int k = j.n_seq++;
            j.base[k] = b->base[i];
            j.start[k] = b->start[i];
            j.ntok[k] = b->ntok[i];
            j.tok0[k] = tok0;
            j.seq[k] = i;
            const int64_t r = (int64_t)b->ntok[i] * j.qpk;
            rows = r > rows ? r : rows;
        }
        tok0 += b->ntok[i];
    }
    const int64_t row_tiles = (rows + 15) / 16;
    p->store = rows <= kStore;
    p->tiles[0] = (int)(row_tiles < kRowTiles ? row_tiles : kRowTiles);
    p->tiles[1] = (int)(row_tiles < kSumTiles ? row_tiles : kSumTiles);
    p->waves = row_tiles <= 2 ? 4 : 8;
    const auto groups = [&](int i) { return ((int64_t)j.ntok[i] * j.qpk + 16 * p->tiles[0] - 1) / (16 * p->tiles[0]); };
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t n = ((int64_t)j.start[i] + j.ntok[i] + kTile - 1) / kTile * n_kv;
        tiles[0] += n * groups(i);
        tiles[1] += n;
    }
    for (int pass = 0; pass < 2; pass++) {
        const int64_t slots = (p->waves == 4 ? 3 : bf16 && pass == 0 ? 2 : 1) * cu_count();
        const int64_t share = (tiles[pass] + slots - 1) / slots;
        for (int i = 0; i < j.n_seq; i++) {
            const int64_t t = (int64_t)j.start[i] + j.ntok[i], n_t = (t + kTile - 1) / kTile;
            int64_t mc = (n_t + share - 1) / share;
            // (offsets from a chunk's first token are 32 bits)
            if (mc < (n_t >> 16) + 1) mc = (n_t >> 16) + 1;
            const int64_t per = (n_t + mc - 1) / mc;
            mc = (n_t + per - 1) / per;
            j.clen[pass][i] = (int)(per * kTile);
            j.pre[pass][i + 1] = j.pre[pass][i] + (int)(mc * n_kv * (pass ? 1 : groups(i)));
            if (pass) continue;
            j.mc[i] = (int)mc;
            j.add[i + 1] = j.add[i] + (int)((t + 4 * kAddThreads - 1) / (4 * kAddThreads)) * n_kv;
            j.stat[i] = stat;
            stat += (int64_t)j.ntok[i] * n_q * mc;
            j.ld_s[i] = n_t * kTile;
            j.score[i] = score;
            score += (int64_t)j.ntok[i] * n_q * j.ld_s[i];
        }
    }
    p->stat_bytes = ((size_t)stat * sizeof(float2) + 255) & ~(size_t)255;
    p->bytes = p->stat_bytes + (p->store ? (size_t)score * sizeof(float) : 0);
}

template <int D, bool F32, int W, bool SUM, bool STORE>
int pass(const eakvd_geom &g, const WeightsPlan &p, const void *q, void *work, float *out, int64_t ld,
         float keep, int vec, hipStream_t st)
{
    constexpr size_t tile = sizeof(Tile<D, F32>) + (SUM ? 0 : W * 64 * sizeof(float2));
    constexpr int most = W == 4 ? 2 : SUM ? kSumTiles : kRowTiles;
    static_assert(W * sizeof(Scales) + most * tile <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> done;
    auto *kern = weights_kernel<D, F32, W, SUM, STORE>;
    const int e = allow_lds((const void *)kern, W * sizeof(Scales) + most * tile, done);
    if (e) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.job.pre[SUM][p.job.n_seq]), dim3(64 * W),
                       W * sizeof(Scales) + p.tiles[SUM] * tile, st, g, p.job, q, (float2 *)work,
                       (float *)((uint8_t *)work + p.stat_bytes), out, ld, keep, EAKV_LOG2E / sqrtf((float)D), vec,
                       p.tiles[SUM]);
    return (int)hipGetLastError();
}

template <int D, bool F32>
int launch(const eakvd_geom &g, const WeightsPlan &p, const void *q, void *work, float *out, int64_t ld,
           float keep, int vec, hipStream_t st)
{
    int e;
    if (p.store) {
        e = pass<D, F32, 4, false, true>(g, p, q, work, out, ld, keep, vec, st);
        if (e) return e;
        hipLaunchKernelGGL(weights_add_kernel, dim3((unsigned)p.job.add[p.job.n_seq]), dim3(kAddThreads), 0, st, p.job,
                           (float2 *)work, (float *)((uint8_t *)work + p.stat_bytes), out, ld, keep);
        return (int)hipGetLastError();
    }
    if (p.waves == 4) {
        e = pass<D, F32, 4, false, false>(g, p, q, work, out, ld, keep, vec, st);
        return e ? e : pass<D, F32, 4, true, false>(g, p, q, work, out, ld, keep, vec, st);
    }
    e = pass<D, F32, 8, false, false>(g, p, q, work, out, ld, keep, vec, st);
    return e ? e : pass<D, F32, 16, true, false>(g, p, q, work, out, ld, keep, vec, st);
}

}  // namespace

extern "C" size_t eakvd_weights_work_bytes(const eakvd_window *b, int n_q, int n_kv, int bf16)
{
    WeightsPlan p;
    weights_plan(b, n_q, n_kv, bf16, &p);
    return p.bytes;
}

extern "C" int eakvd_weights(const eakvd_geom *g, const eakvd_window *b, int layer, const void *q, int bf16,
                             int n_q, int n_kv, float keep, float *out, int64_t ld, void *work, void *stream)
{
    WeightsPlan p;
    weights_plan(b, n_q, n_kv, bf16, &p);
    if (p.job.n_seq == 0) return 0;
    p.job.layer = layer;
    const hipStream_t st = (hipStream_t)stream;
    const int vec = (uintptr_t)q % 16 == 0;
    if (g->head_dim == 64)
        return bf16 ? launch<64, false>(*g, p, q, work, out, ld, keep, vec, st)
                    : launch<64, true>(*g, p, q, work, out, ld, keep, vec, st);
    return bf16 ? launch<128, false>(*g, p, q, work, out, ld, keep, vec, st)
                : launch<128, true>(*g, p, q, work, out, ld, keep, vec, st);
}
