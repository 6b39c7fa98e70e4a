// weights.hip — the attention weight that each cached token gets from a window's queries,
// summed over the queries and the q heads of a kv head and added to what it had:
//
//   w[h][t] = keep * w[h][t] + sum_{i, q heads of h} exp(s_i[t] - M_i) / L_i,
//   s_i[t] = q_i.K[t] / sqrt(d) where query i sees t, M_i = max_t s_i, L_i = sum_t exp(s_i - M_i).
//
// Two passes over K, the scores made on the matrix cores in both (rows16.h; the arithmetic
// of window.hip): the first leaves each row's (M, L) of a chunk of tokens, the second joins
// them and sums the weights.  Rows (window tokens x q heads) are taken 128 at a time, their
// operands in LDS; a wave holds 32 tokens' operands of K in registers and goes through the
// rows.  A token's sum is one wave's: no atomics, the same bits on every call.
#include <string.h>

#include "rows16.h"

namespace {

constexpr int kWaves = 8;
constexpr int kTile = 32 * kWaves;
constexpr int kRowTiles = 8;                    // of a pass over a chunk's tokens
constexpr int kGroupRows = 16 * kRowTiles;

struct WeightsJob {
    int n_seq, n_q, n_kv, qpk, layer;
    const uint8_t *base[EAKVD_MAX_BATCH];
    int start[EAKVD_MAX_BATCH], ntok[EAKVD_MAX_BATCH], tok0[EAKVD_MAX_BATCH];
    int seq[EAKVD_MAX_BATCH];                   // its number in the call
    int mc[EAKVD_MAX_BATCH], clen[EAKVD_MAX_BATCH];
    int pre[EAKVD_MAX_BATCH + 1];               // blocks before this sequence's
    int64_t stat[EAKVD_MAX_BATCH];              // its rows' first (M, L)
};

template <int D, bool F32>
struct __align__(16) WLds {
    static constexpr int NQ = D / 32 * (F32 ? 2 : 1) + 1;       // operands of a row tile
    uint4 q[kRowTiles][NQ][64];
    float rf[kRowTiles][16];
    float2 ml[kRowTiles][16];                   // second pass: M and 1/L of the rows
    struct {
        float ks[D / 64][32], zk[D / 64][32];
    } w[kWaves];
    float2 run[kWaves][kRowTiles][64];          // first pass: a lane's running M and L
};

// SUM: the second pass.
template <int D, bool F32, bool SUM>
__global__ __launch_bounds__(64 * kWaves, 2) void weights_kernel(eakvd_geom geo, WeightsJob job,
                                                                 const void *q, float2 *stat, float *out,
                                                                 int64_t ld, float keep, float ksc, int vec)
{
    constexpr int GPD = D / 64, RB = 32 * GPD;
    typedef WLds<D, F32> Lds;
    extern __shared__ __align__(16) uint8_t lds[];
    Lds &S = *(Lds *)lds;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, blk = lane >> 4, n32 = lane & 31, h = lane >> 5;
    const bool owner = GPD == 2 || h == 0;
    const int gh = GPD == 2 ? h : 0;

    const int c = seq_of(job.pre, job.n_seq, (int)blockIdx.x, lane);
    const int rem = (int)blockIdx.x - job.pre[c];
    const int kvh = rem % job.n_kv, chunk = rem / job.n_kv;
    const int m = job.ntok[c], start = job.start[c], qpk = job.qpk, mc = job.mc[c];
    const int rows = m * qpk, t_end = start + m;
    const int lo = chunk * job.clen[c];
    const int hi = t_end - lo > job.clen[c] ? lo + job.clen[c] : t_end;
    const int n_sub = hi > lo ? (hi - lo + 31) / 32 : 0;
    const int n_i = n_sub > w ? (n_sub - w + kWaves - 1) / kWaves : 0;
    float2 *st = stat + job.stat[c] + (int64_t)kvh * rows * mc;          // [row][chunk]

    const Planes K = planes_of(geo, job.base[c], job.layer, 0);
    const int64_t g0 = (int64_t)kvh * geo.gph + (int64_t)lo * GPD;
    const uint8_t *kw = K.w + g0 * 32;
    const float *ks = K.s + g0, *kb = K.b + g0;
    const int last = hi - 1 - lo;                               // the chunk's last token
    NibConst nc;
    nc.hold();

    for (int r0 = 0; r0 < rows; r0 += kGroupRows) {
        const int nu = min(kRowTiles, (rows - r0 + 15) / 16);
        __syncthreads();
        if (w < nu) {
            const int row = min(r0 + 16 * w + n16, rows - 1), tok = row / qpk;
            Query<D, F32, false> Q;
            Q.load(q, ((int64_t)(job.tok0[c] + tok) * job.n_q + kvh * qpk + row - tok * qpk) * D, vec, blk);
#pragma unroll
            for (int f = 0; f < D / 32; f++) {
                S.q[w][f][lane] = __builtin_bit_cast(uint4, Q.a[f]);
                if constexpr (F32) S.q[w][D / 32 + (F32 ? f : 0)][lane] = __builtin_bit_cast(uint4, Q.b[F32 ? f : 0]);
            }
            S.q[w][Lds::NQ - 1][lane] = __builtin_bit_cast(uint4, Q.bias);
            if (blk == 0) S.rf[w][n16] = Q.rf;
        }
        if constexpr (SUM) {
            // the chunks' (M, L) of a row, 4 lanes to each of 128 rows
            const int r = tid >> 2, row = r0 + r;
            float mm = kMInit;
            if (row < rows)
                for (int k = tid & 3; k < mc; k += 4) {
                    const float2 x = st[(int64_t)row * mc + k];
                    if (x.y != 0.0f) mm = fmaxf(mm, x.x);
                }
            mm = fmaxf(mm, __shfl_xor(mm, 1, 64));
            mm = fmaxf(mm, __shfl_xor(mm, 2, 64));
            float l = 0.0f;
            if (row < rows)
                for (int k = tid & 3; k < mc; k += 4) {
                    const float2 x = st[(int64_t)row * mc + k];
                    if (x.y != 0.0f) l = fmaf(__builtin_amdgcn_exp2f(x.x - mm), x.y, l);
                }
            l += __shfl_xor(l, 1, 64);
            l += __shfl_xor(l, 2, 64);
            if ((tid & 3) == 0) S.ml[r >> 4][r & 15] = float2{mm, l == 0.0f ? 0.0f : 1.0f / l};
        } else {
            for (int u = 0; u < nu; u++) S.run[w][u][lane] = float2{kMInit, 0.0f};
        }
        __syncthreads();

        uint2 kx[2][GPD];
        float s0 = 0.0f, b0 = 0.0f;
        auto load = [&](int i) {
            const int t = 32 * (w + kWaves * i);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int g = 0; g < GPD; g++)
                    kx[k][g] = *(const uint2 *)(kw + (int64_t)min(t + 16 * k + n16, last) * RB + 32 * g + 8 * blk);
            const int64_t gi = (int64_t)min(t + n32, last) * GPD + gh;
            s0 = ks[gi];
            b0 = kb[gi];
        };
        if (n_i > 0) load(0);
        for (int i = 0; i < n_i; i++) {
            const int t0 = lo + 32 * (w + kWaves * i);
            const float zk = zero_nibble(s0, b0), ck = fmaf(zk, s0, b0) * ksc;
            if (owner) {
                S.w[w].ks[gh][n32] = s0 * ksc;
                S.w[w].zk[gh][n32] = zk;
            }
            b8 bias[2];
            bias_operands(owner ? ck : 0.0f, 0.0f, false, bias, n32);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            h8 kl[2][GPD], kh[2][GPD];
            v4f sc[2][GPD];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int g = 0; g < GPD; g++) {
                    k_operands<false>(kx[k][g], S.w[w].zk[g][16 * k + n16], nc, kl[k][g], kh[k][g]);
                    sc[k][g] = *(const v4f *)&S.w[w].ks[g][16 * k + 4 * blk];
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (i + 1 < n_i) load(i + 1);
            float acc[8];
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] = 0.0f;
#pragma unroll 1
            for (int u = 0; u < nu; u++) {
                Query<D, F32, false> Q;
#pragma unroll
                for (int f = 0; f < D / 32; f++) {
                    Q.a[f] = __builtin_bit_cast(h8, S.q[u][f][lane]);
                    if constexpr (F32) Q.b[F32 ? f : 0] = __builtin_bit_cast(h8, S.q[u][D / 32 + (F32 ? f : 0)][lane]);
                }
                const b8 qb = __builtin_bit_cast(b8, S.q[u][Lds::NQ - 1][lane]);
                const float rf = S.rf[u][n16];
                const int row = r0 + 16 * u + n16;
                // positions that the row sees (rows behind the last: none)
                const int vis = row < rows ? start + row / qpk + 1 : 0;
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
                const bool masked = __ballot(t0 + 32 > vis) != 0;
                const int seen = vis - t0 - 4 * blk;            // of the lane's first half on
                if constexpr (SUM) {
                    const float2 ml = S.ml[u][n16];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float y = __builtin_amdgcn_exp2f(fmaf(x[j], rf, -ml.x)) * ml.y;
                        acc[j] += !masked || 16 * (j >> 2) + (j & 3) < seen ? y : 0.0f;
                    }
                } else {
                    if (masked)
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            x[j] = 16 * (j >> 2) + (j & 3) < seen ? x[j] : -__builtin_inff();
                    float2 run = S.run[w][u][lane];
                    float top = fmaxf(x[0], x[1]);
#pragma unroll
                    for (int j = 2; j < 8; j++) top = fmaxf(top, x[j]);
                    const float mn = fmaxf(run.x, top * rf);
                    float l = run.y * __builtin_amdgcn_exp2f(run.x - mn);
#pragma unroll
                    for (int j = 0; j < 8; j++) l += __builtin_amdgcn_exp2f(fmaf(x[j], rf, -mn));
                    S.run[w][u][lane] = float2{mn, l};
                }
            }
            if constexpr (SUM) {
                // over the 16 rows of the tile: lanes with one blk
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    acc[j] += dpp_f<0x128>(acc[j]);             // row_ror 8, 4, 2, 1
                    acc[j] += dpp_f<0x124>(acc[j]);
                    acc[j] += dpp_f<0x122>(acc[j]);
                    acc[j] += dpp_f<0x121>(acc[j]);
                }
                float v = acc[0];
#pragma unroll
                for (int j = 1; j < 8; j++) v = n16 == j ? acc[j] : v;
                const int t = t0 + 16 * ((n16 >> 2) & 1) + 4 * blk + (n16 & 3);
                if (n16 < 8 && t < hi) {
                    float *o = out + ((int64_t)job.seq[c] * job.n_kv + kvh) * ld + t;
                    const float by = r0 == 0 ? keep : 1.0f;
                    *o = by == 0.0f ? v : fmaf(by, *o, v);
                }
            }
        }
        if constexpr (!SUM) {
            // rows' (M, L) of the chunk: over the lanes of a row and the waves
            __syncthreads();
            const int r = tid >> 2, row = r0 + r;
            float mm = kMInit;
            for (int k = 0; k < kWaves; k++) mm = fmaxf(mm, S.run[k][r >> 4][(r & 15) + 16 * (tid & 3)].x);
            mm = fmaxf(mm, __shfl_xor(mm, 1, 64));
            mm = fmaxf(mm, __shfl_xor(mm, 2, 64));
            float l = 0.0f;
            for (int k = 0; k < kWaves; k++) {
                const float2 x = S.run[k][r >> 4][(r & 15) + 16 * (tid & 3)];
                l = x.y == 0.0f ? l : fmaf(__builtin_amdgcn_exp2f(x.x - mm), x.y, l);
            }
            l += __shfl_xor(l, 1, 64);
            l += __shfl_xor(l, 2, 64);
            if ((tid & 3) == 0 && row < rows) st[(int64_t)row * mc + chunk] = float2{mm, l};
        }
    }
}

struct WeightsPlan {
    WeightsJob job;
    size_t bytes;
};

// Chunks of an even share of the tiles for two blocks per CU.
void weights_plan(const eakvd_window *b, int n_q, int n_kv, WeightsPlan *p)
{
    memset(p, 0, sizeof(*p));
    WeightsJob &j = p->job;
    j.n_q = n_q;
    j.n_kv = n_kv;
    j.qpk = n_q / n_kv;
    int64_t tiles = 0, stat = 0;
    int tok0 = 0;
    for (int i = 0; i < b->n_seq; i++) {
        if (b->ntok[i]) {
            const int k = j.n_seq++;
            j.base[k] = b->base[i];
            j.start[k] = b->start[i];
            j.ntok[k] = b->ntok[i];
            j.tok0[k] = tok0;
            j.seq[k] = i;
            tiles += ((int64_t)b->start[i] + b->ntok[i] + kTile - 1) / kTile * n_kv;
        }
        tok0 += b->ntok[i];
    }
    const int64_t slots = 2 * cu_count(), share = (tiles + slots - 1) / slots;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t n_t = ((int64_t)j.start[i] + j.ntok[i] + kTile - 1) / kTile;
        int64_t mc = (n_t + share - 1) / share;
        const int64_t per = (n_t + mc - 1) / mc;
        mc = (n_t + per - 1) / per;
        j.mc[i] = (int)mc;
        j.clen[i] = (int)(per * kTile < INT32_MAX ? per * kTile : INT32_MAX);
        j.pre[i + 1] = j.pre[i] + (int)mc * n_kv;
        j.stat[i] = stat;
        stat += (int64_t)j.ntok[i] * n_q * mc;
    }
    p->bytes = (size_t)stat * sizeof(float2);
}

template <int D, bool F32>
int launch(const eakvd_geom &g, const WeightsJob &job, const void *q, float2 *stat, float *out, int64_t ld,
           float keep, int vec, hipStream_t st)
{
    constexpr size_t bytes = sizeof(WLds<D, F32>);
    static_assert(bytes <= 160 * 1024, "LDS");
    auto run = [&](auto *kern, std::atomic<uint64_t> &done) {
        const int e = allow_lds((const void *)kern, bytes, done);
        if (e) return e;
        hipLaunchKernelGGL(kern, dim3((unsigned)job.pre[job.n_seq]), dim3(64 * kWaves), bytes, st, g, job, q,
                           stat, out, ld, keep, EAKV_LOG2E / sqrtf((float)D), vec);
        return (int)hipGetLastError();
    };
    static std::atomic<uint64_t> done[2];
    const int e = run(weights_kernel<D, F32, false>, done[0]);
    return e ? e : run(weights_kernel<D, F32, true>, done[1]);
}

}  // namespace

extern "C" size_t eakvd_weights_work_bytes(const eakvd_window *b, int n_q, int n_kv)
{
    WeightsPlan p;
    weights_plan(b, n_q, n_kv, &p);
    return p.bytes;
}

extern "C" int eakvd_weights(const eakvd_geom *g, const eakvd_window *b, int layer, const void *q, int bf16,
                             int n_q, int n_kv, float keep, float *out, int64_t ld, void *work, void *stream)
{
    WeightsPlan p;
    weights_plan(b, n_q, n_kv, &p);
    if (p.job.n_seq == 0) return 0;
    p.job.layer = layer;
    const hipStream_t st = (hipStream_t)stream;
    const int vec = (uintptr_t)q % 16 == 0;
    float2 *stat = (float2 *)work;
    if (g->head_dim == 64)
        return bf16 ? launch<64, false>(*g, p.job, q, stat, out, ld, keep, vec, st)
                    : launch<64, true>(*g, p.job, q, stat, out, ld, keep, vec, st);
    return bf16 ? launch<128, false>(*g, p.job, q, stat, out, ld, keep, vec, st)
                : launch<128, true>(*g, p.job, q, stat, out, ld, keep, vec, st);
}
