// window.hip — attention of several new tokens of each sequence over the packed
// cache: query i of a window that begins at position `start` sees the cache's
// tokens before start and, in the window, the tokens up to its own (causal) or
// the ones its mask word names (a tree of drafts).
//
//   out[i][h] = sum_t softmax_t(q[i][h].K[t] / sqrt(d)) V[t],
//   K[t] = n*s + b per group of 64 dims (n the nibble), V likewise.
//
// A kv head's rows (window tokens x the q heads that share it) are the columns
// of both products, so one pass over the packed planes serves all of them:
//   S^T = K Q^T    v_mfma_f32_32x32x16_f16, 32 tokens x 32 rows
//   O^T = V^T P^T  32 dims x 32 rows; a lane's 16 scores belong to one row, and
//                  the tokens of a K = 16 step are numbered so that the scores'
//                  registers are P's operand as they stand.
// K's operands are n - z, exact in f16 (z: the nibble nearest the value 0): score =
// sum over groups of s*(q.(n - z)) + c*sum(q), c = b + z*s, with s applied to the f32
// dots and the c terms computed by one bf16 product of three pieces each (24 bits).
// The nibbles become f16 once per block in LDS, in operand order, and are read
// by all waves that need them (WR waves of 32 rows each x WT waves that take
// different tokens).
//
// Two arithmetics:
//   f32 queries   Q and the weights p*s are pairs of f16 (24 bits together),
//                 V's operands n - z; its c terms are f32 sums of p*c.
//   bf16 queries  Q (8 bits) is exact in f16.  V is dequantized to f16,
//                 (n - z)*s + c with s and c rounded to f16, and p is rounded
//                 to f16: 2^-12 relative each, against the output's 2^-9.
// f16's range: Q rows are scaled by a power of two to below 2^15, V tiles (bf16) by
// theirs; the softmax's reference point M includes the exponent of the
// tile's V, so that every weight operand stays below 2^15 and keeps its
// precision down to 2^-29 of that.
//
// Softmax in the log2 domain, f32: M moves only when a score passes it by
// kTau; sums, weighted sums and M are f32.  Tokens are split into chunks where
// rows alone do not fill the chip; partial (O, M, l) are merged by a second
// launch.  No atomics: results are the same bits on every call.
#include <string.h>

#include "window.h"

namespace {

constexpr int kWinWaves = 8;           // waves of a block: two per SIMD

// LDS of one 32-token sub-tile.
template <int D, bool F32>
struct __align__(16) SubTile {
    static constexpr int GPD = D / 64;
    uint4 k[GPD * 4][64];               // operand (g, octet, nibble), by lane
    uint4 v[GPD * 4][64];               // operand (g, nibble, 16-token step), by lane
    uint4 kb[64];                       // K's biases in bf16 pieces, by lane
    float ks[GPD][32];                  // K's scales
    float vs[F32 ? GPD : 1][32];        // f32: scales and biases of V
    float vc[F32 ? GPD : 1][32];
    int ev[2];                          // exponent of V, by unit
    uint32_t bad[2][2];                 // bf16: tokens with non-finite V, by unit and group
};

// What a lane has in flight of one unit (a 64-lane share of a sub-tile's
// conversion): 16 packed bytes and their scales and biases.
struct Raw {
    uint4 x;
    float s[4], b[4];
};

// Everything a lane keeps of its row.
template <int D, bool F32>
struct Acc {
    v16f o[D / 32];                     // dims 32f + 8(i/4) + 4h + i%4 of register i
    float vc[D / 64];                   // f32: sum p*c by group (this half's tokens)
    float l;                            // sum p (this half's tokens)
    float m;                            // M
};

template <int D, bool F32, int WR, int SPW>
__global__ __launch_bounds__(64 * kWinWaves, 2) void window_kernel(
    eakvd_geom geo, WinJob job, const void *q, const uint64_t *tree, void *out, float *part,
    float rsd, int vec)
{
    constexpr int GPD = D / 64;
    constexpr int WT = kWinWaves / WR;
    constexpr int TS = WT * SPW;                     // sub-tiles of a tile
    constexpr int UPS = 2 * GPD;                     // units of a sub-tile: GPD of K, GPD of V
    constexpr int UPW = TS * UPS / kWinWaves;        // units of a wave
    static_assert(UPW * kWinWaves == TS * UPS, "whole units");
    constexpr int NB = WR == 1 ? 1 : 2;              // buffers; WR == 1: a wave's own sub-tile
    typedef SubTile<D, F32> Sub;
    extern __shared__ __align__(16) uint8_t lds[];
    Sub *sub = (Sub *)lds;

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int wr = w % WR, wt = w / WR;
    const int n32 = lane & 31, h = lane >> 5;

    // this block's sequence, rows, chunk and kv head; long row blocks first
    const int c = seq_of(job.pre, job.n_seq, (int)blockIdx.x, lane);
    int rem = (int)blockIdx.x - job.pre[c];
    const int kvh = rem % job.n_kv;
    rem /= job.n_kv;
    const int mc = job.mc[c], chunk = rem % mc;
    const int m = job.ntok[c], start = job.start[c], qpk = job.qpk;
    const int rows = m * qpk;
    const int n_rb = (rows + 32 * WR - 1) / (32 * WR);
    const int rb = n_rb - 1 - rem / mc;
    const int last_row = min(rows, (rb + 1) * 32 * WR) - 1;
    const int t_end = tree ? start + m : start + last_row / qpk + 1;    // tokens of this block
    const int lo = chunk * job.clen[c];
    const int hi = min(t_end, lo + job.clen[c]);

    const int r0 = rb * 32 * WR + wr * 32;           // this wave's first row
    const bool active = r0 < rows;
    const int row = min(r0 + n32, rows - 1);
    const int tok = row / qpk, head = kvh * qpk + row - tok * qpk;
    const int64_t qrow = ((int64_t)(job.tok0[c] + tok) * job.n_q + head) * D;
    // tokens that this row, the wave's first row and the wave's last row see
    const int vis = start + tok + 1;
    const int vis_min = tree ? start : start + min(r0, rows - 1) / qpk + 1;
    const int vis_max = tree ? start + m : start + min(r0 + 31, rows - 1) / qpk + 1;
    const uint64_t word = tree ? tree[job.tok0[c] + tok] : 0;

    QOp<D, F32> Q;
    build_q<D, F32>(Q, q, qrow, vec, rsd, h);
    const float rf = Q.rf;

    Acc<D, F32> A;
#pragma unroll
    for (int f = 0; f < D / 32; f++)
#pragma unroll
        for (int i = 0; i < 16; i++) A.o[f][i] = 0.0f;
#pragma unroll
    for (int g = 0; g < GPD; g++) A.vc[g] = 0.0f;
    A.l = 0.0f;
    A.m = kMInit;

    const Planes K = planes_of(geo, job.base[c], job.layer, 0);
    const Planes V = planes_of(geo, job.base[c], job.layer, 1);
    const int64_t g0 = (int64_t)kvh * geo.gph;
    const int t_last = t_end - 1;                    // loads stay within the sequence

    // ---- a unit's loads.  K unit g: lane = (token n32, bytes 16h of group g)
    // with the scales of group h.  V unit u: lane = (column quad, h, 16-token
    // step, x): four consecutive tokens' dwords; x is the group (d = 128) or
    // the 4-token half of the operand (d = 64), u the other one.
    const int cq = lane & 7, vh = (lane >> 3) & 1, vstep = (lane >> 4) & 1, vx = lane >> 5;
    auto load_unit = [&](int uu, int t0, Raw &r) {
        const int st = uu / UPS, kind = uu % UPS;
        const int tb = t0 + 32 * st;
        if (kind < GPD) {
            const int64_t t = min(tb + n32, t_last);
            r.x = *(const uint4 *)(K.w + (g0 + t * GPD + kind) * 32 + 16 * h);
            const int64_t gi = g0 + t * GPD + (GPD == 2 ? h : 0);
            r.s[0] = K.s[gi];
            r.b[0] = K.b[gi];
        } else {
            const int u = kind - GPD;
            const int g = GPD == 2 ? vx : 0, jh = GPD == 2 ? u : vx;
            const int tq = tb + 16 * vstep + 8 * jh + 4 * vh;
            uint32_t xx[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t t = min(tq + j, t_last);
                const int64_t gi = g0 + t * GPD + g;
                xx[j] = *(const uint32_t *)(V.w + gi * 32 + 4 * cq);
                r.s[j] = V.s[gi];
                r.b[j] = V.b[gi];
            }
            r.x = uint4{xx[0], xx[1], xx[2], xx[3]};
        }
    };

    // ---- a unit's conversion into the sub-tile's operands
    auto put_unit = [&](int uu, Sub *buf, const Raw &r) {
        const int st = uu / UPS, kind = uu % UPS;
        Sub &S = buf[st];
        if (kind < GPD) {
            const int g = kind;
            // lanes of half g (d = 64: all) hold group g's scale and bias
            float z = zero_nibble(r.s[0], r.b[0]);
            if (GPD == 1 || h == g) {
                const float s = r.s[0], cc = fmaf(z, s, r.b[0]);
                if (GPD == 2 || h == 0) S.ks[g][n32] = s;
                __bf16 p1, p2, p3;
                const __bf16 zero = (__bf16)0.0f;
                pieces(cc, p1, p2, p3);
                b8 v = b8{p1, p1, p1, p2, p2, p3, zero, zero};
                if (GPD == 1 && h == 1) v = b8{zero, zero, zero, zero, zero, zero, zero, zero};
                S.kb[lane] = __builtin_bit_cast(uint4, v);
            }
            if (GPD == 2) z = __shfl(z, 32 * g + n32, 64);
            const h2 off = pk(-z, -z);
            const uint32_t x[4] = {r.x.x, r.x.y, r.x.z, r.x.w};
#pragma unroll
            for (int o = 0; o < 2; o++) {
                uint32_t a[4], bb[4];
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint32_t x0 = x[2 * o + d], x1 = x0 >> 8;
                    a[2 * d] = u_of(nib2<false>(x0, off));
                    a[2 * d + 1] = u_of(nib2<false>(x1, off));
                    bb[2 * d] = u_of(nib2<true>(x0, off));
                    bb[2 * d + 1] = u_of(nib2<true>(x1, off));
                }
                S.k[g * 4 + o * 2][lane] = uint4{a[0], a[1], a[2], a[3]};
                S.k[g * 4 + o * 2 + 1][lane] = uint4{bb[0], bb[1], bb[2], bb[3]};
            }
        } else {
            const int u = kind - GPD;
            const int g = GPD == 2 ? vx : 0, jh = GPD == 2 ? u : vx;
            h2 s16[2], c16[2];
            float z[4];
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] = zero_nibble(r.s[j], r.b[j]);
            const h2 off[2] = {pk(-z[0], -z[2]), pk(-z[1], -z[3])};
            if constexpr (F32) {
                float top = 0.0f;
                float cc[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    cc[j] = fmaf(z[j], r.s[j], r.b[j]);
                    const float a = fabsf(r.s[j]);
                    top = fmaxf(top, a < __builtin_inff() ? a : 0.0f);
                }
                top = wave_top(top);
                const int tq = 16 * vstep + 8 * jh + 4 * vh;
                if (cq == 0) {
                    *(float4 *)&S.vs[g][tq] = make_float4(r.s[0], r.s[1], r.s[2], r.s[3]);
                    *(float4 *)&S.vc[g][tq] = make_float4(cc[0], cc[1], cc[2], cc[3]);
                }
                if (lane == 0) {
                    S.ev[u] = exp_of(top);
                    if (GPD == 1) S.ev[1] = exp_of(top);
                }
            } else {
                float top = 0.0f;
                bool fin[4], all = true;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float a = fmaxf(fabsf(r.b[j]), fabsf(fmaf(15.0f, r.s[j], r.b[j])));
                    fin[j] = a < __builtin_inff() && r.b[j] == r.b[j] && r.s[j] == r.s[j];
                    all = all && fin[j];
                    top = fmaxf(top, fin[j] ? a : 0.0f);
                }
                const int e = exp_of(wave_top(top));
                float ss[4], cc[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    ss[j] = scale2(r.s[j], 15 - e);
                    cc[j] = scale2(fmaf(z[j], r.s[j], r.b[j]), 15 - e);
                }
                if (lane == 0) {
                    S.ev[u] = e;
                    S.bad[u][0] = S.bad[u][1] = 0;
                    if (GPD == 1) {
                        S.ev[1] = e;
                        S.bad[1][0] = S.bad[1][1] = 0;
                    }
                }
                if (__ballot(!all) != 0) {
                    // non-finite groups: 0 in the operand, named in `bad`
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (!fin[j]) {
                            ss[j] = 0.0f;
                            cc[j] = 0.0f;
                            if (cq == 0)
                                atomicOr(&S.bad[u][g], 1u << (16 * vstep + 8 * jh + 4 * vh + j));
                        }
                    }
                }
                s16[0] = pk(ss[0], ss[2]);
                s16[1] = pk(ss[1], ss[3]);
                c16[0] = pk(cc[0], cc[2]);
                c16[1] = pk(cc[1], cc[3]);
            }
            // 4x4 byte transpose: y[i] = column 4cq + i of the four tokens
            const uint32_t x[4] = {r.x.x, r.x.y, r.x.z, r.x.w};
            const uint32_t a0 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);   // 0a 1a 0b 1b
            const uint32_t a1 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
            const uint32_t a2 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
            const uint32_t a3 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
            const uint32_t y[4] = {__builtin_amdgcn_perm(a1, a0, 0x05040100u),
                                   __builtin_amdgcn_perm(a1, a0, 0x07060302u),
                                   __builtin_amdgcn_perm(a3, a2, 0x05040100u),
                                   __builtin_amdgcn_perm(a3, a2, 0x07060302u)};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x0 = y[i], x1 = x0 >> 8;
                h2 v[4] = {nib2<false>(x0, off[0]), nib2<false>(x1, off[1]),
                           nib2<true>(x0, off[0]), nib2<true>(x1, off[1])};
                if constexpr (!F32) {
#pragma unroll
                    for (int p = 0; p < 4; p++)
                        v[p] = __builtin_elementwise_fma(v[p], s16[p & 1], c16[p & 1]);
                }
                const int slot = 32 * vh + 4 * cq + i;
                uint2 *lo2 = (uint2 *)&S.v[g * 4 + 0 + vstep][slot] + jh;
                uint2 *hi2 = (uint2 *)&S.v[g * 4 + 2 + vstep][slot] + jh;
                *lo2 = uint2{u_of(v[0]), u_of(v[1])};
                *hi2 = uint2{u_of(v[2]), u_of(v[3])};
            }
        }
    };

    // ---- one sub-tile's scores, softmax and weighted sum for this wave's rows
    auto step = [&](const Sub &S, int t0, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        v16f s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, S.kb[lane]), Q.bias, s, 0, 0,
                                                    0);
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            v16f acc;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[i] = 0.0f;
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const h8 a = __builtin_bit_cast(h8, S.k[g * 4 + f][lane]);
                if constexpr (F32)
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, Q.b[g * 4 + f], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, Q.a[g * 4 + f], acc, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 sc = *(const float4 *)&S.ks[g][8 * k + 4 * h];
                s[4 * k] = fmaf(sc.x, acc[4 * k], s[4 * k]);
                s[4 * k + 1] = fmaf(sc.y, acc[4 * k + 1], s[4 * k + 1]);
                s[4 * k + 2] = fmaf(sc.z, acc[4 * k + 2], s[4 * k + 2]);
                s[4 * k + 3] = fmaf(sc.w, acc[4 * k + 3], s[4 * k + 3]);
            }
        }
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int t = t0 + 8 * (i >> 2) + 4 * h + (i & 3);
                bool see = t < vis;
                if (tree) {
                    const int d = t - start;
                    see = d < 0 || (d < m && ((word >> (d & 63)) & 1));
                }
                s[i] = see ? s[i] : -__builtin_inff();
            }
        }
        const int ev0 = S.ev[0], ev1 = S.ev[1];
        const int evm = max(ev0, ev1);
        float top = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
        for (int i = 3; i < 16; i++) top = fmaxf(top, s[i]);
        top = half_max(top);
        const float need = fmaf(top, rf, (float)evm - kWinTop);
        if (__ballot(need > A.m + kWinTau) != 0) {
            const float mn = fmaxf(A.m, need);
            const float al = __builtin_amdgcn_exp2f(A.m - mn);
            A.m = mn;
            A.l *= al;
#pragma unroll
            for (int f = 0; f < D / 32; f++)
#pragma unroll
                for (int i = 0; i < 16; i++) A.o[f][i] *= al;
            if constexpr (F32)
#pragma unroll
                for (int g = 0; g < GPD; g++) A.vc[g] *= al;
        }
        if constexpr (F32) {
            float p[16];
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], rf, -A.m));
            A.l += ((((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))) +
                    (((p[8] + p[9]) + (p[10] + p[11])) + ((p[12] + p[13]) + (p[14] + p[15]))));
#pragma unroll
            for (int g = 0; g < GPD; g++) {
                uint32_t a[8], b[8];
                float cs = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float4 sc = *(const float4 *)&S.vs[g][8 * k + 4 * h];
                    const float4 cc = *(const float4 *)&S.vc[g][8 * k + 4 * h];
                    float x[4];
                    if constexpr (MASK) {
                        x[0] = mul_hidden(p[4 * k], sc.x);
                        x[1] = mul_hidden(p[4 * k + 1], sc.y);
                        x[2] = mul_hidden(p[4 * k + 2], sc.z);
                        x[3] = mul_hidden(p[4 * k + 3], sc.w);
                        cs += mul_hidden(p[4 * k], cc.x) + mul_hidden(p[4 * k + 1], cc.y);
                        cs += mul_hidden(p[4 * k + 2], cc.z) + mul_hidden(p[4 * k + 3], cc.w);
                    } else {
                        x[0] = p[4 * k] * sc.x;
                        x[1] = p[4 * k + 1] * sc.y;
                        x[2] = p[4 * k + 2] * sc.z;
                        x[3] = p[4 * k + 3] * sc.w;
                        cs = fmaf(p[4 * k], cc.x, cs);
                        cs = fmaf(p[4 * k + 1], cc.y, cs);
                        cs = fmaf(p[4 * k + 2], cc.z, cs);
                        cs = fmaf(p[4 * k + 3], cc.w, cs);
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const h2 hi2 = pk(x[e], x[e + 2]);
                        a[2 * k + e] = u_of(hi2);
                        b[2 * k + e] = u_of(pk_rest(hi2, x[e], x[e + 2]));
                    }
                }
                A.vc[g] += cs;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    const h8 pa = __builtin_bit_cast(h8, uint4{a[4 * ks], a[4 * ks + 1],
                                                               a[4 * ks + 2], a[4 * ks + 3]});
                    const h8 pb = __builtin_bit_cast(h8, uint4{b[4 * ks], b[4 * ks + 1],
                                                               b[4 * ks + 2], b[4 * ks + 3]});
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const h8 v = __builtin_bit_cast(h8, S.v[g * 4 + n * 2 + ks][lane]);
                        A.o[g * 2 + n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            v, pb, A.o[g * 2 + n], 0, 0, 0);
                        A.o[g * 2 + n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            v, pa, A.o[g * 2 + n], 0, 0, 0);
                    }
                }
            }
        } else {
            // V's unit jh has an exponent of its own: tokens with (i >> 2) & 1
            // = jh (d = 64: one for both)
            const float d0 = (float)ev0 - A.m, d1 = (float)ev1 - A.m;
            float p[16], sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 16; i++) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], rf, (i >> 2) & 1 ? d1 : d0));
                sum[(i >> 2) & 1] += p[i];
            }
            A.l += scale2(sum[0], -ev0) + scale2(sum[1], -ev1);
            uint32_t a[8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                a[2 * k] = u_of(pk_exp(p[4 * k], p[4 * k + 2]));
                a[2 * k + 1] = u_of(pk_exp(p[4 * k + 1], p[4 * k + 3]));
            }
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const h8 pa = __builtin_bit_cast(h8, uint4{a[4 * ks], a[4 * ks + 1], a[4 * ks + 2],
                                                           a[4 * ks + 3]});
#pragma unroll
                for (int f = 0; f < D / 32; f++)
                    A.o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                        __builtin_bit_cast(h8, S.v[(f >> 1) * 4 + (f & 1) * 2 + ks][lane]), pa,
                        A.o[f], 0, 0, 0);
            }
            uint32_t bad[2] = {S.bad[0][0] | S.bad[1][0], S.bad[0][1] | S.bad[1][1]};
            if (__builtin_amdgcn_readfirstlane(bad[0] | bad[1])) {
                // rows that see a token with a non-finite V group: NaN there
                uint32_t seen = 0;
#pragma unroll
                for (int i = 0; i < 16; i++)
                    seen |= (s[i] != -__builtin_inff() ? 1u : 0u)
                            << (8 * (i >> 2) + 4 * h + (i & 3));
                seen |= __shfl_xor(seen, 32, 64);
#pragma unroll
                for (int g = 0; g < GPD; g++)
                    if (seen & bad[g])
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            A.o[2 * g][i] = A.o[2 * g + 1][i] = __builtin_nanf("");
            }
        }
    };

    // ---- tiles of 32 * TS tokens; the next tile's loads are in flight while
    // one is computed
    Raw raw[UPW];
    const int n_tiles = hi > lo ? (hi - lo + 32 * TS - 1) / (32 * TS) : 0;
    auto load_tile = [&](int i) {
#pragma unroll
        for (int k = 0; k < UPW; k++) load_unit(w * UPW + k, lo + 32 * TS * i, raw[k]);
    };
    if (n_tiles) load_tile(0);
    for (int i = 0; i < n_tiles; i++) {
        Sub *buf = sub + (NB == 2 ? (i & 1) * TS : 0);
        // WR == 1: the wave's own sub-tile, ordered by its LDS instructions' order
        if constexpr (WR == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int k = 0; k < UPW; k++) put_unit(w * UPW + k, buf, raw[k]);
        if (i + 1 < n_tiles) load_tile(i + 1);
        if constexpr (WR > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int tb = lo + 32 * TS * i;
#pragma unroll
        for (int k = 0; k < SPW; k++) {
            const int st = WR == 1 ? w : wt * SPW + k;
            const int t0 = tb + 32 * st;
            if (!active || t0 >= min(vis_max, hi)) continue;
            if (t0 + 32 <= vis_min) step(buf[st], t0, std::false_type{});
            else step(buf[st], t0, std::true_type{});
        }
    }

    // ---- both halves of a row's tokens, then the WT waves of these rows
    const float l = A.l + __shfl_xor(A.l, 32, 64);
    if constexpr (F32) {
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            const float cs = A.vc[g] + __shfl_xor(A.vc[g], 32, 64);
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) A.o[2 * g + n][i] += cs;
        }
    } else {
        // the operands carried 2^15
#pragma unroll
        for (int f = 0; f < D / 32; f++)
#pragma unroll
            for (int i = 0; i < 16; i++) A.o[f][i] *= 0x1p-15f;
    }
    const RowOut ro = row_out(job, c, chunk, tok, head, D, qrow, vec, part);
    if constexpr (WT > 1) {
        join_put<D, F32, WT>((float *)lds, wt, wr, WR, lane, A.o, l, A.m, active && r0 + n32 < rows, ro, out,
                             part);
    } else if (active && r0 + n32 < rows) {
        put_rows<D, F32>(ro, A.o, l, A.m, h, out, part);
    }
}

// One wave per (window token, q head) of the sequences with chunks: the
// chunks' (O, M, l) joined.  A chunk without visible tokens has l = 0 and no O.
template <int D, bool F32>
__global__ __launch_bounds__(256) void window_merge_kernel(WinJob job, const float *part,
                                                           void *out, int n_rows)
{
    constexpr int E = D / 64;
    const int r = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (r >= n_rows) return;
    const int tok = r / job.n_q;
    const int c = seq_of(job.lead, job.n_seq, tok, lane);
    const int mc = job.mc[c];
    if (mc == 1) return;
    const int64_t per = (int64_t)job.ntok[c] * job.n_q;
    const int64_t local = r - (int64_t)job.lead[c] * job.n_q;
    const int64_t first = job.part[c] + local;
    const float *ml = part + job.part_rows * D;
    float m = kMInit;
    for (int k = lane; k < mc; k += 64) {
        const float2 x = *(const float2 *)(ml + (first + k * per) * 2);
        if (x.y != 0.0f) m = fmaxf(m, x.x);
    }
    m = wave_max(m);
    float l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    for (int k = 0; k < mc; k++) {
        const float2 x = *(const float2 *)(ml + (first + k * per) * 2);
        if (x.y == 0.0f) continue;
        const float a = __builtin_amdgcn_exp2f(x.x - m);
        l = fmaf(a, x.y, l);
        const float *po = part + (first + k * per) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(a, po[e], o[e]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int64_t at = ((int64_t)job.tok0[c] * job.n_q + local) * D + lane * E + e;
        if constexpr (F32) ((float *)out)[at] = o[e] * inv;
        else ((uint16_t *)out)[at] = (uint16_t)bf16_bits(o[e] * inv);
    }
}

// The sequences of one launch: those of few rows (window_kernel) or of many
// (win_prompt).
struct WinPart {
    WinJob job;
    int wr;                 // window_kernel: waves by rows
    int n_tok;              // window tokens of its sequences
    int64_t subtiles;       // win_prompt: expanded
    size_t part_bytes, bytes;
    bool merge;
};

struct WinPlan {
    WinPart few, many;
};

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int tile_of(int wr, int d)
{
    const int spw = wr == 8 ? (d == 128 ? 2 : 4) : wr == 4 ? (d == 128 ? 1 : 2) : 1;
    return 32 * (kWinWaves / wr) * spw;
}

// Whether a window's K and V are expanded first (never a tree's): where several
// blocks of 256 rows share them.  Expanded against not, 32Q/8KV d128: bf16 256 tokens
// at 30000 192 against 226 us, at 2000 39 against 41, 100 tokens (400 rows) at 30000
// 123 against 130, at 2000 34.6 against 33.1; f32 1000 tokens 71 against 79, but 256
// at 30000 440 against 363 (the products there are twice as many, so conversions
// weigh less).
#ifndef LD_
#define LD_ 1
#endif
constexpr int kLeastDraft = LD_;
bool is_many(int ntok, int qpk, bool bf16)
{
    return ntok > EAKVD_TREE_MAX && (int64_t)ntok * qpk > (bf16 ? 256 : 2048);
}

// Tiles of a chunk, window_kernel and win_draft: an even share of the chip, and at
// least `least`; at most 2^25 tokens (win_draft's offsets from a chunk's first token
// are 32 bits).
int64_t few_share(int64_t tiles, int cus, int tile, int least)
{
    int64_t s = (tiles + cus - 1) / cus;
    s = s < least ? least : s;
    const int64_t most = (1 << 25) / tile;
    return s < most ? s : most;
}

// Tiles of a chunk, win_prompt: the split of the longest context in k that ends first,
// by a model of a launch in tile times (256 rows x 32 tokens: about 1.05 us at d = 128
// in bf16, 1.6 in f32).  Blocks beyond the chip's slots run as slots come free, the
// longest first; partials are written and read at about 5 TB/s, the merge is
// a launch of its own.
int64_t many_share(const WinJob &j, int64_t tiles, int cus, int head_dim, bool bf16)
{
    int64_t longest = 1, blocks = 0, rows = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t n_t = ((int64_t)j.start[i] + j.ntok[i] + 31) / 32;
        const int64_t r = (int64_t)j.ntok[i] * j.qpk;
        longest = n_t > longest ? n_t : longest;
        blocks += (r + 255) / 256 * j.n_kv;
        rows += r * j.n_kv;
    }
    const double tile_us = (bf16 ? 1.05 : 1.6) * head_dim / 128;
    const double merge_k = 2.0 * rows * (head_dim + 2) * 4 / 5e6 / tile_us, merge_0 = 6 / tile_us;
    double best = 0;
    int64_t share = longest;
    for (int k = 1; k <= 64 && (k == 1 || longest / k >= 8); k = k < 4 ? k + 1 : k + k / 2) {
        const int64_t part = (longest + k - 1) / k;
        double t = part;
        if (blocks * k > cus) {
            const double even = (double)tiles / cus + 0.5 * part;
            t = even > t ? even : t;
        }
        if (k > 1) t += merge_0 + merge_k * k;
        if (k == 1 || t < best) {
            best = t;
            share = part;
        }
    }
    return share;
}

void plan_part(const eakvd_geom *g, const eakvd_window *b, int n_q, int n_kv, bool bf16, bool many,
               WinPart *p)
{
    memset(p, 0, sizeof(*p));
    WinJob &j = p->job;
    const int qpk = n_q / n_kv;
    j.n_q = n_q;
    j.n_kv = n_kv;
    j.qpk = qpk;
    int64_t most = 0;
    int tok0 = 0;
    for (int i = 0; i < b->n_seq; i++) {
        if (b->ntok[i] && is_many(b->ntok[i], qpk, bf16) == many) {
            const int k = j.n_seq++;
            const int64_t rows = (int64_t)b->ntok[i] * qpk;
            most = rows > most ? rows : most;
            j.base[k] = b->base[i];
            j.start[k] = b->start[i];
            j.ntok[k] = b->ntok[i];
            j.tok0[k] = tok0;
        }
        tok0 += b->ntok[i];
    }
    p->wr = most <= 32 ? 1 : most <= 64 ? 2 : most <= 128 ? 4 : 8;
    const int rbr = many ? 256 : 32 * p->wr, tile = many ? 32 : tile_of(p->wr, g->head_dim);
    // tiles of all blocks, were no sequence split
    int64_t tiles = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t rows = (int64_t)j.ntok[i] * qpk, nrb = (rows + rbr - 1) / rbr;
        for (int64_t r = 0; r < nrb; r++) {
            const int64_t last = (rows < (r + 1) * rbr ? rows : (r + 1) * rbr) - 1;
            // (a tree's rows may all see the whole window; it is short)
            const int64_t end = (int64_t)j.start[i] + (many ? last / qpk + 1 : j.ntok[i]);
            tiles += (end + tile - 1) / tile * n_kv;
        }
    }
    const int cus = cu_count();
    const int64_t share = many ? many_share(j, tiles, cus, g->head_dim, bf16)
                               : few_share(tiles, cus, tile, p->wr == 1 ? kLeastDraft : 4);
    int64_t part = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t rows = (int64_t)j.ntok[i] * qpk, nrb = (rows + rbr - 1) / rbr;
        const int64_t n_t = ((int64_t)j.start[i] + j.ntok[i] + tile - 1) / tile;
        int64_t mc = (n_t + share - 1) / share;
        const int64_t per = (n_t + mc - 1) / mc;
        mc = (n_t + per - 1) / per;
        j.mc[i] = (int)mc;
        j.clen[i] = (int)(per * tile);
        j.pre[i + 1] = j.pre[i] + (int)(nrb * mc * n_kv);
        j.part[i] = part;
        if (mc > 1) {
            part += rows * n_kv * mc;
            p->merge = true;
        }
        j.lead[i] = p->n_tok;
        p->n_tok += j.ntok[i];
        j.nsub[i] = (j.start[i] + j.ntok[i] + 31) / 32;
        j.img[i] = p->subtiles;
        p->subtiles += (int64_t)j.nsub[i] * n_kv;
    }
    j.part_rows = part;
    p->part_bytes = align256((size_t)part * (g->head_dim + 2) * sizeof(float));
    p->bytes = p->part_bytes;
    if (many && j.n_seq) p->bytes += align256(win_prompt_bytes(g->head_dim, bf16, p->subtiles));
}

void win_plan(const eakvd_geom *g, const eakvd_window *b, int n_q, int n_kv, bool bf16, WinPlan *p)
{
    plan_part(g, b, n_q, n_kv, bf16, false, &p->few);
    plan_part(g, b, n_q, n_kv, bf16, true, &p->many);
}

int merge(const eakvd_geom *g, const WinPart &p, bool bf16, const float *part, void *out,
          hipStream_t st)
{
    if (!p.merge) return 0;
    const int n_rows = p.n_tok * p.job.n_q;
    auto *kern = g->head_dim == 64
                     ? (bf16 ? window_merge_kernel<64, false> : window_merge_kernel<64, true>)
                     : (bf16 ? window_merge_kernel<128, false> : window_merge_kernel<128, true>);
    hipLaunchKernelGGL(kern, dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, st, p.job, part, out,
                       n_rows);
    return (int)hipGetLastError();
}

template <int D, bool F32, int WR, int SPW>
int launch(const eakvd_geom *g, const WinPart &p, const void *q, const uint64_t *tree, void *out,
           float *part, int vec, hipStream_t st)
{
    constexpr int WT = kWinWaves / WR;
    constexpr size_t tiles = (size_t)WT * SPW * (WR == 1 ? 1 : 2) * sizeof(SubTile<D, F32>);
    constexpr size_t join = WT > 1 ? kJoinBytes<D> : 0;
    constexpr size_t bytes = tiles > join ? tiles : join;
    static_assert(bytes <= 160 * 1024, "LDS");
    auto *kern = window_kernel<D, F32, WR, SPW>;
    static std::atomic<uint64_t> done;
    const int e = allow_lds((const void *)kern, bytes, done);
    if (e) return e;
    const float rsd = 1.0f / sqrtf((float)D);
    hipLaunchKernelGGL(kern, dim3((unsigned)p.job.pre[p.job.n_seq]), dim3(64 * kWinWaves), bytes, st,
                       *g, p.job, q, tree, out, part, rsd, vec);
    return (int)hipGetLastError();
}

template <int D, bool F32>
int launch_wr(const eakvd_geom *g, const WinPart &p, const void *q, const uint64_t *tree, void *out,
              float *part, int vec, hipStream_t st)
{
    switch (p.wr) {
    case 1: return win_draft(*g, p.job, !F32, q, tree, out, part, vec, st);
    case 2: return launch<D, F32, 2, 1>(g, p, q, tree, out, part, vec, st);
    case 4: return launch<D, F32, 4, D == 128 ? 1 : 2>(g, p, q, tree, out, part, vec, st);
    default: return launch<D, F32, 8, D == 128 ? 2 : 4>(g, p, q, tree, out, part, vec, st);
    }
}

}  // namespace

extern "C" size_t eakvd_window_work_bytes(const eakvd_geom *g, const eakvd_window *b, int n_q,
                                          int n_kv, int bf16)
{
    WinPlan p;
    win_plan(g, b, n_q, n_kv, bf16, &p);
    return p.few.bytes + p.many.bytes;
}

extern "C" int eakvd_window_attend(const eakvd_geom *g, const eakvd_window *b, int layer,
                                   const void *q, int bf16, int n_q, int n_kv,
                                   const uint64_t *tree, void *out, void *work, void *stream)
{
    WinPlan p;
    win_plan(g, b, n_q, n_kv, bf16, &p);
    p.few.job.layer = p.many.job.layer = layer;
    const hipStream_t st = (hipStream_t)stream;
    // 16-byte loads of q and 16- or 8-byte stores of out
    const int vec = (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0;
    uint8_t *w = (uint8_t *)work;
    int e = 0;
    if (p.many.job.n_seq) {
        e = win_prompt(*g, p.many.job, p.many.subtiles, bf16, q, out, (float *)w,
                       w + p.many.part_bytes, vec, st);
        if (!e) e = merge(g, p.many, bf16, (const float *)w, out, st);
        w += p.many.bytes;
    }
    if (!e && p.few.job.n_seq) {
        float *part = (float *)w;
        if (g->head_dim == 64)
            e = bf16 ? launch_wr<64, false>(g, p.few, q, tree, out, part, vec, st)
                     : launch_wr<64, true>(g, p.few, q, tree, out, part, vec, st);
        else
            e = bf16 ? launch_wr<128, false>(g, p.few, q, tree, out, part, vec, st)
                     : launch_wr<128, true>(g, p.few, q, tree, out, part, vec, st);
        if (!e) e = merge(g, p.few, bf16, part, out, st);
    }
    return e;
}
