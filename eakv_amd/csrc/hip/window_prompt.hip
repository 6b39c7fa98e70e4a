// window_prompt.hip — the window attention of many rows (pieces of prompts): K and V of
// a layer are expanded once into matrix operands in device scratch, and blocks of
// 256 rows read them from there.
//
// One launch writes, for every (kv head, 32 tokens), the operands as LDS holds them:
// 18 KB (d = 128) against 5 KB packed, once per call.  In the attention launch they
// go from the L2 to LDS without passing a register (buffer loads to LDS), so its
// vector instructions are the softmax's alone.
//
// K: n - z, exact, with the scales and biases beside them, as in window.hip.  (Values in
// f16 instead save the scales' 32 instructions per 32 x 32 and a product, 1020-1080 us
// against 1190-1250 for the prompt below; but their 2^-12 enters the scores times the
// scores' size: K on an offset of 100 made outputs 2e-2 off.)  V, f32 queries: likewise; bf16 queries:
// values n*s + b (f32) scaled by the token's power of two and rounded to f16, 2^-12
// relative.
//
// Attention: 8 waves per block, two per SIMD, 32 rows each, through a ring of 8 sub-tiles
// in LDS with a barrier every kStep.  A step of a wave is the products (the next
// sub-tile's scores and this one's weighted sum), then the softmax; a SIMD's two
// waves are in different halves of it.
//
// Bound by the matrix cores and the vector ALUs in turn: 2048 tokens at 30720 of
// 32Q/8KV, bf16 (1.07 Tflop): 1190-1250 us, 850-890 Tflop/s, with the matrix cores busy 45
// and the vector ALUs 46 of 100 cycles at about 2.0 GHz.  f32, twice the products and 320
// vector instructions for 32 x 32: 2.2 us per 32 tokens of a block against 1.2.
#include <string.h>

#include "window.h"

namespace {

constexpr int kRing = 8;
constexpr int kPRows = 256;             // of a block: 32 of each wave
constexpr int kPWaves = kPRows / 32;
// Sub-tiles between barriers: 3 measured 1076 us (2048 tokens at 30720, 32Q/8KV d128
// bf16), 2 1096, 1 1128.
constexpr int kStep = 3;

typedef __attribute__((address_space(3))) void *lds_p;

// Bytes of an expanded sub-tile: K operands (g, octet, nibble), V operands (g, nibble,
// 16-token step), 1 KB each; K's operand of the bias product (1 KB), then scales of K
// [group][token], 2^-e of the tokens' exponents e of V, and (f32) 2^-e of the scales and
// biases of V [group][token].
template <int D, bool F32>
struct Img {
    static constexpr int GPD = D / 64;
    static constexpr int V = GPD * 4 * 1024;
    static constexpr int KB = 2 * V;
    static constexpr int KS = KB + 1024;
    static constexpr int W = KS + GPD * 128;
    static constexpr int VS = W + 128;
    static constexpr int VC = VS + GPD * 128;
    static constexpr int BYTES = F32 ? VC + GPD * 128 : VS;
    static constexpr int N = (BYTES + 1023) / 1024;         // pieces of 1 KB, the last one
                                                            // over the end of the one before
    static constexpr int LOADS = N / kPWaves;            // of each wave; the first
    static constexpr int MORE = N % kPWaves;             // MORE waves one more
};

// Per sub-tile: tokens with non-finite V, by group.
struct Meta {
    uint32_t bad[2];
};

// One block per (sub-tile, kv head), two operands of 1 KB to a wave: wave j < 2 GPD makes
// K's of (g, octet), the others V's of (g, 16-token step).
template <int D, bool F32>
__global__ __launch_bounds__(64 * 4 * (D / 64)) void expand_kernel(eakvd_geom geo, WinJob job,
                                                                   uint8_t *img, Meta *meta, float ksc)
{
    constexpr int GPD = D / 64;
    typedef Img<D, F32> I;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n32 = lane & 31, h = lane >> 5;
    int c = 0;
    while (c + 1 < job.n_seq && (int64_t)blockIdx.x >= job.img[c + 1]) c++;
    const int rem = (int)((int64_t)blockIdx.x - job.img[c]);
    const int nsub = job.nsub[c];
    const int kvh = rem / nsub, sub = rem - kvh * nsub;
    const int t_last = job.start[c] + job.ntok[c] - 1;
    uint8_t *o = img + (int64_t)blockIdx.x * I::BYTES;
    const bool is_v = w >= 2 * GPD;
    const int g = (w >> 1) % GPD, x = w & 1;             // x: octet (K), 16-token step (V)
    const Planes P = planes_of(geo, job.base[c], job.layer, is_v);
    const int64_t g0 = (int64_t)kvh * geo.gph;
    const int t0 = 32 * sub;
    // scales of (token n32, group h or the only one)
    const int64_t tn = min(t0 + n32, t_last);
    const int64_t gi = g0 + tn * GPD + (GPD == 2 ? h : 0);
    const float s = P.s[gi], b = P.b[gi];
    // V's scales, finite or not, and its token's exponent
    const Planes Pv = planes_of(geo, job.base[c], job.layer, 1);
    const float vs = is_v ? s : Pv.s[gi], vb = is_v ? b : Pv.b[gi];
    const float a = fmaxf(fabsf(vb), fabsf(fmaf(15.0f, vs, vb)));
    const bool fin = a < __builtin_inff() && vs == vs;
    const float top = fin ? v_size<F32>(vs, a) : 0.0f;
    const int e = exp_of(GPD == 2 ? half_max(top) : top);
    if (!is_v) {
        const uint2 by = *(const uint2 *)(P.w + (g0 + tn * GPD + g) * 32 + 16 * h + 8 * x);
        const uint32_t xs[2] = {by.x, by.y};
        const float sg = GPD == 2 ? __shfl(s, 32 * g + n32, 64) : s;
        const float bg = GPD == 2 ? __shfl(b, 32 * g + n32, 64) : b;
        uint32_t lo[4], hi[4];
        const float z = zero_nibble(sg, bg);
        const h2 off_l = nib_off<false>(z, z), off_h = nib_off<true>(z, z);
        NibConst nc;
        nc.hold();
#pragma unroll
        for (int d = 0; d < 2; d++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t y = xs[d] >> (8 * p);     // bytes p and p + 2
                lo[2 * d + p] = u_of(nib2<false>(y, off_l, nc));
                hi[2 * d + p] = u_of(nib2<true>(y, off_h, nc));
            }
        uint4 *ok = (uint4 *)o + (g * 4 + 2 * x) * 64 + lane;
        ok[0] = uint4{lo[0], lo[1], lo[2], lo[3]};
        ok[64] = uint4{hi[0], hi[1], hi[2], hi[3]};
        if (x == 0 && (GPD == 1 || h == g)) {
            const float k = fmaf(z, s, b) * (ksc * kKBias<F32>);
            *((uint4 *)(o + I::KB) + lane) =
                __builtin_bit_cast(uint4, k_bias(GPD == 1 && h == 1 ? 0.0f : k, e, h));
            if (GPD == 2 || h == 0) ((float *)(o + I::KS))[32 * g + n32] = s * ksc;
        }
    } else {
        const uint64_t bad = __ballot(!fin);
        if (g == 0 && x == 0 && lane == 0) {
            meta[blockIdx.x].bad[0] = (uint32_t)bad;
            meta[blockIdx.x].bad[1] = GPD == 2 ? (uint32_t)(bad >> 32) : 0;
        }
        if (g == 0 && x == 0 && h == 0) ((float *)(o + I::W))[n32] = scale2(1.0f, -e);
        // column n32 of group g; tokens 16x + 8(j/4) + 4h + j%4
        float v0[8], v1[8];
        uint32_t n0[8];
        float zz[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int tl = 16 * x + 8 * (j >> 2) + 4 * h + (j & 3);
            const int64_t t = min(t0 + tl, t_last);
            n0[j] = P.w[(g0 + t * GPD + g) * 32 + n32];
            const float sj = __shfl(s, (GPD == 2 ? 32 * g : 0) + tl, 64);
            const float bj = __shfl(b, (GPD == 2 ? 32 * g : 0) + tl, 64);
            const bool fj = (bad >> ((GPD == 2 ? 32 * g : 0) + tl)) & 1;
            if constexpr (F32) {
                zz[j] = zero_nibble(sj, bj);
                v0[j] = (float)(n0[j] & 15) - zz[j];
                v1[j] = (float)(n0[j] >> 4) - zz[j];
            } else {
                const int ej = __shfl(e, tl, 64);
                v0[j] = fj ? 0.0f : scale2(fmaf((float)(n0[j] & 15), sj, bj), 15 - ej);
                v1[j] = fj ? 0.0f : scale2(fmaf((float)(n0[j] >> 4), sj, bj), 15 - ej);
            }
        }
        uint4 *ov = (uint4 *)(o + I::V) + (g * 4 + x) * 64 + lane;
        ov[0] = uint4{u_of(pk(v0[0], v0[2])), u_of(pk(v0[1], v0[3])), u_of(pk(v0[4], v0[6])),
                      u_of(pk(v0[5], v0[7]))};
        ov[128] = uint4{u_of(pk(v1[0], v1[2])), u_of(pk(v1[1], v1[3])), u_of(pk(v1[4], v1[6])),
                        u_of(pk(v1[5], v1[7]))};
        if constexpr (F32) {
            if (g == 0 && x == 0 && (GPD == 2 || h == 0)) {
                // (a non-finite group counts as zeros and makes the rows that see it NaN)
                const float z = zero_nibble(s, b);
                ((float *)(o + I::VS))[lane] = fin ? scale2(s, -e) : 0.0f;
                ((float *)(o + I::VC))[lane] = fin ? scale2(fmaf(z, s, b), -e) : 0.0f;
            }
        }
    }
}

// PF: operands are read from LDS ahead of their step.  d = 64 in bf16 without: two blocks
// to a CU.
template <int D, bool F32, bool PF>
__global__ __launch_bounds__(64 * kPWaves, D == 64 && !F32 && !PF ? 4 : 2) void prompt_kernel(
    WinJob job, const uint8_t *img, const Meta *meta, const void *q, void *out, float *part, int vec)
{
    constexpr int GPD = D / 64;
    typedef Img<D, F32> I;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n32 = lane & 31, h = lane >> 5;

    const int c = seq_of(job.pre, job.n_seq, (int)blockIdx.x, lane);
    int rem = (int)blockIdx.x - job.pre[c];
    const int kvh = rem % job.n_kv;
    rem /= job.n_kv;
    const int mc = job.mc[c], chunk = rem % mc;
    const int m = job.ntok[c], start = job.start[c], qpk = job.qpk;
    const int rows = m * qpk;
    const int n_rb = (rows + kPRows - 1) / kPRows;
    const int rb = n_rb - 1 - rem / mc;
    const int first_row = rb * kPRows, last_row = min(rows, first_row + kPRows) - 1;
    const int t_end = start + last_row / qpk + 1;
    const int lo = chunk * job.clen[c];
    const int hi = t_end - lo > job.clen[c] ? lo + job.clen[c] : t_end;
    const int n_i = hi > lo ? (hi - lo + 31) / 32 : 0;   // sub-tiles of this block
    // the first that some row of the block does not see whole
    const int vis_min = start + first_row / qpk + 1;

    const int r0 = first_row + w * 32;
    const int row = min(r0 + n32, rows - 1);
    const int tok = row / qpk, head = kvh * qpk + row - tok * qpk;
    const int64_t qrow = ((int64_t)(job.tok0[c] + tok) * job.n_q + head) * D;
    const int vis = start + tok + 1;
    QOp<D, F32> Q;
    {
        QRaw<D, F32> raw;
        load_q<D, F32>(raw, q, qrow, vec, h);
        build_q<D, F32, false>(Q, raw, h);
    }
    const bool own_rf = F32 || __ballot(Q.rf != 1.0f) != 0;
    Soft<D, F32> R;
    R.clear();
    // sub-tiles that a row of this wave sees
    const int vis_max = r0 < rows ? start + min(r0 + 31, rows - 1) / qpk + 1 : 0;
    const int n_w = min(n_i, vis_max > lo ? (vis_max - lo + 31) / 32 : 0);

    const int64_t tile0 = job.img[c] + (int64_t)kvh * job.nsub[c] + lo / 32;
    const uint8_t *src = img + tile0 * I::BYTES;
    const Meta *mt = meta + tile0;
    // f32: lane j holds whether sub-tile 64k + j has non-finite V (scalar loads would be
    // waited for with the phase's LDS reads: 183 against 175 us for 2000 tokens of
    // 32Q/32KV); bf16: scalars of this sub-tile (readlane instead: 1113 against 1096 us for
    // 2048 tokens at 30720 of 32Q/8KV)
    uint32_t m_bad = 0;
    auto load_meta = [&](int i) __attribute__((always_inline)) {
        if constexpr (F32) {
            if (i % 64 == 0) {
                const Meta &x = mt[min(i + lane, n_i - 1)];
                m_bad = x.bad[0] | x.bad[1];
            }
        } else {
            typedef const __attribute__((address_space(4))) Meta *Const;
            const Const x = (Const)(uintptr_t)mt + min(i, n_i - 1);
            m_bad = x->bad[0] | x->bad[1];
        }
    };

    // sub-tile i into its ring slot: this wave's pieces of 1 KB.  (Lanes all load, or else
    // the compiler may split and join loads, and sync counts them.)
    auto fetch = [&](int i) {
        const int j = min(i, n_i - 1);
        const uint8_t *p = src + (int64_t)j * I::BYTES;
        uint8_t *slot = lds + (i & (kRing - 1)) * I::BYTES;
#pragma unroll
        for (int k = 0; k < I::LOADS + 1; k++) {
            if (k == I::LOADS && w >= I::MORE) break;
            const int at = min((w + kPWaves * k) * 1024, I::BYTES - 1024);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)(p + at + lane * 16), (lds_p)(slot + at), 16,
                0, 0);
        }
    };

    // What passes from one phase to the next: the dots of a sub-tile (K's bias terms,
    // then each group's), then its weights as operands (f32: by group, high and low parts).
    constexpr int NS = GPD + 1, NP = F32 ? 2 * GPD : 1;
    v16f S[NS];
    h8 P[NP][2];
#pragma unroll
    for (int n = 0; n < NP; n++)
        P[n][0] = P[n][1] = __builtin_bit_cast(h8, uint4{0, 0, 0, 0});

    auto kb_op = [&](int i) {
        return __builtin_bit_cast(b8, ((const uint4 *)(lds + (i & (kRing - 1)) * I::BYTES + I::KB))[lane]);
    };
    auto k_op = [&](int i, int f) {
        return __builtin_bit_cast(h8, ((const uint4 *)(lds + (i & (kRing - 1)) * I::BYTES))[f * 64 + lane]);
    };
    // operand of dims 32f, 16-token step ks
    auto v_op = [&](int i, int f, int ks) {
        return __builtin_bit_cast(h8, ((const uint4 *)(lds + (i & (kRing - 1)) * I::BYTES + I::V))
                                          [((f >> 1) * 4 + (f & 1) * 2 + ks) * 64 + lane]);
    };
    // operands read ahead of their phase: K of sub-tile i, V of i - 1
    b8 KB;
    h8 KF[PF ? GPD * 4 : 1], VF[PF ? GPD * 4 : 1];
    auto read_ahead = [&](int i) {
        if constexpr (PF) {
            KB = kb_op(i);
#pragma unroll
            for (int f = 0; f < GPD * 4; f++) KF[f] = k_op(i, f);
#pragma unroll
            for (int f = 0; f < GPD * 4; f++) VF[f] = v_op(max(i - 1, 0), f >> 1, f & 1);
        }
    };

    // matrix phase of sub-tile i: the dots of i, the weighted sum of sub-tile i - 1
    // (i = 0: of weights 0)
    auto products = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int k = 0; k < 16; k++) S[n][k] = 0.0f;
        const uint8_t *t = lds + (i & (kRing - 1)) * I::BYTES;
        // K's scales (bf16: read ahead of the products, 1193 us for the prompt above against
        // 1212, and 277 against 292 for 4 x 1100 at 5003 of 32Q/4KV, d = 64)
        auto scale_of = [&](int n) __attribute__((always_inline)) {
            return *(const v4f *)((const float *)(t + I::KS) + 32 * (n >> 2) + 8 * (n & 3) + 4 * h);
        };
        v4f ks[F32 ? 1 : 4 * GPD];
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < 4 * GPD; n++) ks[n] = scale_of(n);
            __builtin_amdgcn_sched_barrier(0);
        }
        S[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(PF ? KB : kb_op(i), Q.bias, S[0], 0, 0, 0);
#pragma unroll
        for (int f = 0; f < GPD * 4; f++) {
            const h8 a = PF ? KF[PF ? f : 0] : k_op(i, f);
            const int n = 1 + f / 4;
            if constexpr (F32) S[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, Q.b[f], S[n], 0, 0, 0);
            S[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, Q.a[f], S[n], 0, 0, 0);
        }
        auto weigh = [&](int ks, int f) __attribute__((always_inline)) {
            const h8 v = PF ? VF[PF ? 2 * f + ks : 0] : v_op(max(i - 1, 0), f, ks);
            if constexpr (F32)
                R.O[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, P[2 * (f >> 1) + 1][ks], R.O[f], 0, 0, 0);
            R.O[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, P[F32 ? 2 * (f >> 1) : 0][ks], R.O[f], 0, 0, 0);
        };
        if constexpr (F32)
#pragma unroll
            for (int n = 0; n < D / 16; n++) weigh(n / (D / 32), n % (D / 32));
        // (bf16: the scaling beside V's products, 1251 us against 1290)
#pragma unroll
        for (int n = 0; n < 4 * GPD; n++) {
            const int g = n >> 2, k = n & 3;
            const v4f sc = F32 ? scale_of(n) : ks[F32 ? 0 : n];
#pragma unroll
            for (int e = 0; e < 4; e++)
                S[0][4 * k + e] = fmaf(sc[e], S[1 + g][4 * k + e], S[0][4 * k + e]);
            if constexpr (!F32) weigh(n / (D / 32), n % (D / 32));
        }
    };

    // vector phase: scores, M, weights
    uint32_t poison = 0;                // groups of this row that are NaN
    auto softmax = [&](int i) __attribute__((always_inline)) {
        const uint8_t *t = lds + (i & (kRing - 1)) * I::BYTES;
        const uint32_t bad = F32 ? __builtin_amdgcn_readlane(m_bad, i & 63) : m_bad;
        v16f &s = S[0];
        if constexpr (!F32)
            if (own_rf)
#pragma unroll
                for (int k = 0; k < 16; k++) s[k] *= Q.rf;
        const bool masked = lo + 32 * (i + 1) > vis_min;
        if (masked) {
            const int n = vis - (lo + 32 * i + 4 * h);   // tokens seen from this lane's first on
#pragma unroll
            for (int k = 0; k < 16; k++)
                s[k] = 8 * (k >> 2) + (k & 3) < n ? s[k] : -__builtin_inff();
        }
        if (bad) {
            // rows that see a token with a non-finite V group
            uint32_t seen = 0;
#pragma unroll
            for (int k = 0; k < 16; k++)
                seen |= s[k] != -__builtin_inff() ? 1u << (8 * (k >> 2) + (k & 3)) : 0u;
            seen <<= 4 * h;
            poison |= (seen & mt[i].bad[0] ? 1u : 0u) | (seen & mt[i].bad[1] ? 2u : 0u);
        }
        float p[16];
        R.weights(s, Q, (const float *)(t + I::W), h, p);
        if constexpr (F32) {
#pragma unroll
            for (int g = 0; g < GPD; g++) {
                uint32_t a[8], b[8];
                float cs = 0.0f, ls = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const v4f sc = *(const v4f *)((const float *)(t + I::VS) + 32 * g + 8 * k + 4 * h);
                    const v4f cc = *(const v4f *)((const float *)(t + I::VC) + 32 * g + 8 * k + 4 * h);
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = p[4 * k + e] * sc[e];
                        cs = fmaf(p[4 * k + e], cc[e], cs);
                    }
                    if (g == GPD - 1) {
                        const v4f w4 = *(const v4f *)((const float *)(t + I::W) + 8 * k + 4 * h);
#pragma unroll
                        for (int e = 0; e < 4; e++) ls = fmaf(p[4 * k + e], w4[e], ls);
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const h2 hi2 = pk(x[e], x[e + 2]);
                        a[2 * k + e] = u_of(hi2);
                        b[2 * k + e] = u_of(pk_rest(hi2, x[e], x[e + 2]));
                    }
                }
                R.C[g] += cs;
                R.L += ls;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    P[2 * g][ks] = __builtin_bit_cast(
                        h8, uint4{a[4 * ks], a[4 * ks + 1], a[4 * ks + 2], a[4 * ks + 3]});
                    P[2 * g + 1][ks] = __builtin_bit_cast(
                        h8, uint4{b[4 * ks], b[4 * ks + 1], b[4 * ks + 2], b[4 * ks + 3]});
                }
            }
        } else {
            Soft<D, F32>::operand(p, P[0]);
        }
    };

    // At the end of sub-tile i, every kStep ones: this wave's loads of sub-tiles up to
    // i + kStep are done, behind the barrier every wave's, and the ones before i are
    // read by none any more: their slots are filled again.
    auto sync = [&](int i) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        if (w < I::MORE) wait_loads<(kRing - 1 - 2 * kStep) * (I::LOADS + 1)>();
        else wait_loads<(kRing - 1 - 2 * kStep) * I::LOADS>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int k = kStep - 1; k >= 0; k--) fetch(i + kRing - 1 - k);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (n_i > 0) {
        for (int i = 0; i < kRing - 1 - kStep; i++) fetch(i);
        sync(-1);
        read_ahead(0);
        for (int i = 0; i <= n_i; i++) {
            load_meta(i);
            if (i <= n_w) products(i);
            if (i < n_w) softmax(i);
            if (i % kStep == kStep - 1) sync(i);
            if (i < n_w) read_ahead(i + 1);
        }
        wait_loads<0>();
    }

    const float l = R.finish(poison | __shfl_xor(poison, 32, 64));
    if (r0 + n32 < rows)
        put_rows<D, F32>(row_out(job, c, chunk, tok, head, D, qrow, vec, part), R.O, l, R.M, h, out, part);
}

template <int D, bool F32>
int launch(const eakvd_geom &g, const WinJob &job, int64_t subtiles, const void *q, void *out,
           float *part, uint8_t *img, bool vec, hipStream_t st)
{
    typedef Img<D, F32> I;
    Meta *meta = (Meta *)(img + subtiles * I::BYTES);
    hipLaunchKernelGGL((expand_kernel<D, F32>), dim3((unsigned)subtiles), dim3(64 * 4 * (D / 64)), 0, st,
                       g, job, img, meta, kKScale<F32> / sqrtf((float)D));
    constexpr int bytes = kRing * I::BYTES;
    static_assert(bytes <= 160 * 1024, "LDS");
    const unsigned blocks = (unsigned)job.pre[job.n_seq];
    auto run = [&](auto *kern, std::atomic<uint64_t> &done) {
        const int e = allow_lds((const void *)kern, bytes, done);
        if (e) return e;
        hipLaunchKernelGGL(kern, dim3(blocks), dim3(64 * kPWaves), bytes, st, job, img, meta, q, out, part,
                           (int)vec);
        return (int)hipGetLastError();
    };
    // d = 64 in bf16: where no CU gets two blocks, one that reads ahead (2000 tokens at 30000 of
    // 32Q/4KV, 252 blocks, 711 us against 758); at d = 128 that takes all registers (2048 at
    // 30720 of 32Q/8KV 1231 against 1212)
    static std::atomic<uint64_t> done[2];
    if constexpr (D == 64 && !F32)
        if (blocks <= (unsigned)cu_count()) return run(prompt_kernel<D, F32, true>, done[0]);
    return run(prompt_kernel<D, F32, false>, done[1]);
}

}  // namespace

size_t win_prompt_bytes(int head_dim, bool bf16, int64_t subtiles)
{
    const int per = head_dim == 64 ? (bf16 ? Img<64, false>::BYTES : Img<64, true>::BYTES)
                                   : (bf16 ? Img<128, false>::BYTES : Img<128, true>::BYTES);
    return (size_t)subtiles * (per + sizeof(Meta));
}

int win_prompt(const eakvd_geom &g, const WinJob &job, int64_t subtiles, bool bf16, const void *q,
               void *out, float *part, uint8_t *img, bool vec, hipStream_t st)
{
    if (g.head_dim == 64)
        return bf16 ? launch<64, false>(g, job, subtiles, q, out, part, img, vec, st)
                    : launch<64, true>(g, job, subtiles, q, out, part, img, vec, st);
    return bf16 ? launch<128, false>(g, job, subtiles, q, out, part, img, vec, st)
                : launch<128, true>(g, job, subtiles, q, out, part, img, vec, st);
}
