// window.h — what the window attention's kernels share (window.hip, window_draft.hip,
// window_prompt.hip; the mathematics stands in window.hip).
#pragma once

#include <atomic>
#include <type_traits>

#include "common.h"

struct WinJob {
    int n_seq, n_q, n_kv, qpk, layer;
    const uint8_t *base[EAKVD_MAX_BATCH];
    int start[EAKVD_MAX_BATCH];
    int ntok[EAKVD_MAX_BATCH];
    int tok0[EAKVD_MAX_BATCH];          // the window's first row of q and out
    int mc[EAKVD_MAX_BATCH];            // chunks
    int clen[EAKVD_MAX_BATCH];          // tokens per chunk
    int pre[EAKVD_MAX_BATCH + 1];       // blocks before this sequence's
    int lead[EAKVD_MAX_BATCH];          // window tokens of this launch's sequences before it
    int64_t part[EAKVD_MAX_BATCH];      // first partial row
    int64_t part_rows;                  // partial rows in all
    int64_t img[EAKVD_MAX_BATCH];       // expanded sub-tiles before this sequence's
    int nsub[EAKVD_MAX_BATCH];          // expanded sub-tiles of one kv head
};

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kWinTau = 4.0f;        // headroom of the lazy M, log2 units
constexpr float kWinTop = 11.0f;       // M's distance when set: weights below 2^(11 + 4)
constexpr float kMInit = -3.4028234664e38f;
constexpr int kExpLow = -60;           // exponents of q and V below this count as this
// bf16 queries of usual sizes are read as 2^kQUp of their values
constexpr int kQUp = 8;

__device__ __forceinline__ uint32_t u_of(h2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2 h_of(uint32_t v) { return __builtin_bit_cast(h2, v); }
// Two roundings to nearest even.  The empty asm (no instruction that the compiler's
// hazard handling would miss behind a transcendental) holds the result to one rounding:
// the compiler otherwise rounds a product straight to f16 in one place and by way of
// f32 in another, and a pair's low part must be what the high part left.
__device__ __forceinline__ h2 pk(float a, float b)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    uint32_t r = u_of(__builtin_convertvector((f2{a, b}), h2));
    asm("" : "+v"(r));
    return h_of(r);
}
// pk of two transcendentals' results (nothing to fuse with)
__device__ __forceinline__ h2 pk_exp(float a, float b)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector((f2{a, b}), h2);
}
// What pk(a, b) left of a and b, in f16 (the differences are exact in f32).  minus: -1
// in a register, or else the compiler makes a conversion, a difference and another
// conversion of what is one v_fma_mix of each value.
__device__ __forceinline__ h2 pk_rest(h2 hi, float a, float b)
{
    float minus = -1.0f;
    asm("" : "+s"(minus));
    return h2{(_Float16)fmaf((float)hi[0], minus, a), (_Float16)fmaf((float)hi[1], minus, b)};
}

// n - z of the low (HI false) or high nibbles of bytes 0 and 2 of x, exact: the
// nibble is put into the mantissa of 1024 (its lowest bits) or of 64 (four bits up)
// and 1024 + z or 64 + z taken off.  off: minus that, of the two bytes; c: the
// exponents, in registers, so that mask and exponent are one instruction.
struct NibConst {
    uint32_t lo = 0x64006400u, hi = 0x54005400u;
    __device__ __forceinline__ void hold() { asm("" : "+v"(lo), "+v"(hi)); }
};
template <bool HI>
__device__ __forceinline__ h2 nib2(uint32_t x, h2 off, const NibConst &c)
{
    return h_of(HI ? (x & 0x00f000f0u) | c.hi : (x & 0x000f000fu) | c.lo) + off;
}
// the offsets of z
template <bool HI>
__device__ __forceinline__ h2 nib_off(float z0, float z1)
{
    constexpr float k = HI ? -64.0f : -1024.0f;
    return pk(k - z0, k - z1);
}

// The nibbles as they stand, as subnormal f16: n * 2^-24 (low) or n * 2^-20 (high).
// The matrix cores' products with them are exact, their sums are not: terms are aligned as if such an
// operand were 2^-14, so that sums of 32 terms lose up to 2^-11.4 (low) and 2^-15.6 (high) of one step
// (n = 1) times the largest other operand, one term alone nothing (measured; with n - z, which is no
// subnormal, 2^-24 of the terms' sum).
template <bool HI>
__device__ __forceinline__ uint32_t nib_sub(uint32_t x)
{
    return x & (HI ? 0x00f000f0u : 0x000f000fu);
}

// z: the nibble whose value is nearest 0, so that (n - z)*s and c = b + z*s are of
// the size of the value and cancel nothing (a group with an outlier has b and
// s far above its other values).
__device__ __forceinline__ float zero_nibble(float s, float b)
{
    const float z = __builtin_rintf(-b * __builtin_amdgcn_rcpf(s));
    return fminf(fmaxf(z, 0.0f), 15.0f);
}

__device__ __forceinline__ int exp_of(float a)
{
    const int e = (int)(__float_as_uint(a) >> 23) - 126;     // a < 2^e
    return e < kExpLow ? kExpLow : e;
}
// What a token's exponent is taken of, a group's scale and largest value given: f32, the
// scale, or 2^-24 of the value where that is more (weights times biases stay in range).
template <bool F32>
__device__ __forceinline__ float v_size(float s, float top)
{
    return F32 ? fmaxf(fabsf(s), top * 0x1p-24f) : top;
}
// x * 2^e, one rounding, for any e
__device__ __forceinline__ float scale2(float x, int e)
{
    return __builtin_amdgcn_ldexpf(x, e);
}

// Three bf16 pieces of x, together 24 bits.
__device__ __forceinline__ void pieces(float x, __bf16 &a, __bf16 &b, __bf16 &c)
{
    a = (__bf16)x;
    const float r = __fsub_rn(x, (float)a);
    b = (__bf16)r;
    c = (__bf16)__fsub_rn(r, (float)b);
}

// A lane's share of a row of q as it stands in memory: the 8 consecutive dims of each
// operand (QOp).  Rows are 16-byte aligned (vec) or read by elements.
template <int D, bool F32>
struct QRaw {
    uint4 x[F32 ? D / 8 : D / 16];
};

template <int D, bool F32>
__device__ __forceinline__ void load_q(QRaw<D, F32> &r, const void *q, int64_t qrow, bool vec, int h)
{
    constexpr int W = F32 ? 2 : 1;                   // 16-byte pieces of an operand
#pragma unroll
    for (int f = 0; f < D / 16; f++) {
        const int64_t at = qrow + (f >> 2) * 64 + 32 * (f & 1) + 16 * h + 8 * ((f >> 1) & 1);
#pragma unroll
        for (int j = 0; j < W; j++) {
            if (vec) {
                r.x[W * f + j] = *(const uint4 *)((const uint8_t *)q + at * (F32 ? 4 : 2) + 16 * j);
            } else if constexpr (F32) {
                const uint32_t *p = (const uint32_t *)q + at + 4 * j;
                r.x[W * f + j] = uint4{p[0], p[1], p[2], p[3]};
            } else {
                const uint16_t *p = (const uint16_t *)q + at;
                r.x[f] = uint4{p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16,
                               p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16};
            }
        }
    }
}

__device__ __forceinline__ uint32_t bf16_bits(float x)
{
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x);
}

template <bool F32>
__device__ __forceinline__ void store4(void *out, int64_t at, bool vec, const float *o)
{
    if constexpr (F32) {
        float *p = (float *)out + at;
        if (vec) *(v4f *)p = v4f{o[0], o[1], o[2], o[3]};
        else
            for (int j = 0; j < 4; j++) p[j] = o[j];
    } else {
        uint16_t *p = (uint16_t *)out + at;
        if (vec)
            *(uint2 *)p = uint2{bf16_bits(o[0]) | bf16_bits(o[1]) << 16,
                                bf16_bits(o[2]) | bf16_bits(o[3]) << 16};
        else
            for (int j = 0; j < 4; j++) p[j] = (uint16_t)bf16_bits(o[j]);
    }
}

// The maximum of a lane's value and the other half's (lane ^ 32), in both.
__device__ __forceinline__ float half_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A row's query as the columns' operand of S^T = K Q^T, one lane's share: operand
// (g, octet o, nibble n) of half h holds dims 64g + 32n + 16h + 8o + 0..7 in nib2's
// order (0 2 1 3 4 6 5 7).  The row is scaled by a power of two to below 2^15; bf16 rows
// of usual sizes all by the same one, so that their dots need no factor of their own.
// SUB: against nib_sub's operands: the high nibbles' dims 2^-4 of that; the dots come
// out 2^-24 of theirs, which K's scales make up for (in rf those 2^24 would pass f32's
// range for queries from 2^121 on).
template <int D, bool F32>
struct QOp {
    h8 a[D / 16];                       // f16, high parts
    h8 b[F32 ? D / 16 : 1];             // f32 queries: low parts
    b8 bias;                            // half h: pieces of group h's sum of q; two more
    float rf;                           // score = dot * rf, a power of two
};

// What K's scales and (bf16: against sums of q at 2^-24) biases carry beside 1/sqrt(d).
template <bool F32>
constexpr float kKScale = F32 ? EAKV_LOG2E : EAKV_LOG2E * (1.0f / (1 << kQUp));
template <bool F32>
constexpr float kKBias = F32 ? 1.0f : 0x1p24f;

// K's operand of the bias product, token's half h: c's pieces against the query's, then
// 1 1 (h = 0) or 1 and the exponent of the token's V.
__device__ __forceinline__ b8 k_bias(float c, int e, int h)
{
    __bf16 p1, p2, p3;
    const __bf16 one = (__bf16)1.0f;
    pieces(c, p1, p2, p3);
    return b8{p1, p1, p1, p2, p2, p3, one, h ? (__bf16)(float)e : one};
}

template <int D, bool F32, bool SUB>
__device__ __forceinline__ void build_q(QOp<D, F32> &Q, const QRaw<D, F32> &raw, int h)
{
    constexpr int GPD = D / 64;
    auto dim = [&](int f, int j) {                   // dim j of operand f
        if constexpr (F32) {
            const uint4 &x = raw.x[2 * f + (j >> 2)];
            return __uint_as_float((j & 3) == 0 ? x.x : (j & 3) == 1 ? x.y : (j & 3) == 2 ? x.z : x.w);
        } else {
            const uint4 &x = raw.x[f];
            const uint32_t y = (j >> 1) == 0 ? x.x : (j >> 1) == 1 ? x.y : (j >> 1) == 2 ? x.z : x.w;
            return __uint_as_float(j & 1 ? y & 0xffff0000u : y << 16);
        }
    };
    float top = 0.0f;
#pragma unroll
    for (int f = 0; f < D / 16; f++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(dim(f, j)));
    top = half_max(top);
    // q' = q * 2^up
    int up = 15 - exp_of(top);
    if (!F32 && (top == 0.0f || (top >= 0x1p-7f && top < 0x1p7f))) up = kQUp;
    const float scale = scale2(1.0f, up), less = SUB ? scale * 0x1p-4f : scale;
    float qs[GPD];
#pragma unroll
    for (int g = 0; g < GPD; g++) {
        v16f sum;                                    // of the group's 64 dims, in every register
#pragma unroll
        for (int k = 0; k < 16; k++) sum[k] = 0.0f;
#pragma unroll
        for (int f = 4 * g; f < 4 * g + 4; f++) {
            const float by = f & 1 ? less : scale;
            const _Float16 one = (_Float16)(SUB && (f & 1) ? 16.0f : 1.0f);
            const h8 ones = h8{one, one, one, one, one, one, one, one};
            uint32_t a[4], b[4];
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const int j = (p >> 1) * 4 + (p & 1);
                const float y0 = dim(f, j) * by, y1 = dim(f, j + 2) * by;
                const h2 hi2 = pk(y0, y1);
                a[p] = u_of(hi2);
                if constexpr (F32) b[p] = u_of(pk_rest(hi2, y0, y1));
            }
            Q.a[f] = __builtin_bit_cast(h8, uint4{a[0], a[1], a[2], a[3]});
            sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones, Q.a[f], sum, 0, 0, 0);
            if constexpr (F32) {
                Q.b[f] = __builtin_bit_cast(h8, uint4{b[0], b[1], b[2], b[3]});
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones, Q.b[f], sum, 0, 0, 0);
            }
        }
        qs[g] = sum[0];
    }
    const int down = (F32 ? 0 : kQUp) - up;
    Q.rf = scale2(1.0f, down);
    // half h of the bias product's 16 terms: group h's sum of q in pieces, against K's
    // c1 c1 c1 c2 c2 c3; then pieces of minus the reference point (hold_ref) against 1, and,
    // last, 1/rf against the exponent of the token's V
    __bf16 p1, p2, p3;
    const float z = GPD == 2 ? (h ? qs[GPD - 1] : qs[0]) : (h ? 0.0f : qs[0]);
    pieces(z * (1.0f / kKBias<F32>), p1, p2, p3);
    const __bf16 zero = (__bf16)0.0f;
    Q.bias = b8{p1, p2, p3, p1, p2, p1, zero, h ? (__bf16)scale2(1.0f, -down) : zero};
}

// bf16: the bias product takes m off the scores from here on; what it does take off is
// returned (pieces below bf16's normal range are dropped).
template <int D>
__device__ __forceinline__ float hold_ref(QOp<D, false> &Q, float m, int h)
{
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(Q.rf));
    __bf16 p[3];
    pieces(-m * inv, p[0], p[1], p[2]);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 3; i++) {
        p[i] = fabsf((float)p[i]) < 0x1p-126f ? (__bf16)0.0f : p[i];
        sum += (float)p[i];
    }
    Q.bias[6] = h ? p[2] : p[0];
    Q.bias[7] = h ? Q.bias[7] : p[1];
    return -sum * Q.rf;
}

// The running softmax of a lane's row.
template <int D, bool F32>
struct Soft {
    v16f O[D / 32];
    float M = kMInit, L = 0.0f, C[D / 64];
    float high = -__builtin_inff();     // bf16: M moves when a score passes this

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int f = 0; f < D / 32; f++)
#pragma unroll
            for (int k = 0; k < 16; k++) O[f][k] = 0.0f;
#pragma unroll
        for (int g = 0; g < D / 64; g++) C[g] = 0.0f;
    }
    // M rises by -d.  L by halves of it: where V's sizes differ by some 2^126 the rest of O is
    // nothing beside what is to come, but the rest of L may be most of it.
    __device__ __forceinline__ void rescale(float d)
    {
        const float al = __builtin_amdgcn_exp2f(d), half = __builtin_amdgcn_exp2f(0.5f * d);
        L = L * half * half;
#pragma unroll
        for (int f = 0; f < D / 32; f++)
#pragma unroll
            for (int k = 0; k < 16; k++) O[f][k] *= al;
        if constexpr (F32)
#pragma unroll
            for (int g = 0; g < D / 64; g++) C[g] *= al;
    }
    // s: the masked scores (log2) of 16 tokens with their V's exponents added, in units
    // of rf and, bf16, less M.  On return the weights, 2^e of the softmax's.  w: 2^-e, for
    // L (f32: which the caller adds up beside V's other sums, 121 us against 127 for 8
    // drafts of 8 sequences at 32768 of 32Q/8KV).
    // M follows the largest weight that the row sees: rows move it one by one, so that
    // no row's result depends on another's tokens.
    __device__ __forceinline__ void weights(v16f &s, QOp<D, F32> &Q, const float *w, int h, float *p)
    {
        // (read here, their latency passes behind the maximum)
        v4f w4[4];
        if constexpr (!F32) {
#pragma unroll
            for (int k = 0; k < 4; k++) w4[k] = *(const v4f *)(w + 8 * k + 4 * h);
            __builtin_amdgcn_sched_barrier(0);
        }
        float top = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
        for (int k = 3; k < 16; k++) top = fmaxf(top, s[k]);
        top = half_max(top);
        if constexpr (F32) {
            const float need = fmaf(top, Q.rf, -kWinTop);
            if (__ballot(need > M + kWinTau) != 0) {
                const float mn = need > M + kWinTau ? need : M;
                rescale(M - mn);
                M = mn;
            }
#pragma unroll
            for (int k = 0; k < 16; k++) p[k] = __builtin_amdgcn_exp2f(fmaf(s[k], Q.rf, -M));
        } else {
            if (__ballot(top > high) != 0) {
                // (before a row's first tokens nothing is taken off and M is not set)
                const bool first = high < 0.0f, move = top > high;
                const float old = first ? 0.0f : M;
                const float mn = hold_ref(Q, move ? old + (top - kWinTop) : old, h);
                const float by = mn - old;
                rescale(first ? -__builtin_inff() : -by);
#pragma unroll
                for (int k = 0; k < 16; k++) s[k] -= by;
                M = move ? mn : M;
                high = move ? kWinTop + kWinTau : high;
            }
#pragma unroll
            for (int k = 0; k < 16; k++) p[k] = __builtin_amdgcn_exp2f(s[k]);
        }
        if constexpr (!F32) {
            float sum[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    sum[e] = k ? fmaf(p[4 * k + e], w4[k][e], sum[e]) : p[e] * w4[0][e];
            L += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
    }
    // After the last token: O whole (NaN in the groups that are named) and the row's L.
    __device__ __forceinline__ float finish(uint32_t nan_groups)
    {
        if constexpr (F32) {
#pragma unroll
            for (int g = 0; g < D / 64; g++) {
                const float cs = C[g] + __shfl_xor(C[g], 32, 64);
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int k = 0; k < 16; k++) O[2 * g + n][k] += cs;
            }
        } else {
#pragma unroll
            for (int f = 0; f < D / 32; f++)
#pragma unroll
                for (int k = 0; k < 16; k++) O[f][k] *= 0x1p-15f;          // V's operands carried 2^15
        }
        if (nan_groups)
#pragma unroll
            for (int f = 0; f < D / 32; f++)
                if (nan_groups >> (f >> 1) & 1)
#pragma unroll
                    for (int k = 0; k < 16; k++) O[f][k] = __builtin_nanf("");
        return L + __shfl_xor(L, 32, 64);
    }
    // The 16 weights in operand order for bf16 queries.
    __device__ __forceinline__ static void operand(const float *p, h8 (&P)[2])
    {
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const float *pp = p + 8 * ks;
            P[ks] = __builtin_bit_cast(h8, uint4{u_of(pk_exp(pp[0], pp[2])), u_of(pk_exp(pp[1], pp[3])),
                                                 u_of(pk_exp(pp[4], pp[6])), u_of(pk_exp(pp[5], pp[7]))});
        }
    }
};

// The row that a lane writes: final outputs (mc == 1) or its chunk's partial.
struct RowOut {
    int64_t at;                         // first value, in out or in part
    float *ml;                          // the partial's M and l, or NULL
    bool final, vec;
};

__device__ __forceinline__ RowOut row_out(const WinJob &job, int c, int chunk, int tok, int head,
                                          int D, int64_t qrow, bool vec, float *part)
{
    RowOut r;
    r.final = job.mc[c] == 1;
    r.vec = vec;
    r.at = qrow;
    r.ml = nullptr;
    if (!r.final) {
        const int64_t prow = job.part[c] + (int64_t)chunk * job.ntok[c] * job.n_q +
                             (int64_t)tok * job.n_q + head;
        r.at = prow * D;
        r.ml = part + job.part_rows * D + prow * 2;
    }
    return r;
}

// Four values of a row: dims d..d+3, unscaled.  (A partial with l = 0 has no O.)
template <bool F32>
__device__ __forceinline__ void put4(const RowOut &r, int d, const float *o, float l, void *out,
                                     float *part)
{
    if (r.final) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const float o4[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        store4<F32>(out, r.at + d, r.vec, o4);
    } else if (l != 0.0f) {
        *(v4f *)(part + r.at + d) = v4f{o[0], o[1], o[2], o[3]};
    }
}

// A wave's whole rows: o[f][i] holds dim 32f + 8(i/4) + 4h + i%4.
template <int D, bool F32>
__device__ __forceinline__ void put_rows(const RowOut &r, const v16f *o, float l, float m, int h,
                                         void *out, float *part)
{
#pragma unroll
    for (int f = 0; f < D / 32; f++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float o4[4] = {o[f][4 * k], o[f][4 * k + 1], o[f][4 * k + 2], o[f][4 * k + 3]};
            put4<F32>(r, 32 * f + 8 * k + 4 * h, o4, l, out, part);
        }
    if (r.ml && h == 0) {
        r.ml[0] = m;
        r.ml[1] = l;
    }
}

// Joins the WT waves of a block that hold the same rows (O, l, M of other tokens)
// through LDS and writes the rows: every wave its WT-th part of the dims.  All waves of
// the block call it, with kJoinBytes of LDS.  (In a tree of log2(WT) steps instead, a
// draft of 4 tokens at 500 of 32Q/8KV took 14.0 us against 12.8.)
template <int D>
constexpr size_t kJoinBytes = (size_t)8 * (D / 2 + 2) * 64 * 4;

template <int D, bool F32, int WT>
__device__ __forceinline__ void join_put(float *lds, int wt, int lane,
                                         const v16f *o, float l, float m, bool live, const RowOut &r,
                                         void *out, float *part)
{
    constexpr int OW = D / 2 * 64, N = D / 2 / WT;       // floats of a wave's O; of a lane's part
    float *ml = lds + 8 * OW;
    const int h = lane >> 5;
    __syncthreads();
    {
        v4f *po = (v4f *)(lds + (size_t)wt * OW) + lane;
#pragma unroll
        for (int f = 0; f < D / 32; f++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                po[(f * 4 + i) * 64] = v4f{o[f][4 * i], o[f][4 * i + 1], o[f][4 * i + 2], o[f][4 * i + 3]};
        ml[wt * 128 + lane] = m;
        ml[wt * 128 + 64 + lane] = l;
    }
    __syncthreads();
    float a[WT], mm = kMInit, ll = 0.0f;
#pragma unroll
    for (int t = 0; t < WT; t++) {
        a[t] = ml[t * 128 + lane];
        mm = fmaxf(mm, a[t]);
    }
#pragma unroll
    for (int t = 0; t < WT; t++) {
        // (l by halves, as Soft::rescale)
        const float half = __builtin_amdgcn_exp2f(0.5f * (a[t] - mm));
        a[t] = __builtin_amdgcn_exp2f(a[t] - mm);
        ll = fmaf(half * ml[t * 128 + 64 + lane], half, ll);
    }
#pragma unroll
    for (int k = 0; k < N / 4; k++) {
        const int e = wt * N + 4 * k;                    // register f * 16 + i
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < WT; t++) {
            const v4f po = ((const v4f *)(lds + (size_t)t * OW))[(e >> 2) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = fmaf(a[t], po[j], x[j]);
        }
        if (live) put4<F32>(r, 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * h, x, ll, out, part);
    }
    if (live && r.ml && h == 0 && wt == 0) {
        r.ml[0] = mm;
        r.ml[1] = ll;
    }
}

// The sequence of block b: the last one whose first block is not behind it.
__device__ __forceinline__ int seq_of(const int *pre, int n_seq, int b, int lane)
{
    if (n_seq == 1) return 0;
    // (pre has EAKVD_MAX_BATCH entries at least)
    const bool past = lane > 0 && lane < n_seq && b >= pre[lane < EAKVD_MAX_BATCH ? lane : 0];
    return (int)__popcll(__ballot(past));
}

// Lets a kernel use `bytes` of dynamic LDS on the current device, once per device
// (`done`: the devices it was done on, of one kernel).
inline int allow_lds(const void *kern, size_t bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit & done.load(std::memory_order_relaxed)) return 0;
    e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return (int)e;
}

// s_waitcnt vmcnt(N) alone (gfx9 encoding)
template <int N>
__device__ __forceinline__ void wait_loads()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

}  // namespace

// Attends without scratch but for the chunks' partials (window_draft.hip); a chunk is a
// whole number of tiles of kDraftTile tokens.
constexpr int kDraftTile = 256;
int win_draft(const eakvd_geom &g, const WinJob &job, bool bf16, const void *q, const uint64_t *tree,
              void *out, float *part, bool vec, hipStream_t st);
// Expands K and V of the sequences' kv heads into `img` and attends
// (window_prompt.hip).  img: win_prompt_bytes() of device scratch; job.img: each
// sequence's first sub-tile there.
size_t win_prompt_bytes(int head_dim, bool bf16, int64_t subtiles);
int win_prompt(const eakvd_geom &g, const WinJob &job, int64_t subtiles, bool bf16, const void *q,
               void *out, float *part, uint8_t *img, bool vec, hipStream_t st);
