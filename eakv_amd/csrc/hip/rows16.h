// rows16.h — 16 rows of queries against 16 tokens of packed K on the matrix cores: what the
// attention over pages (paged.hip) and the attention's weights (weights.hip) share.
//
// v_mfma_f32_16x16x32: a lane's operand is row or column lane % 16, 8 values of k-block b =
// lane / 16; its results are column lane % 16, rows 4b + 0..3.  A token's group of 64 dims
// is two operands: bytes 8b + 0..7 of the group, low nibbles (dims 8b + j) and high (32 +
// 8b + j), in nib2's order.
#pragma once

#include "window.h"

namespace {

// One instruction (the compiler puts another before each input that it cannot prove quiet).
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// The maximum of a lane's value and those of the other three lanes of its row.
__device__ __forceinline__ float row_max(float v)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = max3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float v)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16 rows' queries as the columns' operand, one lane's share: row lane % 16, of the
// operand (g, nibble) the dims 64g + 32 nibble + 8b + 0..7, b = lane / 16, in nib2's order.
// Rows are scaled by a power of two to below 2^15; against subnormals (SUB) the high
// nibbles' dims to 2^-4 of that.
template <int D, bool F32, bool SUB>
struct Query {
    h8 a[D / 32];
    h8 b[F32 ? D / 32 : 1];             // f32: low parts
    b8 bias;                            // pieces of the sum of q of group b / 2; b < 2: 1/rf
    float rf;                           // score = dot * rf

    __device__ __forceinline__ void load(const void *q, int64_t at, bool vec, int blk)
    {
        constexpr int GPD = D / 64;
        float x[D / 32][8];
        float top = 0.0f;
#pragma unroll
        for (int f = 0; f < D / 32; f++) {
            const int64_t p = at + (f >> 1) * 64 + (f & 1) * 32 + 8 * blk;
            if constexpr (F32) {
                const float *s = (const float *)q + p;
                if (vec) {
                    const v4f lo = *(const v4f *)s, hi = *(const v4f *)(s + 4);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[f][j] = j < 4 ? lo[j & 3] : hi[j & 3];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[f][j] = s[j];
                }
            } else {
                const uint16_t *s = (const uint16_t *)q + p;
                if (vec) {
                    const uint4 y = *(const uint4 *)s;
                    const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        x[f][j] = __uint_as_float(j & 1 ? ys[j >> 1] & 0xffff0000u : ys[j >> 1] << 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[f][j] = __uint_as_float((uint32_t)s[j] << 16);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[f][j]));
        }
        const int up = 15 - exp_of(row_max(top));
        const float scale = scale2(1.0f, up), less = SUB ? scale * 0x1p-4f : scale;
        float sum[GPD];
#pragma unroll
        for (int f = 0; f < D / 32; f++) {
            const float by = f & 1 ? less : scale;
            float part = 0.0f;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int j = (k >> 1) * 4 + (k & 1);
                const float y0 = x[f][j] * by, y1 = x[f][j + 2] * by;
                part += x[f][j] * scale + x[f][j + 2] * scale;
                const h2 h = pk(y0, y1);
                hi[k] = u_of(h);
                if constexpr (F32) lo[k] = u_of(pk_rest(h, y0, y1));
            }
            a[f] = __builtin_bit_cast(h8, uint4{hi[0], hi[1], hi[2], hi[3]});
            if constexpr (F32) b[f] = __builtin_bit_cast(h8, uint4{lo[0], lo[1], lo[2], lo[3]});
            sum[f >> 1] = f & 1 ? sum[f >> 1] + part : part;
        }
#pragma unroll
        for (int g = 0; g < GPD; g++) sum[g] = row_sum(sum[g]);
        rf = scale2(1.0f, -up);
        __bf16 p1, p2, p3;
        pieces(GPD == 2 && blk >= 2 ? sum[GPD - 1] : sum[0], p1, p2, p3);
        const __bf16 zero = (__bf16)0.0f;
        bias = b8{p1, p2, p3, p1, p2, p1, blk < 2 ? (__bf16)scale : zero, zero};
    }
};

// K's operands of one token's group, from the lane's 8 bytes of it: n - z, or (SUB) the nibbles'
// own bits as subnormals, 2^-24 and 2^-20 of them.
template <bool SUB>
__device__ __forceinline__ void k_operands(const uint2 &x, float z, const NibConst &nc, h8 &lo, h8 &hi)
{
    h2 off_l, off_h;
    if constexpr (!SUB) {
        off_l = nib_off<false>(z, z);
        off_h = nib_off<true>(z, z);
    }
    const uint32_t xs[2] = {x.x, x.y};
    uint32_t a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t y = xs[k >> 1] >> (8 * (k & 1));
        a[k] = SUB ? nib_sub<false>(y) : u_of(nib2<false>(y, off_l, nc));
        b[k] = SUB ? nib_sub<true>(y) : u_of(nib2<true>(y, off_h, nc));
    }
    lo = __builtin_bit_cast(h8, uint4{a[0], a[1], a[2], a[3]});
    hi = __builtin_bit_cast(h8, uint4{b[0], b[1], b[2], b[3]});
}

// K's operands of the bias product for 32 tokens: lane l holds c of token l % 32, group l /
// 32, and stands in its own k-block of its half's operand, nothing in the other's.  e: what is
// added to the token's scores, in units of 1.
__device__ __forceinline__ b8 bias_own(float c, float e, bool first)
{
    __bf16 p1, p2, p3;
    pieces(c, p1, p2, p3);
    const __bf16 none = (__bf16)0.0f;
    return b8{p1, p1, p1, p2, p2, p3, first ? (__bf16)e : none, none};
}
__device__ __forceinline__ void bias_halves(const b8 &own, b8 (&half)[2], int n32)
{
    const __bf16 none = (__bf16)0.0f;
    const b8 zero = {none, none, none, none, none, none, none, none};
    half[0] = n32 < 16 ? own : zero;
    half[1] = n32 < 16 ? zero : own;
}
__device__ __forceinline__ void bias_operands(float c, float e, bool first, b8 (&half)[2], int n32)
{
    bias_halves(bias_own(c, e, first), half, n32);
}

// The dots of one group of 16 tokens with 16 rows.
template <int D, bool F32, bool SUB>
__device__ __forceinline__ v4f group_dots(const h8 &lo, const h8 &hi, const Query<D, F32, SUB> &Q, int g)
{
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (F32) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, Q.b[F32 ? 2 * g : 0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, Q.b[F32 ? 2 * g + 1 : 0], acc, 0, 0, 0);
    }
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, Q.a[2 * g], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, Q.a[2 * g + 1], acc, 0, 0, 0);
}

}  // namespace
