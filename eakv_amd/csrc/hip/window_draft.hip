// window_draft.hip — the window attention of few rows per kv head (some drafted tokens),
// where reading the packed planes once is the work: the mathematics of window.hip with
// nothing shared between waves.
//
// A block has 32 rows; its 8 waves take 32-token sub-tiles in turn and join at the end.
// Each wave
//   - keeps kAhead sub-tiles in flight, by buffer loads whose tile offset is scalar:
//     K's bytes and the scales to registers, V's bytes to LDS;
//   - makes K's operands in registers (a lane's bytes are its operand's);
//   - reads V's bytes back transposed (ds_read_b64_tr_b8: 8 tokens of a byte column
//     per lane) and makes its operands in registers, the tokens' scales from LDS, in
//     operand order;
// so no operand passes through LDS as f16, and no wave waits for another.
//
// Bound by vector instructions: per 32 tokens x 32 rows at d = 128 a wave issues about 390
// (f32 540) beside 17 (33) matrix products and 5 KB of loads.  8 sequences of 8 tokens
// at 32768 of 32Q/8KV (32 rows, 336 MB): bf16 75 us in the kernel, 4.5 TB/s; f32 107-125.
// Fewer rows cost the same: one bf16 token each 74.
// Rows beyond 32 read the planes again, out of the caches: a block of 64 rows with
// shared operands in LDS was slower at most sizes up to 512 rows (64 rows of 8 at 20000 of
// 64Q/8KV bf16 158 against 164 us, but 192 rows of 6: 350 against 274; 64 of 4 at 4000,
// d = 64: 31 against 24).  For small contexts a block's way bounds it: 1.4 us of
// arguments and addresses, 2.4 for q, 2.7 for a sub-tile, 2 for the join.
#include "window.h"

namespace {

constexpr int kDWaves = 8;
static_assert(kDraftTile == 32 * kDWaves, "a sub-tile for each wave");
// Slots of V's bytes.  bf16: two sub-tiles are in flight while one is worked on.  f32: the
// next one is asked for as soon as K's registers are free, in the middle of one.
template <bool F32>
constexpr int kAheadOf = F32 ? 2 : 3;

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i *lds_v2i;
typedef __attribute__((address_space(3))) void *lds_v;

template <int D, bool F32>
struct __align__(16) DraftLds {
    static constexpr int GPD = D / 64, kAhead = kAheadOf<F32>;
    uint8_t v[kAhead][32 * 32 * GPD];   // V's bytes: rows of 32 GPD, their 16-byte units swizzled
    float ks[GPD][32];                  // K's scales
    float w[32];                        // 2^-e, e the exponent of a token's V
    float vs[F32 ? GPD : 1][32];        // f32: V's scales and biases, 2^-e of them
    float vc[F32 ? GPD : 1][32];
    // of V's operand (g, 16-token step, h), 8 tokens in operand order: -(1024 + z),
    // -(64 + z); bf16: scales and biases in f16, 2^(15 - e) of them
    _Float16 zl[GPD][2][2][8], zh[GPD][2][2][8];
    _Float16 s16[F32 ? 1 : GPD][2][2][8], c16[F32 ? 1 : GPD][2][2][8];
};

struct Stage {
    uint4 k[2];
    float ks, kb, vs, vb;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, int64_t bytes)
{
    // dword3 0x00020000: raw 32-bit buffer; reads beyond `bytes` return 0
    const int64_t most = 0xfffffff0ll;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0,
                                             (int)(uint32_t)(bytes < most ? bytes : most), 0x00020000);
}

// the unit permutation of token row t
template <int GPD>
__device__ __forceinline__ int swz(int t)
{
    return GPD == 2 ? (t >> 2) & 3 : (t >> 3) & 1;
}

template <int D, bool F32>
__global__ __launch_bounds__(64 * kDWaves, 2) void draft_kernel(eakvd_geom geo, WinJob job,
                                                                const void *q, const uint64_t *tree,
                                                                void *out, float *part, float ksc,
                                                                int vec)
{
    constexpr int GPD = D / 64, RB = 32 * GPD, kAhead = kAheadOf<F32>;
    constexpr int kStages = F32 ? 1 : kAhead;
    typedef DraftLds<D, F32> Lds;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    Lds &S = ((Lds *)lds)[w];
    const int n32 = lane & 31, h = lane >> 5;

    const int c = seq_of(job.pre, job.n_seq, (int)blockIdx.x, lane);
    int rem = (int)blockIdx.x - job.pre[c];
    const int kvh = rem % job.n_kv;
    rem /= job.n_kv;
    const int m = job.ntok[c], start = job.start[c], qpk = job.qpk;
    // row blocks of one kv head and chunk run side by side and share its planes in the caches
    const int rows = m * qpk, n_rb = (rows + 31) / 32;
    const int chunk = rem / n_rb, r0 = 32 * (rem - chunk * n_rb);
    const int t_end = start + (tree ? m : (min(r0 + 32, rows) - 1) / qpk + 1);
    const int lo = chunk * job.clen[c];
    const int hi = t_end - lo > job.clen[c] ? lo + job.clen[c] : t_end;

    const int row = min(r0 + n32, rows - 1);
    const int tok = row / qpk, head = kvh * qpk + row - tok * qpk;
    const int64_t qrow = ((int64_t)(job.tok0[c] + tok) * job.n_q + head) * D;
    const int vis = start + tok + 1;
    const int vis_min = tree ? start : start + r0 / qpk + 1;
    const uint64_t word = tree ? tree[job.tok0[c] + tok] : 0;

    // ---- the planes of this kv head from token lo on
    const Planes K = planes_of(geo, job.base[c], job.layer, 0);
    const Planes V = planes_of(geo, job.base[c], job.layer, 1);
    const int64_t g0 = (int64_t)kvh * geo.gph + (int64_t)lo * GPD;
    const int64_t room = (int64_t)(geo.max_seq_len - lo) * GPD;          // groups
    const auto rkw = rsrc(K.w + g0 * 32, room * 32), rvw = rsrc(V.w + g0 * 32, room * 32);
    const auto rks = rsrc(K.s + g0, room * 4), rkb = rsrc(K.b + g0, room * 4);
    const auto rvs = rsrc(V.s + g0, room * 4), rvb = rsrc(V.b + g0, room * 4);
    // K: token n32, bytes 16h of each group; scales: token n32, group h
    const int ok = n32 * RB + 16 * h;
    const int os = (n32 * GPD + (GPD == 2 ? h : 0)) * 4;
    // V: 16-byte unit `lane` of a slot's first KB is unit (lane % UPT) of row lane / UPT
    constexpr int UPT = RB / 16;
    const int vt = lane / UPT, ov = vt * RB + 16 * ((lane % UPT) ^ swz<GPD>(vt));
    constexpr int NV = RB * 32 / 1024;
    constexpr int kLoads = NV + GPD + 4;
    auto load = [&](int i, Stage &s) __attribute__((always_inline)) {
        const int t = __builtin_amdgcn_readfirstlane(32 * (w + kDWaves * i));
        uint8_t *slot = S.v[i % kAhead];
#pragma unroll
        for (int j = 0; j < NV; j++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rvw, (lds_v)(slot + 1024 * j), 16, ov, t * RB + 1024 * j,
                                                     0, 2);
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b128(rkw, ok + 32 * g, t * RB, 2);
            s.k[g] = uint4{x[0], x[1], x[2], x[3]};
        }
        const int ts = t * GPD * 4;
        s.ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rks, os, ts, 2));
        s.kb = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rkb, os, ts, 2));
        s.vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rvs, os, ts, 2));
        s.vb = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rvb, os, ts, 2));
    };
    // transposed reads of V: lane supplies 8 bytes of row j = lane%16 / 2 of its 16-lane
    // group's 8 tokens and gets 8 tokens of byte column n32
    const int jr = (lane & 15) >> 1, trow = 8 * (jr >> 2) + 4 * h + (jr & 3);
    int vrd[GPD];
#pragma unroll
    for (int g = 0; g < GPD; g++)
        vrd[g] = trow * RB + 16 * ((2 * g + ((lane >> 4) & 1)) ^ swz<GPD>(trow)) + 8 * (lane & 1);
    // where this lane's token (n32, group h) stands among V's operands
    const int pj = 4 * ((n32 >> 3) & 1) + (n32 & 3);
    const int pos = (pj & 4) | ((pj & 1) << 1) | ((pj >> 1) & 1);
    const int p_step = n32 >> 4, p_half = (n32 >> 2) & 1;
    const bool owner = GPD == 2 || h == 0;

    // this wave's sub-tiles; the first loads are on their way while Q is made, behind Q's
    // own (loads behind the last sub-tile stay within the planes or return 0)
    QRaw<D, F32> raw;
    load_q<D, F32>(raw, q, qrow, vec, h);
    const int n_sub = hi > lo ? (hi - lo + 31) / 32 : 0;
    const int n_i = n_sub > w ? (n_sub - w + kDWaves - 1) / kDWaves : 0;
    Stage st[kStages];
    if (n_i > 0)
#pragma unroll
        for (int k = 0; k < kAhead - 1; k++) load(k, st[k]);

    QOp<D, F32> Q;
    build_q<D, F32, !F32>(Q, raw, h);
    const bool own_rf = F32 || __ballot(Q.rf != 1.0f) != 0;
    Soft<D, F32> R;
    R.clear();
    uint32_t poison = 0;
    NibConst nc;
    nc.hold();

    auto consume = [&](int i, Stage &st) __attribute__((always_inline)) {
        const int t0 = lo + 32 * (w + kDWaves * i);
        // tokens behind the last have no part in this (their bytes may be anything)
        const bool live = t0 + n32 < t_end;
        // (bf16: K's nibbles as they stand, z = 0 and 2^-24 of their values)
        const float zk = F32 ? zero_nibble(st.ks, st.kb) : 0.0f;
        const float ck = (F32 ? fmaf(zk, st.ks, st.kb) : st.kb) * (ksc * kKBias<F32>);
        // (a non-finite group counts as zeros and makes the rows that see it NaN)
        const float va = fmaxf(fabsf(st.vb), fabsf(fmaf(15.0f, st.vs, st.vb)));
        const bool fin = va < __builtin_inff() && st.vs == st.vs;
        const uint64_t bad = __ballot(live && !fin);
        const float vs = live && fin ? st.vs : 0.0f, vb = live && fin ? st.vb : 0.0f;
        const float zv = zero_nibble(vs, vb), cv = fmaf(zv, vs, vb);
        // the token's exponent, of both groups
        const float x = live && fin ? v_size<F32>(vs, va) : 0.0f;
        const int ev = exp_of(GPD == 2 ? half_max(x) : x);
        // ---- scales to LDS
        S.w[n32] = scale2(1.0f, -ev);
        if (owner) S.ks[GPD == 2 ? h : 0][n32] = st.ks * (F32 ? ksc : ksc * 0x1p24f);
        if (owner) {
            S.zl[GPD == 2 ? h : 0][p_step][p_half][pos] = (_Float16)(-1024.0f - zv);
            S.zh[GPD == 2 ? h : 0][p_step][p_half][pos] = (_Float16)(-64.0f - zv);
        }
        if constexpr (F32) {
            if (owner) {
                S.vs[GPD == 2 ? h : 0][n32] = scale2(vs, -ev);
                S.vc[GPD == 2 ? h : 0][n32] = scale2(cv, -ev);
            }
        } else {
            if (owner) {
                S.s16[GPD == 2 ? h : 0][p_step][p_half][pos] = (_Float16)scale2(vs, 15 - ev);
                S.c16[GPD == 2 ? h : 0][p_step][p_half][pos] = (_Float16)scale2(cv, 15 - ev);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // ---- scores
        v16f s;
#pragma unroll
        for (int k = 0; k < 16; k++) s[k] = 0.0f;
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_bias(owner ? ck : 0.0f, ev, h), Q.bias, s, 0, 0, 0);
        float zg[2] = {zk, zk};
        if constexpr (F32 && GPD == 2) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(zk), __float_as_uint(zk), false,
                                                            false);
            zg[0] = __uint_as_float(r[0]);
            zg[1] = __uint_as_float(r[1]);
        }
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            const h2 off_l = nib_off<false>(zg[g], zg[g]), off_h = nib_off<true>(zg[g], zg[g]);
            const uint32_t x[4] = {st.k[g].x, st.k[g].y, st.k[g].z, st.k[g].w};
            v16f acc;
#pragma unroll
            for (int k = 0; k < 16; k++) acc[k] = 0.0f;
#pragma unroll
            for (int o = 0; o < 2; o++) {
                uint32_t a[4], b[4];
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint32_t x0 = x[2 * o + d], x1 = x0 >> 8;
                    a[2 * d] = F32 ? u_of(nib2<false>(x0, off_l, nc)) : nib_sub<false>(x0);
                    a[2 * d + 1] = F32 ? u_of(nib2<false>(x1, off_l, nc)) : nib_sub<false>(x1);
                    b[2 * d] = F32 ? u_of(nib2<true>(x0, off_h, nc)) : nib_sub<true>(x0);
                    b[2 * d + 1] = F32 ? u_of(nib2<true>(x1, off_h, nc)) : nib_sub<true>(x1);
                }
                const h8 ka = __builtin_bit_cast(h8, uint4{a[0], a[1], a[2], a[3]});
                const h8 kb = __builtin_bit_cast(h8, uint4{b[0], b[1], b[2], b[3]});
                const int f = g * 4 + 2 * o;
                if constexpr (F32) {
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, Q.b[f], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kb, Q.b[f + 1], acc, 0, 0, 0);
                }
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, Q.a[f], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kb, Q.a[f + 1], acc, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const v4f sc = *(const v4f *)&S.ks[g][8 * k + 4 * h];
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * k + e] = fmaf(sc[e], acc[4 * k + e], s[4 * k + e]);
            }
        }
        // ---- V's bytes, transposed (their loads are done: K's of the same sub-tile,
        // issued behind them, are)
        v2i vx[GPD][2];
        const uint8_t *slot = S.v[i % kAhead];
#pragma unroll
        for (int g = 0; g < GPD; g++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
                vx[g][ks] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(slot + vrd[g] + 16 * ks * RB));
        if constexpr (F32) {
            __builtin_amdgcn_sched_barrier(0);
            load(i + 1, st);
            __builtin_amdgcn_sched_barrier(0);
        }
        // ---- softmax
        if constexpr (!F32)
            if (own_rf)
#pragma unroll
                for (int k = 0; k < 16; k++) s[k] *= Q.rf;
        const bool masked = t0 + 32 > vis_min;
        if (masked) {
            const int d0 = t0 + 4 * h - start;           // this lane's first token, of the window
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const int d = d0 + 8 * (k >> 2) + (k & 3);
                const bool see = tree ? d < 0 || (d < m && ((word >> (d & 63)) & 1)) : d + start < vis;
                s[k] = see ? s[k] : -__builtin_inff();
            }
        }
        if (bad) {
            // rows that see a token with a non-finite V group
            uint32_t seen = 0;
#pragma unroll
            for (int k = 0; k < 16; k++)
                seen |= s[k] != -__builtin_inff() ? 1u << (8 * (k >> 2) + (k & 3)) : 0u;
            seen <<= 4 * h;
            poison |= (seen & (uint32_t)bad ? 1u : 0u) |
                      (GPD == 2 && (seen & (uint32_t)(bad >> 32)) ? 2u : 0u);
        }
        float p[16];
        R.weights(s, Q, S.w, h, p);
        // ---- weighted sum
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            h8 P[F32 ? 2 : 1][2];
            if constexpr (F32) {
                uint32_t a[8], b[8];
                float cs = 0.0f, ls = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const v4f sc = *(const v4f *)&S.vs[g][8 * k + 4 * h];
                    const v4f cc = *(const v4f *)&S.vc[g][8 * k + 4 * h];
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = p[4 * k + e] * sc[e];
                        cs = fmaf(p[4 * k + e], cc[e], cs);
                    }
                    if (g == GPD - 1) {
                        const v4f w4 = *(const v4f *)&S.w[8 * k + 4 * h];
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
                    P[0][ks] = __builtin_bit_cast(h8, uint4{a[4 * ks], a[4 * ks + 1], a[4 * ks + 2],
                                                            a[4 * ks + 3]});
                    P[F32 ? 1 : 0][ks] = __builtin_bit_cast(h8, uint4{b[4 * ks], b[4 * ks + 1],
                                                                      b[4 * ks + 2], b[4 * ks + 3]});
                }
            } else {
                Soft<D, F32>::operand(p, P[0]);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const uint4 zl = *(const uint4 *)S.zl[g][ks][h], zh = *(const uint4 *)S.zh[g][ks][h];
                const uint32_t zls[4] = {zl.x, zl.y, zl.z, zl.w}, zhs[4] = {zh.x, zh.y, zh.z, zh.w};
                uint32_t a[4], b[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t y = (uint32_t)vx[g][ks][k >> 1] >> (8 * (k & 1));
                    h2 lo2 = nib2<false>(y, h_of(zls[k]), nc);
                    h2 hi2 = nib2<true>(y, h_of(zhs[k]), nc);
                    if constexpr (!F32) {
                        const h2 ss = h_of(((const uint32_t *)S.s16[g][ks][h])[k]);
                        const h2 cc = h_of(((const uint32_t *)S.c16[g][ks][h])[k]);
                        lo2 = __builtin_elementwise_fma(lo2, ss, cc);
                        hi2 = __builtin_elementwise_fma(hi2, ss, cc);
                    }
                    a[k] = u_of(lo2);
                    b[k] = u_of(hi2);
                }
                const h8 va = __builtin_bit_cast(h8, uint4{a[0], a[1], a[2], a[3]});
                const h8 vb8 = __builtin_bit_cast(h8, uint4{b[0], b[1], b[2], b[3]});
                if constexpr (F32) {
                    R.O[2 * g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, P[F32 ? 1 : 0][ks], R.O[2 * g], 0, 0, 0);
                    R.O[2 * g + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb8, P[F32 ? 1 : 0][ks],
                                                                          R.O[2 * g + 1], 0, 0, 0);
                }
                R.O[2 * g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, P[0][ks], R.O[2 * g], 0, 0, 0);
                R.O[2 * g + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb8, P[0][ks], R.O[2 * g + 1], 0, 0, 0);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };

    if (n_i > 0) {
        for (int i = 0; i < n_i; i += kAhead) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (i + k >= n_i) break;
                // all loads but those of the sub-tiles behind this one
                if constexpr (!F32) load(i + k + kAhead - 1, st[(k + kAhead - 1) % kAhead]);
                __builtin_amdgcn_sched_barrier(0);
                wait_loads<F32 ? 0 : (kAhead - 1) * kLoads>();
                __builtin_amdgcn_sched_barrier(0);
                consume(i + k, st[F32 ? 0 : k]);
            }
        }
        wait_loads<0>();
    }

    uint32_t nan_groups = poison | __shfl_xor(poison, 32, 64);
    const float l = R.finish(nan_groups);
    join_put<D, F32, kDWaves>((float *)lds, w, lane, R.O, l, R.M, r0 + n32 < rows,
                              row_out(job, c, chunk, tok, head, D, qrow, vec, part), out, part);
}

template <int D, bool F32>
int launch(const eakvd_geom &g, const WinJob &job, const void *q, const uint64_t *tree, void *out,
           float *part, bool vec, hipStream_t st)
{
    constexpr size_t tiles = kDWaves * sizeof(DraftLds<D, F32>), join = kJoinBytes<D>;
    constexpr size_t bytes = tiles > join ? tiles : join;
    auto *kern = draft_kernel<D, F32>;
    static std::atomic<uint64_t> done;
    const int e = allow_lds((const void *)kern, bytes, done);
    if (e) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)job.pre[job.n_seq]), dim3(64 * kDWaves), bytes, st, g, job, q,
                       tree, out, part, kKScale<F32> / sqrtf((float)D), (int)vec);
    return (int)hipGetLastError();
}

}  // namespace

int win_draft(const eakvd_geom &g, const WinJob &job, bool bf16, const void *q, const uint64_t *tree,
              void *out, float *part, bool vec, hipStream_t st)
{
    if (g.head_dim == 64)
        return bf16 ? launch<64, false>(g, job, q, tree, out, part, vec, st)
                    : launch<64, true>(g, job, q, tree, out, part, vec, st);
    return bf16 ? launch<128, false>(g, job, q, tree, out, part, vec, st)
                : launch<128, true>(g, job, q, tree, out, part, vec, st);
}
