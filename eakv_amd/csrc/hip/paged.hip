// paged.hip — attention of new tokens over K and V in pages of a pool: position t of
// sequence s is token table[s][t / P] * P + t % P of the pool, an ordinary cache, for
// pages of P tokens.  Query i of n is at position len - n + i and sees the positions up to
// its own:
//
//   out[i][h] = sum_t softmax_t(q[i][h].K[t] / sqrt(d)) V[t],
//   K[t] = n*s + b per group of 64 dims (n the nibble), V likewise.
//
// Lengths, tables and rows are device data, so a recorded graph follows them; the host
// knows bounds only.  The work is therefore split on the device: a unit is a row block (new
// tokens x the q heads of one kv head) of one sequence and kv head, its length the tiles that it
// sees.  All units stand in one line, which the blocks share evenly, whatever the lengths; every
// block finds its part from the lengths' prefix sum.  A unit that is cut leaves partial (O, M, l),
// at most two a block, which a second launch joins.  No atomics: results are the same bits on
// every call.
//
// Two forms.  Rows are few, or the work is small: units of up to 16 or 32 rows, whose 32-token
// sub-tiles a block's 4 waves take in turn, to join at the end.  Prompts: units of 128 to 256
// rows, a wave's 32 to 64 its own, for which the waves make K's and V's operands in LDS by turns,
// 128 tokens at a time; units of up to 16 rows beside them (single tokens) as before.  (In the
// first form making operands was a third of a prompt's instructions, and beginning, joining
// and ending units a fifth.)
//
// A sub-tile is two 16-token halves, each inside one page, so a page's address is scalar; pages of
// 64 sub-tiles are read at once, one to a lane.  K and V come through registers, a sub-tile ahead,
// by buffers of a half's own (loads to LDS would make every read of LDS wait for them).  Per
// sub-tile a wave computes
//   S^T = K Q^T    v_mfma_f32_16x16x32_f16, 16 tokens x 16 rows of each half
//   O^T = V^T P^T  16 dims x 16 rows; a lane's 8 scores belong to one row, and the
//                  tokens of the step are numbered so that the scores' registers are P's
//                  operand as they stand.
//
// K's operands: bf16 queries, the nibbles' own bits as subnormal f16 (2^-24 of them; a group's sum is
// good to 2^-11 of a step times the largest of q, against 2^-9 of q itself: nib_sub, window.h); f32
// queries, n - z with z the nibble nearest the value 0.
// Scales are applied to the f32 dots; the biases c = b + z*s enter by one product of three
// bf16 pieces each (24 bits).
// V: the weights carry the scales, x = p s.
//   bf16 queries  (prompts' units: V's values in f16, made once for all rows, and p)
//                 O[g] = sum_t x n + (p c - x z), nibbles as subnormals and the same rounded x
//                 in both places, so that n - z cancels what it should; the second term is
//                 one product with -z and one with c in every operand row.  x, p and c are
//                 rounded to f16, 2^-12 each, against the output's 2^-9.  The first sum is good
//                 to 2^-11 of the largest x for each 32 tokens (nib_sub; f32 results would show it).
//   f32 queries   O[g] = sum_t x (n - z) + p c, x a pair of f16 (24 bits), p c by f32 sums.
// Softmax, V's exponents and the reference point M: as in window.hip.
//
// Bound by instructions issued: single tokens' vector ALUs 68 % and all kinds together 94 % of the
// cycles, at nine tenths of HBM's rate at the same time; prompts' 59 to 64 and 76 to 82 %, matrix cores 31 to
// 36 %, with waits for operands, barriers and (d = 128) spilled registers of two waves to a SIMD, then
// 16 to 20 us of joining parts.  Measured (with the join; a copy of the same bytes at 5.17 TB/s, a library product 1257
// Tflop/s): a bf16 token of 32 q / 8 kv heads, d = 128, 64 sequences of 1000 to 16384 92-102 us (copy
// 87), 8 of 32768 77 us (65), one of 32768 27 us (8), one of 2048 11.2-11.6 us, two launches' latency;
// f32 tokens of the 64 sequences 133-147 us; prompts of 1500 of 4 sequences to 6001, 32 q / 4 kv, d =
// 64, 268-290 us (480 Tflop/s); 512 and 15 tokens f32 to 8200, 64 q / 8 kv, 360-411 us (370).
#include <string.h>

#include "pages.h"
#include "rows16.h"

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 8;                // log2 of a tile's tokens
constexpr int kRowsTile = 6;            // of units whose rows are divided among the waves
// M's distance from the maximum when it is set, and the headroom of a lazy M (log2 units): weights
// stay below 2^15.  A small distance moves M less often (every move scales O); weights keep f16's
// precision down to 2^-18 (f32: of their pairs, 2^-21) of the largest, and 2^-29 (2^-32) of it below.
template <bool F32>
constexpr float kTop = F32 ? 7.0f : 4.0f;
template <bool F32>
constexpr float kTau = F32 ? 8.0f : 11.0f;
// -z is held 2^11 times (30720 at most), as c with it, which f16 then holds to 2^-25
constexpr float kZUp = 0x1p11f;

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i *lds_v2i;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, int64_t bytes)
{
    // dword3 0x00020000: raw 32-bit buffer; reads beyond `bytes` return 0
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)(uint32_t)bytes, 0x00020000);
}

struct PagedJob {
    eakvd_pages b;
    const uint8_t *base;
    int layer, n_pages, log2p;
    int n_q, n_kv, qpk;
    int qinv;               // r / qpk = r * qinv >> 16 for the rows r of a block
    int tb, hb;             // tokens of a row block; row blocks of a token (else 1)
    int rbr;                // rows of a row block, at most 256
    int mixed;              // units of more than 16 rows divide these among the waves
    int whole;              // units are not cut
    const void *q;
    void *out;
    int64_t ld_q, ld_out;
    float ksc;
    int vec;
    float *part;            // [grid][2][rbr][D], then [grid][2][rbr][2]
    struct PagedCut *cut;   // [grid]
};

// A unit that begins in a block and ends in a later one.
struct PagedCut {
    int n;                  // blocks that hold a part of it, or 0
    int tok, rows;          // its first row of q and out, and its rows
    int head;               // its first q head
};

__device__ __forceinline__ int row_blocks(const PagedJob &J, int n)
{
    if (J.b.max_new <= J.tb) return n > 0 ? J.hb : 0;
    return n > 0 ? (n + J.tb - 1) / J.tb * J.hb : 0;
}

// Positions that row block rb of a sequence sees, and its length in the line.
__device__ __forceinline__ int seen_by(const PagedJob &J, const Seq &q, int rb)
{
    const int k = J.hb == 1 ? rb : rb / J.hb;
    return q.pos + min((k + 1) * J.tb, q.n);
}
// Its rows.
__device__ __forceinline__ int rows_of(const PagedJob &J, const Seq &q, int rb)
{
    return J.hb == 1 ? min(J.tb, q.n - rb * J.tb) * J.qpk : min(J.rbr, J.qpk - rb % J.hb * J.rbr);
}
// log2 of the tokens of a tile of the line: the wave's work for one is much the same either way.
__device__ __forceinline__ int tile_of(const PagedJob &J, const Seq &q, int rb)
{
    return J.mixed && rows_of(J, q, rb) > 16 ? kRowsTile : kTile;
}
__device__ __forceinline__ int length_of(const PagedJob &J, const Seq &q, int rb)
{
    if (J.whole) return 1;
    const int tile = tile_of(J, q, rb);
    return max(((seen_by(J, q, rb) - 1) >> tile) + 1, 1);
}

__device__ __forceinline__ int wave_sum_i(int v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The line's length of one kv head of the lanes' sequences.
__device__ __forceinline__ int head_length(const PagedJob &J, const Seq &q, int lane)
{
    const int nrb = row_blocks(J, q.n);
    int v = nrb ? length_of(J, q, 0) : 0;
    // sequences of several row blocks one after the other, the wave's lanes on their blocks
    uint64_t many = __ballot(nrb > 1);
    while (many) {
        const int k = __ffsll((unsigned long long)many) - 1;
        many &= many - 1;
        const Seq x = {0, __builtin_amdgcn_readlane(q.n, k), __builtin_amdgcn_readlane(q.pos, k)};
        const int all = __builtin_amdgcn_readlane(nrb, k);
        int sum = 0;
        for (int r = lane; r < all; r += 64) sum += length_of(J, x, r);
        sum = wave_sum_i(sum);
        if (lane == k) v = sum;
    }
    return v;
}

// The line, in LDS; its length is the result.  Up to 64 sequences: one to a lane, every wave for
// itself (all write the same), [5][64]: its length of one kv head, that before it, and itself, so
// that no barrier and, at a unit, no memory is waited for (0.9 us less of the 11.8 of a token of
// 512).  More: pre[s], the length of one kv head before sequence s, s <= n_seqs.  A list of rows that
// falls gives no line: its length might pass 32 bits, and blocks lose their places in it.
constexpr int kFew = 64;
__device__ __forceinline__ int line_of(const PagedJob &J, int *pre, int *sums, int tid)
{
    const int lane = tid & 63, w = tid >> 6, n = J.b.n_seqs;
    if (n <= kFew) {
        Seq q = {0, 0, 0};
        bool fell = false;
        if (lane < n) {
            q = seq_at(J.b, lane);
            fell = falls_at(J.b, lane);
        }
        const int len = head_length(J, q, lane), upto = wave_scan_i(len);
        const int x[5] = {len, upto - len, q.row, q.n, q.pos};
#pragma unroll
        for (int k = 0; k < 5; k++) pre[k * kFew + lane] = x[k];
        return __ballot(fell) ? 0 : __builtin_amdgcn_readlane(upto, 63) * J.n_kv;
    }
    int carry = 0, fallen = 0;
    for (int s0 = 0; s0 < n; s0 += 64 * kWaves) {
        const int s = s0 + tid;
        Seq q = {0, 0, 0};
        bool fell = false;
        if (s < n) {
            q = seq_at(J.b, s);
            fell = falls_at(J.b, s);
        }
        const int v = head_length(J, q, lane);
        const int upto = wave_scan_i(v);
        const uint64_t any = __ballot(fell);
        __syncthreads();
        if (lane == 63) {
            sums[w] = upto;
            sums[kWaves + w] = any != 0;
        }
        __syncthreads();
        int before = carry;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            const int x = sums[i];
            before += i < w ? x : 0;
            carry += x;
            fallen |= sums[kWaves + i];
        }
        if (s < n) pre[s] = before + upto - v;
    }
    if (tid == 0) pre[n] = carry;
    __syncthreads();
    return uni(fallen) ? 0 : uni(carry) * J.n_kv;
}

// Where place x of the line is.
struct Unit {
    int s, kvh, rb;
    int at, len;            // x's place in the unit and the unit's length
    Seq q;
    int seen;
};

__device__ __forceinline__ Unit unit_at(const PagedJob &J, const int *pre, int x, int lane)
{
    const int n = J.b.n_seqs;
    Unit u;
    // the last sequence that does not begin behind x; among many in two steps (n <= 4096)
    int first, per;
    if (n <= kFew) {
        int y[5];
#pragma unroll
        for (int k = 0; k < 5; k++) y[k] = pre[k * kFew + lane];
        u.s = uni((int)__popcll(__ballot(lane < n && y[1] * J.n_kv <= x))) - 1;
#pragma unroll
        for (int k = 0; k < 5; k++) y[k] = __builtin_amdgcn_readlane(y[k], u.s);
        per = y[0];
        first = y[1];
        u.q = Seq{y[2], y[3], y[4]};
    } else {
        const int i = lane * 64;
        int s = 64 * (uni((int)__popcll(__ballot(i < n && pre[min(i, n)] * J.n_kv <= x))) - 1);
        s += uni((int)__popcll(__ballot(s + lane < n && pre[min(s + lane, n)] * J.n_kv <= x))) - 1;
        u.s = s;
        const Seq q = seq_at(J.b, s);
        first = uni(pre[s]);
        per = uni(pre[s + 1]) - first;
        u.q.row = uni(q.row);
        u.q.n = uni(q.n);
        u.q.pos = uni(q.pos);
    }
    int z = x - first * J.n_kv;
    u.kvh = -1;
    for (int k = 0; k < J.n_kv; k += 64)
        u.kvh += uni((int)__popcll(__ballot(k + lane < J.n_kv && (k + lane) * per <= z)));
    z -= u.kvh * per;
    const int nrb = row_blocks(J, u.q.n);
    u.rb = 0;
    if (nrb > 1) {
        for (int r0 = 0; r0 < nrb; r0 += 64) {
            const int v = r0 + lane < nrb ? length_of(J, u.q, r0 + lane) : 0;
            const int upto = wave_scan_i(v);
            const uint64_t hit = __ballot(z < upto);
            if (hit) {
                const int k = __ffsll((unsigned long long)hit) - 1;
                u.rb = r0 + k;
                z -= __builtin_amdgcn_readlane(upto - v, k);
                break;
            }
            z -= __builtin_amdgcn_readlane(upto, 63);
        }
    }
    u.seen = seen_by(J, u.q, u.rb);
    u.len = length_of(J, u.q, u.rb);
    u.at = z;
    return u;
}

// Blocks of one XCD (every eighth) take a contiguous part of the line, so that the row
// blocks of a kv head share its planes in one L2.
__device__ __forceinline__ int line_block(int b, int grid)
{
    return grid % 8 == 0 ? (b & 7) * (grid >> 3) + (b >> 3) : b;
}

// Row tiles of a wave whose rows are its own: what 256 registers hold beside their queries.
// (bf16, 1500 x 4 to 6001 of 32Q/4KV, d = 64: 3 293 us, 4 289, 5 310; 8 kv heads, d = 128: 2 506, 3 485.  f32,
// the first of these: 3 427, 4 452; 512 and 15 tokens to 8200 of 64Q/8KV, d = 128: 1 609, 2 442.)  At d = 128
// they hold too much: 43 registers of bf16's and 35 of f32's are in scratch memory (168 and 136 bytes a
// lane), and what make() reads of it waits for all loads in flight.
template <int D, bool F32>
constexpr int kMany = D == 64 ? (F32 ? 3 : 4) : (F32 ? 2 : 3);

// What the form that divides tokens among the waves holds where.  NR row tiles of 16 share a
// wave's operands of K and V.  One (decode): queries in registers, 3 blocks to a CU.  Two: queries in
// LDS, which the waves of the block share, 2 blocks to a CU.
template <int D, bool F32, int NR>
struct Form {
    static constexpr int GPD = D / 64;
    static constexpr bool kShared = NR > 1;             // queries in LDS
    static constexpr int NQ = D / 32 * (F32 ? 2 : 1) + 1;

    struct __align__(16) Wave {
        uint8_t v[32 * 32 * GPD];               // V's bytes: rows of 32 GPD, their 16-byte units swizzled
        float ks[GPD][32];                      // K's scales
        float w[32];                            // 2^-e, e the exponent of a token's V
        float vs[GPD][32];                      // V's scales, 2^-e of them
        float vc[F32 ? GPD : 1][32];            // f32: V's biases c, 2^-e of them
        float zk[F32 ? GPD : 1][32];            // f32: K's z
        // of V's operands (block of 8 tokens, operand order): -(1024 + z) and -(64 + z), or
        // (bf16: scales in the weights, subnormals) -z and c
        _Float16 z0[GPD][4][8], z1[GPD][4][8];
    };
    struct Rows {
        uint4 q[NR][NQ][64];
        float rf[NR][16];
        int vis[NR][16];
    };
    static constexpr size_t kWaveBytes = kWaves * sizeof(Wave);
    static constexpr size_t kJoinRows = (size_t)kWaves * (D / 16) * 64 * 16;    // a row tile's sums
    static constexpr int kBuffers = NR > 1 && D == 64 ? 2 : 1;  // (two at d = 128 and one block is all that fits)
    static constexpr size_t kJoin = kBuffers * (kJoinRows + kWaves * 16 * sizeof(float2));
    static constexpr size_t kRows = kWaveBytes > kJoin ? kWaveBytes : kJoin;    // where the rows are
    static constexpr size_t kLine = kRows + (kShared ? sizeof(Rows) : 0);       // and the line
};

template <int GPD>
struct Stage {
    uint2 k[2][GPD];                    // (half, group)
    uint32_t v[2][2 * GPD];             // of each half, in order
    float ks, kb, vs, vb;
    int at_a, at_b;                     // the halves' tokens in the pool, or -1
};

// the unit permutation of token row t
template <int GPD>
__device__ __forceinline__ int unit_swz(int t)
{
    return GPD == 2 ? ((t >> 2) & 1) | ((t >> 3) & 2) : (t >> 4) & 1;
}

// A block's part of the line, unit by unit.  What a unit needs:
struct Piece {
    int lo, hi;             // positions
    int rows, tok0, head0;  // its rows, the sequence's new token and the q head that they begin with
    int slot;               // of its partial sums
    bool whole;
};
template <class Do>
__device__ __forceinline__ void walk(const PagedJob &J, uint8_t *lds, int *pre, int tid, const Do &unit)
{
    const int lane = tid & 63;
    const int grid = (int)gridDim.x, total = line_of(J, pre, (int *)lds, tid);
    const int share = max(1, (total + grid - 1) / grid);
    const int bl = line_block((int)blockIdx.x, grid);
    // (bl * share may pass 32 bits where there is little work for a large grid: no work then)
    const int x1 = (int)min((int64_t)total, ((int64_t)bl + 1) * share);
    int x = (int)min((int64_t)total, (int64_t)bl * share);
    PagedCut cut = {0, 0, 0, 0};
    while (x < x1) {
        const Unit U = unit_at(J, pre, x, lane);
        const int end = min(U.len, U.at + (x1 - x)), tile = tile_of(J, U.q, U.rb);
        Piece P;
        P.whole = U.at == 0 && end == U.len;
        const int hb = J.hb == 1 ? 0 : U.rb % J.hb, tb = J.hb == 1 ? U.rb : U.rb / J.hb;
        P.tok0 = tb * J.tb;                                     // of the sequence's new tokens
        P.rows = rows_of(J, U.q, U.rb);
        P.head0 = U.kvh * J.qpk + hb * J.rbr;
        P.lo = U.at << tile;
        P.hi = J.whole || end == U.len ? U.seen : end << tile;
        P.slot = 2 * bl + (U.at == 0 ? 1 : 0);
        unit(U, P);
        __syncthreads();
        if (U.at == 0 && !P.whole) {
            cut.n = (x + U.len - 1) / share - bl + 1;
            cut.tok = U.q.row + P.tok0;
            cut.rows = P.rows;
            cut.head = P.head0;
        }
        x += end - U.at;
    }
    if (!J.whole && tid == 0) J.cut[bl] = cut;
}

// A lane's places.
template <int GPD>
struct Lanes {
    static constexpr int RB = 32 * GPD;
    int n16, blk, n32, h, gh;
    bool owner;
    int pb, pos;            // of token n32 in V's operands: block of 8 tokens, place
    int ok;                 // its bytes of a half of K: token n16, bytes 8 blk of each group
    int vw, vr;             // of V in LDS: see write_at, read_at

    __device__ __forceinline__ explicit Lanes(int lane)
    {
        n16 = lane & 15, blk = lane >> 4, n32 = lane & 31, h = lane >> 5;
        ok = n16 * RB + 8 * blk;
        const int pj = (n32 & 3) | ((n32 >> 4) << 2);
        pb = (n32 >> 2) & 3;
        pos = (pj & 4) | ((pj & 1) << 1) | ((pj >> 1) & 1);
        const int t = lane >> 2, at = 8 * GPD * (lane & 3);
        vw = t * RB + 16 * ((at >> 4) ^ unit_swz<GPD>(t)) + (at & 15);
        const int jr = n16 >> 1, trow = 4 * blk + (jr & 3) + 16 * (jr >> 2);
        vr = trow * RB + 16 * unit_swz<GPD>(trow) + 8 * (lane & 1);
        owner = GPD == 2 || h == 0;
        gh = GPD == 2 ? h : 0;
    }
    // 8 GPD bytes of half k, which are part lane % 4 of row lane / 4 (the second half's rows have the
    // other unit permutation)
    __device__ __forceinline__ int write_at(int k) const { return k ? (vw ^ 16 * GPD) + 16 * RB : vw; }
    // transposed reads: the lane supplies 8 bytes of row j = n16 / 2 of its block's tokens
    __device__ __forceinline__ int read_at(int g, int c) const { return vr ^ 16 * (2 * g + c); }
};

// A wave's sub-tiles of a unit: w, w + 4, ..
template <int GPD>
struct Source {
    static constexpr int RB = 32 * GPD;
    const int32_t *table;
    const uint8_t *kw, *vw;
    __amdgpu_buffer_rsrc_t ks, kb, vs, vb;
    int log2p, n_pages, lo, hi, w, n_i;
    // pages of the wave's sub-tiles i, i + 1, .. i + 63: lane j holds where the halves of
    // i + j are in the pool (-1: nowhere)
    int pg_a = -1, pg_b = -1;

    __device__ __forceinline__ Source(const eakvd_geom &geo, const PagedJob &J, const Unit &U, const Piece &P, int wave)
        : log2p(J.log2p), n_pages(J.n_pages), lo(P.lo), hi(P.hi), w(wave)
    {
        const Planes K = planes_of(geo, J.base, J.layer, 0), V = planes_of(geo, J.base, J.layer, 1);
        const int64_t g0 = (int64_t)U.kvh * geo.gph;
        table = J.b.tables + (int64_t)U.s * J.b.ld_table;
        kw = K.w + g0 * 32, vw = V.w + g0 * 32;
        const int64_t plane = geo.gph * 4;
        ks = rsrc(K.s + g0, plane), kb = rsrc(K.b + g0, plane);
        vs = rsrc(V.s + g0, plane), vb = rsrc(V.b + g0, plane);
        const int n_sub = hi > lo ? (hi - lo + 31) / 32 : 0;
        n_i = n_sub > w ? (n_sub - w + kWaves - 1) / kWaves : 0;
    }
    __device__ __forceinline__ void pages(int i)
    {
        const int t = min(lo + 32 * (w + kWaves * (i + (int)(threadIdx.x & 63))), hi - 1) & ~31;
        pg_a = place_of(table, t, log2p, n_pages);
        pg_b = place_of(table, min(t + 16, (hi - 1) & ~15), log2p, n_pages);
    }
    // sub-tile i (the last one again behind it): K, the scales; then V.  A half's bytes by
    // buffers of its own: pages are anywhere in the plane.  AUX 2: read once.
    template <int AUX>
    __device__ __forceinline__ void load(int i, Stage<GPD> &st, const Lanes<GPD> &ln) const
    {
        i = min(i, n_i - 1);
        st.at_a = __builtin_amdgcn_readlane(pg_a, i & 63);
        st.at_b = __builtin_amdgcn_readlane(pg_b, i & 63);
        const int a = max(st.at_a, 0), b = max(st.at_b, 0);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const auto r = rsrc(kw + (int64_t)(k ? b : a) * RB, 16 * RB);
#pragma unroll
            for (int g = 0; g < GPD; g++) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b64(r, ln.ok + 32 * g, 0, AUX);
                st.k[k][g] = uint2{y[0], y[1]};
            }
        }
        const uint32_t at = (uint32_t)((ln.n32 < 16 ? a : b) + (ln.n32 & 15)) * (4 * GPD) + 4 * ln.gh;
        st.ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ks, at, 0, AUX));
        st.kb = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(kb, at, 0, AUX));
        st.vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vs, at, 0, AUX));
        st.vb = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vb, at, 0, AUX));
    }
    template <int AUX>
    __device__ __forceinline__ void load_v(Stage<GPD> &st) const
    {
        const int a = max(st.at_a, 0), b = max(st.at_b, 0), lane = (int)threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const auto r = rsrc(vw + (int64_t)(k ? b : a) * RB, 16 * RB);
            if constexpr (GPD == 2) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane, 0, AUX);
                st.v[k][0] = y[0], st.v[k][1] = y[1], st.v[k][GPD] = y[2], st.v[k][2 * GPD - 1] = y[3];
            } else {
                const auto y = __builtin_amdgcn_raw_buffer_load_b64(r, 8 * lane, 0, AUX);
                st.v[k][0] = y[0], st.v[k][1] = y[1];
            }
        }
    }
};

// A sub-tile's scales to LDS, and K's own operand of the bias product; the result: tokens whose
// V has a group that is not finite.  VALUES: V's operands will be its values.
template <int D, bool F32, bool VALUES, class Scales>
__device__ __forceinline__ uint64_t put_scales(Scales &S, const Stage<D / 64> &st, const Lanes<D / 64> &ln, bool live,
                                               float ksc, b8 &own)
{
    constexpr int GPD = D / 64;
    constexpr bool SUB = !F32 && !VALUES;
    const float zk = F32 ? zero_nibble(st.ks, st.kb) : 0.0f;
    const float ck = (F32 ? fmaf(zk, st.ks, st.kb) : st.kb) * ksc;
    // (a non-finite group counts as zeros and makes the rows that see it NaN)
    const float va = fmaxf(fabsf(st.vb), fabsf(fmaf(15.0f, st.vs, st.vb)));
    const bool fin = va < __builtin_inff() && st.vs == st.vs;
    const uint64_t bad = __ballot(live && !fin);
    const float sv = live && fin ? st.vs : 0.0f, bv = live && fin ? st.vb : 0.0f;
    const float zv = zero_nibble(sv, bv), cv = fmaf(zv, sv, bv);
    const float size = live && fin ? v_size<F32>(sv, va) : 0.0f;
    const int ev = exp_of(GPD == 2 ? half_max(size) : size);
    S.w[ln.n32] = scale2(1.0f, -ev);
    if (ln.owner) {
        S.ks[ln.gh][ln.n32] = st.ks * (F32 ? ksc : ksc * 0x1p24f);
        S.z0[ln.gh][ln.pb][ln.pos] = (_Float16)(SUB ? -zv * kZUp : -1024.0f - zv);
        S.z1[ln.gh][ln.pb][ln.pos] = (_Float16)(SUB ? scale2(cv, 11 - ev) : -64.0f - zv);
        if constexpr (VALUES) {
            S.s16[ln.gh][ln.pb][ln.pos] = (_Float16)scale2(sv, 15 - ev);
            S.c16[ln.gh][ln.pb][ln.pos] = (_Float16)scale2(cv, 15 - ev);
        } else {
            S.vs[ln.gh][ln.n32] = scale2(sv, -ev);
        }
        if constexpr (F32) {
            S.vc[F32 ? ln.gh : 0][ln.n32] = scale2(cv, -ev);
            S.zk[F32 ? ln.gh : 0][ln.n32] = zk;
        }
    }
    own = bias_own(ln.owner ? ck : 0.0f, (float)ev, ln.h == 0);
    return bad;
}

// V's bytes through LDS, transposed: the operands' bytes of each group and 16 dims.
template <int GPD>
__device__ __forceinline__ void turn(uint8_t *v, const Stage<GPD> &st, const Lanes<GPD> &ln, v2i (&vx)[GPD][2])
{
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if constexpr (GPD == 2)
            *(uint4 *)(v + ln.write_at(k)) = uint4{st.v[k][0], st.v[k][1], st.v[k][GPD], st.v[k][2 * GPD - 1]};
        else
            *(uint2 *)(v + ln.write_at(k)) = uint2{st.v[k][0], st.v[k][1]};
    }
#pragma unroll
    for (int g = 0; g < GPD; g++)
#pragma unroll
        for (int c = 0; c < 2; c++) vx[g][c] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(v + ln.read_at(g, c)));
}

// Rows that see a token with a non-finite V group: two bits of each row tile, of 8 scores s.
template <int GPD>
__device__ __forceinline__ uint32_t poison_of(const float (&s)[8], uint64_t bad, int blk)
{
    uint32_t seen = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) seen |= s[j] != -__builtin_inff() ? 1u << (16 * (j >> 2) + (j & 3)) : 0u;
    seen <<= 4 * blk;
    return (seen & (uint32_t)bad ? 1u : 0u) | (GPD == 2 && (seen & (uint32_t)(bad >> 32)) ? 2u : 0u);
}

__device__ __forceinline__ float max8(const float (&s)[8])
{
    return max3(max3(max3(s[0], s[1], s[2]), s[3], s[4]), max3(s[5], s[6], s[7]), s[7]);
}

// A unit of up to 16 NR rows: the block's waves take its sub-tiles in turn and join.
template <int D, bool F32, int NR>
__device__ __forceinline__ void unit_tokens(const eakvd_geom &geo, const PagedJob &J, uint8_t *lds,
                                            const Lanes<D / 64> &places, const NibConst &nc, const Unit &U,
                                            const Piece &P, int grid, int lane, int w)
{
    typedef Form<D, F32, NR> Fm;
    constexpr int GPD = D / 64, NF = D / 16, NP = F32 ? 2 : 1;
    constexpr bool kSub = !F32;
    constexpr int NC = kSub ? GPD : 1;
    typename Fm::Wave &S = ((typename Fm::Wave *)lds)[w];
    typename Fm::Rows &R = *(typename Fm::Rows *)(lds + Fm::kRows);
    const int n16 = lane & 15, blk = lane >> 4, rows = P.rows, tok0 = P.tok0, head0 = P.head0, lo = P.lo,
              hi = P.hi, slot = P.slot;
    const bool whole = P.whole;
    Source<GPD> src(geo, J, U, P, w);
    const int n_i = src.n_i;

    // row 16 u + n16: its token (of the unit's) and q head
    auto row_at = [&](int u, int &t, int &hd) __attribute__((always_inline)) {
        const int r = min(16 * u + n16, rows - 1);
        t = J.hb == 1 ? (int)((uint32_t)(r * J.qinv) >> 16) : 0;
        hd = r - t * J.qpk;
    };
    Query<D, F32, kSub> Q[Fm::kShared ? 1 : NR];
    int vis1 = 0;
    float rf1 = 0.0f;
#pragma unroll
    for (int u = 0; u < NR; u++) {
        int t, hd;
        row_at(u, t, hd);
        const int vis = U.q.pos + tok0 + t + 1;              // positions that the row sees
        if (!Fm::kShared || (u % kWaves == w && 16 * u < rows)) {
            auto &q = Q[Fm::kShared ? 0 : u];
            q.load(J.q, (int64_t)(U.q.row + tok0 + t) * J.ld_q + (int64_t)(head0 + hd) * D, J.vec & 1, blk);
            if constexpr (Fm::kShared) {
#pragma unroll
                for (int f = 0; f < D / 32; f++) {
                    R.q[u][f][lane] = __builtin_bit_cast(uint4, q.a[f]);
                    if constexpr (F32) R.q[u][D / 32 + (F32 ? f : 0)][lane] = __builtin_bit_cast(uint4, q.b[F32 ? f : 0]);
                }
                R.q[u][Fm::NQ - 1][lane] = __builtin_bit_cast(uint4, q.bias);
                if (blk == 0) {
                    R.rf[u][n16] = q.rf;
                    R.vis[u][n16] = vis;
                }
            } else {
                vis1 = vis;
                rf1 = q.rf;
            }
        }
    }
    if constexpr (Fm::kShared) __syncthreads();
    const int vis_min = U.q.pos + tok0 + 1;

    constexpr int aux = NR == 1 ? 2 : 0;                         // (read once, or again by other rows)
    v4f O[NR][NF], C[NR][NC];
    float M[NR], L[NR], cs[NR][F32 ? GPD : 1];
    uint32_t poison = 0;                                     // two bits of each row tile: NaN groups
#pragma unroll
    for (int u = 0; u < NR; u++) {
#pragma unroll
        for (int f = 0; f < NF; f++) O[u][f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < NC; g++) C[u][g] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < (F32 ? GPD : 1); g++) cs[u][g] = 0.0f;
        M[u] = kMInit;
        L[u] = 0.0f;
    }

    // N: row tiles that the unit has (1, or NR)
    auto consume = [&](auto count, int i, Stage<GPD> &st) __attribute__((always_inline)) {
        constexpr int N = decltype(count)::value;
        const int t0 = lo + 32 * (w + kWaves * i);
        const bool ok_a = st.at_a >= 0, ok_b = st.at_b >= 0;
        // (d = 128: worked out again rather than kept, f32's in scratch memory, whose reads wait for the
        // loads in flight: 152 against 162 us for f32 tokens of 64 sequences, bf16 8 at 32768 78 against 83.
        // 17 of f32's registers still are there, read once a unit)
        int l = lane;
        if constexpr (D == 128) asm("" : "+v"(l));
        const Lanes<GPD> ln = D == 128 ? Lanes<GPD>(l) : places;
        const int n32 = ln.n32;
        // tokens behind the last, or in no page, have no part in this
        const bool live = t0 + n32 < hi && (n32 < 16 ? ok_a : ok_b);
        // ---- scales to LDS
        b8 own, bias[2];
        const uint64_t bad = put_scales<D, F32, false>(S, st, ln, live, J.ksc, own);
        bias_halves(own, bias, n32);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        v2i vx[GPD][2];
        if constexpr (NR == 1) turn<GPD>(S.v, st, ln, vx);
        // ---- the next sub-tile
        __builtin_amdgcn_sched_barrier(0);
        if (((i + 1) & 63) == 0 && i + 1 < n_i) src.pages(i + 1);
        uint2 kx[2][GPD];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int g = 0; g < GPD; g++) kx[k][g] = st.k[k][g];
        src.template load<aux>(i + 1, st, ln);
        if constexpr (NR == 1) src.template load_v<aux>(st);
        __builtin_amdgcn_sched_barrier(0);
        // ---- K's operands
        h8 kl[2][GPD], kh[2][GPD];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int g = 0; g < GPD; g++)
                k_operands<!F32>(kx[k][g], F32 ? S.zk[F32 ? g : 0][16 * k + n16] : 0.0f, nc, kl[k][g], kh[k][g]);
        const bool masked = t0 + 32 > vis_min || !ok_a || !ok_b;
        // ---- scores
        float s[N][8];
#pragma unroll
        for (int u = 0; u < N; u++) {
            auto &q = Q[0];
            if constexpr (Fm::kShared) {
                if constexpr (N > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int f = 0; f < D / 32; f++) {
                    q.a[f] = __builtin_bit_cast(h8, R.q[u][f][lane]);
                    if constexpr (F32) q.b[F32 ? f : 0] = __builtin_bit_cast(h8, R.q[u][D / 32 + (F32 ? f : 0)][lane]);
                }
                q.bias = __builtin_bit_cast(b8, R.q[u][Fm::NQ - 1][lane]);
            }
            v4f t[2];
#pragma unroll
            for (int k = 0; k < 2; k++)
                t[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias[k], q.bias, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
            for (int g = 0; g < GPD; g++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const v4f acc = group_dots(kl[k][g], kh[k][g], q, g);
                    const v4f sc = *(const v4f *)&S.ks[g][16 * k + 4 * blk];
#pragma unroll
                    for (int e = 0; e < 4; e++) t[k][e] = fmaf(sc[e], acc[e], t[k][e]);
                }
#pragma unroll
            for (int j = 0; j < 8; j++) s[u][j] = t[j >> 2][j & 3];
        }
        if constexpr (N > 1) __builtin_amdgcn_sched_barrier(0);
        // ---- softmax, all row tiles side by side
        if (masked) {
#pragma unroll
            for (int u = 0; u < N; u++) {
                const int n = (Fm::kShared ? R.vis[u][n16] : vis1) - t0 - 4 * blk;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool see = 16 * (j >> 2) + (j & 3) < n && (j >> 2 ? ok_b : ok_a);
                    s[u][j] = see ? s[u][j] : -__builtin_inff();
                }
            }
        }
        if (bad) {
#pragma unroll
            for (int u = 0; u < N; u++) poison |= poison_of<GPD>(s[u], bad, blk) << 2 * u;
        }
        // (a lane looks at its own scores; a row's lanes join where one of them moves M)
        float rf[N], top[N];
        bool move = false;
        auto moves = [&](int u) __attribute__((always_inline)) {
            return fmaf(top[u], rf[u], -(kTop<F32> + kTau<F32>)) > M[u];
        };
#pragma unroll
        for (int u = 0; u < N; u++) {
            rf[u] = Fm::kShared ? R.rf[u][n16] : rf1;
            top[u] = max8(s[u]);
            move |= moves(u);
        }
        if (__ballot(move) != 0) {
#pragma unroll
            for (int u = 0; u < N; u++) {
                if (N > 1 && __ballot(moves(u)) == 0) continue;
                top[u] = row_max(top[u]);
                const float mn = moves(u) ? fmaf(top[u], rf[u], -kTop<F32>) : M[u], d = M[u] - mn;
                // (L by halves, as in window.h)
                const float al = __builtin_amdgcn_exp2f(d), half = __builtin_amdgcn_exp2f(0.5f * d);
                L[u] = L[u] * half * half;
#pragma unroll
                for (int f = 0; f < NF; f++)
#pragma unroll
                    for (int e = 0; e < 4; e++) O[u][f][e] *= al;
                if constexpr (kSub)
#pragma unroll
                    for (int g = 0; g < NC; g++)
#pragma unroll
                        for (int e = 0; e < 4; e++) C[u][g][e] *= al;
                if constexpr (F32)
#pragma unroll
                    for (int g = 0; g < GPD; g++) cs[u][g] *= al;
                M[u] = mn;
            }
        }
        h8 X[N][NP][GPD], W16[F32 ? 1 : N];
        const v4f w0 = *(const v4f *)&S.w[4 * blk], w1 = *(const v4f *)&S.w[16 + 4 * blk];
#pragma unroll
        for (int u = 0; u < N; u++) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(fmaf(s[u][j], rf[u], -M[u]));
            float ls = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) ls = fmaf(p[j], j < 4 ? w0[j & 3] : w1[j & 3], ls);
            L[u] += ls;
            // weights as operands
#pragma unroll
                for (int g = 0; g < GPD; g++) {
                    uint32_t xh[4], xl[4];
                    float c = 0.0f;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const v4f sc = *(const v4f *)&S.vs[g][16 * k + 4 * blk];
                        float y[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = p[4 * k + e] * sc[e];
                        if constexpr (F32) {
                            const v4f cc = *(const v4f *)&S.vc[F32 ? g : 0][16 * k + 4 * blk];
#pragma unroll
                            for (int e = 0; e < 4; e++) c = fmaf(p[4 * k + e], cc[e], c);
                        }
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const h2 hi2 = pk(y[e], y[e + 2]);
                            xh[2 * k + e] = u_of(hi2);
                            if constexpr (F32) xl[2 * k + e] = u_of(pk_rest(hi2, y[e], y[e + 2]));
                        }
                    }
                    X[u][0][g] = __builtin_bit_cast(h8, uint4{xh[0], xh[1], xh[2], xh[3]});
                    if constexpr (F32) {
                        X[u][NP - 1][g] = __builtin_bit_cast(h8, uint4{xl[0], xl[1], xl[2], xl[3]});
                        cs[u][F32 ? g : 0] += c;
                    }
                }
            if constexpr (!F32)
                W16[F32 ? 0 : u] = __builtin_bit_cast(h8, uint4{u_of(pk_exp(p[0], p[2])), u_of(pk_exp(p[1], p[3])),
                                                              u_of(pk_exp(p[4], p[6])), u_of(pk_exp(p[5], p[7]))});
        }
        if constexpr (NR > 1) {
            __builtin_amdgcn_sched_barrier(0);
            turn<GPD>(S.v, st, ln, vx);
            src.template load_v<aux>(st);
            __builtin_amdgcn_sched_barrier(0);
        }
        // ---- weighted sums
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            if constexpr (NR > 1) __builtin_amdgcn_sched_barrier(0);
            const uint4 z0 = *(const uint4 *)S.z0[g][blk], z1 = *(const uint4 *)S.z1[g][blk];
            const uint32_t zl[4] = {z0.x, z0.y, z0.z, z0.w}, zh[4] = {z1.x, z1.y, z1.z, z1.w};
            if constexpr (kSub) {
#pragma unroll
                for (int u = 0; u < N; u++) {
                    v4f &c = C[u][kSub ? g : 0];
                    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, z0), X[u][0][g], c, 0, 0, 0);
                    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, z1), W16[F32 ? 0 : u], c, 0, 0, 0);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if constexpr (NR > 1) __builtin_amdgcn_sched_barrier(0);
                uint32_t a[4], b[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t y = (uint32_t)vx[g][c][k >> 1] >> (8 * (k & 1));
                    if constexpr (kSub) {
                        a[k] = nib_sub<false>(y);
                        b[k] = nib_sub<true>(y);
                    } else {
                        a[k] = u_of(nib2<false>(y, h_of(zl[k]), nc));
                        b[k] = u_of(nib2<true>(y, h_of(zh[k]), nc));
                    }
                }
                const h8 vl = __builtin_bit_cast(h8, uint4{a[0], a[1], a[2], a[3]});
                const h8 vh = __builtin_bit_cast(h8, uint4{b[0], b[1], b[2], b[3]});
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const int f = 4 * g + 2 * c;
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--) {
                        const h8 &y = X[u][k][g];
                        O[u][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, y, O[u][f], 0, 0, 0);
                        O[u][f + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, y, O[u][f + 1], 0, 0, 0);
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };

    if (n_i > 0) {
        src.pages(0);
        Stage<GPD> st;
        src.template load<aux>(0, st, places);
        src.template load_v<aux>(st);
        if (NR > 1 && rows > 16)
            for (int i = 0; i < n_i; i++) consume(std::integral_constant<int, NR>(), i, st);
        else
            for (int i = 0; i < n_i; i++) consume(std::integral_constant<int, 1>(), i, st);
    }

    // ---- the waves joined, 16 rows at a time
    // (two buffers: one is read while the next is written)
    const bool poisoned = __ballot(poison != 0) != 0;
    if (poisoned) {
        poison |= __shfl_xor(poison, 16, 64);
        poison |= __shfl_xor(poison, 32, 64);
    }
#pragma unroll
    for (int u = 0; u < NR; u++) {
        if (u > 0 && 16 * u >= rows) break;
        float *jo = (float *)(lds + u % Fm::kBuffers * Fm::kJoinRows);            // [wave][NF][64][4]
        float2 *jml = (float2 *)(lds + Fm::kBuffers * Fm::kJoinRows) + u % Fm::kBuffers * kWaves * 16;   // [wave][16]
        // a lane has its row's sums of its own tokens only
        const float l = row_sum(L[u]);
        if (u == 0 || Fm::kBuffers == 1) __syncthreads();
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            const float c = F32 ? row_sum(cs[u][F32 ? g : 0]) : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int f = 4 * g + k;
                v4f o;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    o[e] = F32 ? O[u][f][e] + c
                               : fmaf(O[u][f][e], k & 1 ? 0x1p20f : 0x1p24f, C[u][kSub ? g : 0][e] * (1.0f / kZUp));
                }
                if (poisoned && (poison >> (2 * u + g) & 1))
                    o = v4f{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
                *((v4f *)jo + (w * NF + f) * 64 + lane) = o;
            }
        }
        if (blk == 0) jml[w * 16 + n16] = float2{M[u], l};
        __syncthreads();
        float al[kWaves], m = kMInit, ll = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; k++) {
            al[k] = jml[k * 16 + n16].x;
            m = fmaxf(m, al[k]);
        }
#pragma unroll
        for (int k = 0; k < kWaves; k++) {
            const float half = __builtin_amdgcn_exp2f(0.5f * (al[k] - m));
            al[k] = __builtin_amdgcn_exp2f(al[k] - m);
            ll = fmaf(half * jml[k * 16 + n16].y, half, ll);
        }
        const bool row_ok = 16 * u + n16 < rows;
        for (int f = w; f < NF; f += kWaves) {
            v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kWaves; k++) {
                const v4f o = *((const v4f *)jo + (k * NF + f) * 64 + lane);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = fmaf(al[k], o[e], y[e]);
            }
            const int dim = (f >> 2) * 64 + (f & 1) * 32 + ((f >> 1) & 1) * 16 + 4 * blk;
            if (row_ok && whole) {
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                const float o4[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
                int t, hd;
                row_at(u, t, hd);
                store4<F32>(J.out, (int64_t)(U.q.row + tok0 + t) * J.ld_out + (int64_t)(head0 + hd) * D + dim,
                            J.vec & 2, o4);
            } else if (row_ok) {
                *(v4f *)(J.part + ((int64_t)slot * J.rbr + 16 * u + n16) * D + dim) = y;
            }
        }
        if (!whole && row_ok && blk == 0 && w == 0) {
            float *ml = J.part + (int64_t)grid * 2 * J.rbr * D + ((int64_t)slot * J.rbr + 16 * u + n16) * 2;
            ml[0] = m;
            ml[1] = ll;
        }
    }
}

template <int D, bool F32, int NR>
__global__ __launch_bounds__(64 * kWaves, NR > 1 ? 2 : 3) void paged_kernel(eakvd_geom geo, PagedJob J)
{
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
    const Lanes<D / 64> ln(lane);
    NibConst nc;
    nc.hold();
    walk(J, lds, (int *)(lds + Form<D, F32, NR>::kLine), tid,
         [&](const Unit &U, const Piece &P) __attribute__((always_inline)) {
             unit_tokens<D, F32, NR>(geo, J, lds, ln, nc, U, P, (int)gridDim.x, lane, w);
         });
}

// What the waves of a block share of 32 tokens: K's and V's operands and scales.  (What only the
// wave that makes them needs is among them: v's room holds V's bytes first.)
template <int D, bool F32>
struct __align__(16) Slot {
    static constexpr int GPD = D / 64;
    uint4 k[2][GPD][2][64];                     // half, group, nibble
    uint4 v[GPD][2][2][64];                     // group, 16 dims, nibble
    b8 bias[64];
    float ks[GPD][32], w[32];
    float vs[F32 ? GPD : 1][32], vc[F32 ? GPD : 1][32], zk[F32 ? GPD : 1][32];
    _Float16 z0[GPD][4][8], z1[GPD][4][8], s16[F32 ? 1 : GPD][4][8], c16[F32 ? 1 : GPD][4][8];
    uint64_t bad;
    int ok, pad;                                // whether the halves are in pages
};

// A unit of more rows: each wave has up to NR row tiles of its own, and the waves make the operands
// of 32 tokens each for all.  So these cost a row tile a quarter, a unit has four times the rows,
// and its waves have nothing to join.
template <int D, bool F32, int NR>
__device__ __forceinline__ void unit_rows(const eakvd_geom &geo, const PagedJob &J, uint8_t *lds,
                                          const NibConst &nc, const Unit &U, const Piece &P, int grid, int lane, int w)
{
    constexpr int GPD = D / 64, NF = D / 16, NP = F32 ? 2 : 1;
    Slot<D, F32> *slots = (Slot<D, F32> *)lds;
    const int n16 = lane & 15, blk = lane >> 4, rows = P.rows, lo = P.lo, hi = P.hi;
    const int n_u = ((rows + 15) / 16 + kWaves - 1) / kWaves, r0 = 16 * n_u * w;     // row tiles of a wave, its first row
    Source<GPD> src(geo, J, U, P, w);
    const int n_sub = hi > lo ? (hi - lo + 31) / 32 : 0;
    auto token = [&](int r) __attribute__((always_inline)) {     // row r's, of the unit's
        return J.hb == 1 ? (int)((uint32_t)(min(r, rows - 1) * J.qinv) >> 16) : 0;
    };
    const int pos0 = U.q.pos + P.tok0 + 1;                       // positions that token 0's rows see
    const int vis_min = pos0 + token(r0), vis_max = r0 < rows ? pos0 + token(r0 + 16 * n_u - 1) : 0;
    // (f32 at d = 128: V as its tokens' turn comes; a step ahead it does not fit the registers)
    constexpr bool late = F32 && D == 128;
    Stage<GPD> st;
    if (src.n_i > 0) {
        src.pages(0);
        src.template load<0>(0, st, Lanes<GPD>(lane));
        if constexpr (!late) src.template load_v<0>(st);
    }
    // (a lane's places are worked out again where they are wanted, not kept in registers)
    auto again = [&]() __attribute__((always_inline)) {
        int l = lane;
        asm("" : "+v"(l));
        return l;
    };
    // a wave's own 32 tokens of a step
    auto make = [&](int i) __attribute__((always_inline)) {
        Slot<D, F32> &S = slots[w];
        const Lanes<GPD> ln(again());
        if constexpr (late) src.template load_v<0>(st);
        const int t0 = lo + 32 * (w + kWaves * i);
        const bool ok_a = st.at_a >= 0, ok_b = st.at_b >= 0;
        const bool live = t0 + ln.n32 < hi && (ln.n32 < 16 ? ok_a : ok_b);
        b8 own;
        const uint64_t bad = put_scales<D, F32, !F32>(S, st, ln, live, J.ksc, own);
        S.bias[lane] = own;
        if (lane == 0) {
            S.bad = bad;
            S.ok = (ok_a ? 1 : 0) | (ok_b ? 2 : 0);
        }
        v2i vx[GPD][2];
        turn<GPD>((uint8_t *)S.v, st, ln, vx);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int g = 0; g < GPD; g++) {
                h8 kl, kh;
                k_operands<!F32>(st.k[k][g], F32 ? S.zk[F32 ? g : 0][16 * k + n16] : 0.0f, nc, kl, kh);
                S.k[k][g][0][lane] = __builtin_bit_cast(uint4, kl);
                S.k[k][g][1][lane] = __builtin_bit_cast(uint4, kh);
            }
#pragma unroll
        for (int g = 0; g < GPD; g++) {
            const uint4 z0 = *(const uint4 *)S.z0[g][blk], z1 = *(const uint4 *)S.z1[g][blk];
            const uint32_t zl[4] = {z0.x, z0.y, z0.z, z0.w}, zh[4] = {z1.x, z1.y, z1.z, z1.w};
            uint32_t ss[4], cc[4];
            if constexpr (!F32) {
                const uint4 a = *(const uint4 *)S.s16[F32 ? 0 : g][blk], b = *(const uint4 *)S.c16[F32 ? 0 : g][blk];
                ss[0] = a.x, ss[1] = a.y, ss[2] = a.z, ss[3] = a.w;
                cc[0] = b.x, cc[1] = b.y, cc[2] = b.z, cc[3] = b.w;
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t a[4], b[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t y = (uint32_t)vx[g][c][k >> 1] >> (8 * (k & 1));
                    h2 lo2 = nib2<false>(y, h_of(zl[k]), nc), hi2 = nib2<true>(y, h_of(zh[k]), nc);
                    if constexpr (!F32) {
                        lo2 = __builtin_elementwise_fma(lo2, h_of(ss[k]), h_of(cc[k]));
                        hi2 = __builtin_elementwise_fma(hi2, h_of(ss[k]), h_of(cc[k]));
                    }
                    a[k] = u_of(lo2);
                    b[k] = u_of(hi2);
                }
                S.v[g][c][0][lane] = uint4{a[0], a[1], a[2], a[3]};
                S.v[g][c][1][lane] = uint4{b[0], b[1], b[2], b[3]};
            }
        }
        // ---- the next ones
        if (((i + 1) & 63) == 0 && i + 1 < src.n_i) src.pages(i + 1);
        src.template load<0>(i + 1, st, ln);
        if constexpr (!late) src.template load_v<0>(st);
    };

    // N: row tiles of a wave (1, or NR)
    auto run = [&](auto count) __attribute__((always_inline)) {
        constexpr int N = decltype(count)::value;
        typedef Query<D, F32, !F32> Qy;
        Qy Q[N];
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int r = min(r0 + 16 * u + n16, rows - 1), t = token(r);
            Q[u].load(J.q, (int64_t)(U.q.row + P.tok0 + t) * J.ld_q + (int64_t)(P.head0 + r - t * J.qpk) * D,
                      J.vec & 1, blk);
        }
        v4f O[N][NF];
        float M[N], L[N], cs[N][F32 ? GPD : 1];
        uint32_t poison = 0;
#pragma unroll
        for (int u = 0; u < N; u++) {
#pragma unroll
            for (int f = 0; f < NF; f++) O[u][f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < (F32 ? GPD : 1); g++) cs[u][g] = 0.0f;
            M[u] = kMInit;
            L[u] = 0.0f;
        }
        auto consume = [&](const Slot<D, F32> &S, int t0) __attribute__((always_inline)) {
            const int ok = uni(S.ok);
            b8 bias[2];
            bias_halves(S.bias[lane], bias, lane & 31);
            float s[N][8];
            v4f t[N][2];
#pragma unroll
            for (int u = 0; u < N; u++)
#pragma unroll
                for (int k = 0; k < 2; k++)
                    t[u][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias[k], Q[u].bias, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
            for (int g = 0; g < GPD; g++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const h8 kl = __builtin_bit_cast(h8, S.k[k][g][0][lane]), kh = __builtin_bit_cast(h8, S.k[k][g][1][lane]);
                    const v4f sc = *(const v4f *)&S.ks[g][16 * k + 4 * blk];
#pragma unroll
                    for (int u = 0; u < N; u++) {
                        const v4f acc = group_dots(kl, kh, Q[u], g);
#pragma unroll
                        for (int e = 0; e < 4; e++) t[u][k][e] = fmaf(sc[e], acc[e], t[u][k][e]);
                    }
                }
#pragma unroll
            for (int u = 0; u < N; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) s[u][j] = t[u][j >> 2][j & 3];
            if (t0 + 32 > vis_min || ok != 3) {
                const int l = again();
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const int n = pos0 + token(r0 + 16 * u + (l & 15)) - t0 - 4 * (l >> 4);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const bool see = 16 * (j >> 2) + (j & 3) < n && (ok >> (j >> 2) & 1);
                        s[u][j] = see ? s[u][j] : -__builtin_inff();
                    }
                }
            }
            const uint32_t bad_a = (uint32_t)uni((int)(uint32_t)S.bad), bad_b = (uint32_t)uni((int)(uint32_t)(S.bad >> 32));
            if (bad_a | bad_b) {
#pragma unroll
                for (int u = 0; u < N; u++) poison |= poison_of<GPD>(s[u], (uint64_t)bad_b << 32 | bad_a, blk) << 2 * u;
            }
            float top[N];
            bool move = false;
            auto moves = [&](int u) __attribute__((always_inline)) {
                return fmaf(top[u], Q[u].rf, -(kTop<F32> + kTau<F32>)) > M[u];
            };
#pragma unroll
            for (int u = 0; u < N; u++) {
                top[u] = max8(s[u]);
                move |= moves(u);
            }
            if (__ballot(move) != 0) {
#pragma unroll
                for (int u = 0; u < N; u++) {
                    if (N > 1 && __ballot(moves(u)) == 0) continue;
                    top[u] = row_max(top[u]);
                    const float mn = moves(u) ? fmaf(top[u], Q[u].rf, -kTop<F32>) : M[u], d = M[u] - mn;
                    const float al = __builtin_amdgcn_exp2f(d), half = __builtin_amdgcn_exp2f(0.5f * d);
                    L[u] = L[u] * half * half;
#pragma unroll
                    for (int f = 0; f < NF; f++)
#pragma unroll
                        for (int e = 0; e < 4; e++) O[u][f][e] *= al;
                    if constexpr (F32)
#pragma unroll
                        for (int g = 0; g < GPD; g++) cs[u][g] *= al;
                    M[u] = mn;
                }
            }
            h8 X[N][NP][F32 ? GPD : 1];         // f32: weights times V's scales, in two parts; else the weights
            const v4f w0 = *(const v4f *)&S.w[4 * blk], w1 = *(const v4f *)&S.w[16 + 4 * blk];
#pragma unroll
            for (int u = 0; u < N; u++) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(fmaf(s[u][j], Q[u].rf, -M[u]));
                float ls = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) ls = fmaf(p[j], j < 4 ? w0[j & 3] : w1[j & 3], ls);
                L[u] += ls;
                if constexpr (F32) {
#pragma unroll
                    for (int g = 0; g < GPD; g++) {
                        uint32_t xh[4], xl[4];
                        float c = 0.0f;
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const v4f sc = *(const v4f *)&S.vs[F32 ? g : 0][16 * k + 4 * blk],
                                      cc = *(const v4f *)&S.vc[F32 ? g : 0][16 * k + 4 * blk];
                            float y[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                y[e] = p[4 * k + e] * sc[e];
                                c = fmaf(p[4 * k + e], cc[e], c);
                            }
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const h2 hi2 = pk(y[e], y[e + 2]);
                                xh[2 * k + e] = u_of(hi2);
                                xl[2 * k + e] = u_of(pk_rest(hi2, y[e], y[e + 2]));
                            }
                        }
                        X[u][0][F32 ? g : 0] = __builtin_bit_cast(h8, uint4{xh[0], xh[1], xh[2], xh[3]});
                        X[u][NP - 1][F32 ? g : 0] = __builtin_bit_cast(h8, uint4{xl[0], xl[1], xl[2], xl[3]});
                        cs[u][F32 ? g : 0] += c;
                    }
                } else {
                    X[u][0][0] = __builtin_bit_cast(h8, uint4{u_of(pk_exp(p[0], p[2])), u_of(pk_exp(p[1], p[3])),
                                                              u_of(pk_exp(p[4], p[6])), u_of(pk_exp(p[5], p[7]))});
                }
            }
#pragma unroll
            for (int g = 0; g < GPD; g++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const h8 vl = __builtin_bit_cast(h8, S.v[g][c][0][lane]), vh = __builtin_bit_cast(h8, S.v[g][c][1][lane]);
                    const int f = 4 * g + 2 * c;
#pragma unroll
                    for (int u = 0; u < N; u++)
#pragma unroll
                        for (int k = NP - 1; k >= 0; k--) {
                            const h8 &y = X[u][k][F32 ? g : 0];
                            O[u][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, y, O[u][f], 0, 0, 0);
                            O[u][f + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, y, O[u][f + 1], 0, 0, 0);
                        }
                }
        };
        for (int i = 0; kWaves * i < n_sub; i++) {
            if (i < src.n_i) make(i);
            __syncthreads();
            const int t1 = min(min(hi, vis_max), lo + 32 * kWaves * (i + 1));
#pragma unroll 1
            for (int j = 0; j < kWaves; j++) {
                const int t0 = lo + 32 * (kWaves * i + j);
                if (t0 >= t1) break;
                consume(slots[j], t0);
            }
            __syncthreads();
        }
        const bool poisoned = __ballot(poison != 0) != 0;
        if (poisoned) {
            poison |= __shfl_xor(poison, 16, 64);
            poison |= __shfl_xor(poison, 32, 64);
        }
        const int l1 = again();
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int r = r0 + 16 * u + (l1 & 15), t = token(r);
            const bool mine = u < n_u && r < rows;
            const float l = row_sum(L[u]);
            const float inv = P.whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            float *part = J.part + ((int64_t)P.slot * J.rbr + r) * D;
            const int64_t out = (int64_t)(U.q.row + P.tok0 + t) * J.ld_out + (int64_t)(P.head0 + r - t * J.qpk) * D;
#pragma unroll
            for (int g = 0; g < GPD; g++) {
                const float c = F32 ? row_sum(cs[u][F32 ? g : 0]) : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int f = 4 * g + k, dim = g * 64 + (k & 1) * 32 + (k >> 1) * 16 + 4 * (l1 >> 4);
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[e] = (F32 ? O[u][f][e] + c : O[u][f][e] * 0x1p-15f) * inv;
                        if (poisoned && (poison >> (2 * u + g) & 1)) o[e] = __builtin_nanf("");
                    }
                    if (mine && P.whole) store4<F32>(J.out, out + dim, J.vec & 2, o);
                    if (mine && !P.whole) *(v4f *)(part + dim) = v4f{o[0], o[1], o[2], o[3]};
                }
            }
            if (mine && !P.whole && blk == 0) {
                float *ml = J.part + (int64_t)grid * 2 * J.rbr * D + ((int64_t)P.slot * J.rbr + r) * 2;
                ml[0] = M[u];
                ml[1] = l;
            }
        }
    };
    if (n_u == 1) run(std::integral_constant<int, 1>());
    else run(std::integral_constant<int, NR>());
}

// Prompts, and single tokens beside them.
template <int D, bool F32>
constexpr size_t kRowsLds = sizeof(Slot<D, F32>) * kWaves > Form<D, F32, 1>::kLine ? sizeof(Slot<D, F32>) * kWaves
                                                                                  : Form<D, F32, 1>::kLine;
template <int D, bool F32, int NR>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_rows_kernel(eakvd_geom geo, PagedJob J)
{
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
    walk(J, lds, (int *)(lds + kRowsLds<D, F32>), tid, [&](const Unit &U, const Piece &P) __attribute__((always_inline)) {
        int l = lane;
        asm("" : "+v"(l));
        NibConst nc;
        nc.hold();
        if (P.rows > 16) unit_rows<D, F32, NR>(geo, J, lds, nc, U, P, (int)gridDim.x, l, w);
        else unit_tokens<D, F32, 1>(geo, J, lds, Lanes<D / 64>(l), nc, U, P, (int)gridDim.x, l, w);
    });
}

// Parts k, k + step, .. of `n` joined, eight at a time (their loads in flight together): M, l and 4
// dims of O.
struct Joined {
    float m, l;
    v4f o;
};
template <class ML, class O>
__device__ __forceinline__ Joined join_parts(int k, int step, int n, const ML &ml, const O &sums)
{
    Joined j = {kMInit, 0.0f, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
    for (; k < n; k += 8 * step) {
        float2 x[8];
        v4f v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = k + i * step;
            x[i] = ml(min(at, n - 1));
            v[i] = sums(min(at, n - 1));
            if (at >= n) x[i].y = 0.0f;
        }
        float top = j.m;
#pragma unroll
        for (int i = 0; i < 8; i++) top = x[i].y != 0.0f ? fmaxf(top, x[i].x) : top;      // (0: nothing seen there)
        const float was = __builtin_amdgcn_exp2f(j.m - top), half = __builtin_amdgcn_exp2f(0.5f * (j.m - top));
        j.l = j.l * half * half;
#pragma unroll
        for (int e = 0; e < 4; e++) j.o[e] *= was;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (x[i].y == 0.0f) continue;
            const float al = __builtin_amdgcn_exp2f(x[i].x - top), h = __builtin_amdgcn_exp2f(0.5f * (x[i].x - top));
            j.l = fmaf(h * x[i].y, h, j.l);
#pragma unroll
            for (int e = 0; e < 4; e++) j.o[e] = fmaf(al, v[i][e], j.o[e]);
        }
        j.m = top;
    }
    return j;
}

// The parts of units that were cut, joined: a block for each 16 rows of a cut, 4 dims and a row to
// a thread.  Fewer rows: several threads to these, each with a share of the parts.
template <int D, bool F32>
__global__ __launch_bounds__(D * 4) void paged_join_kernel(PagedJob J, int grid)
{
    __shared__ float2 sml[D * 4];
    __shared__ v4f so[D * 4];
    const int b = line_block((int)blockIdx.x, grid), tid = threadIdx.x, dim = tid % (D / 4) * 4, slot = tid / (D / 4);
    const PagedCut c = J.cut[b];
    const int rows = min(16, c.rows - 16 * (int)blockIdx.y);
    if (c.n == 0 || rows <= 0) return;
    // (up to 16 parts by one thread: 1 us less than their sharing costs)
    const int log2r = c.n <= 16 ? 4 : rows <= 1 ? 0 : 32 - __clz(rows - 1), rp = 1 << log2r, groups = 16 >> log2r;
    const int r = slot & (rp - 1), j = 16 * (int)blockIdx.y + r;
    if (groups == 1 && r >= rows) return;
    const float *po = J.part, *pm = J.part + (int64_t)grid * 2 * J.rbr * D;
    auto row = [&](int k) { return (int64_t)(k ? 2 * (b + k) : 2 * b + 1) * J.rbr + j; };
    Joined y = join_parts(slot >> log2r, groups, c.n, [&](int k) { return *(const float2 *)(pm + row(k) * 2); },
                          [&](int k) { return *(const v4f *)(po + row(k) * D + dim); });
    if (groups > 1) {
        sml[tid] = float2{y.m, y.l};
        so[tid] = y.o;
        __syncthreads();
        if (slot >= rp) return;
        y = join_parts(0, 1, groups, [&](int k) { return sml[tid + k * rp * (D / 4)]; },
                       [&](int k) { return so[tid + k * rp * (D / 4)]; });
    }
    if (r >= rows) return;
    const float inv = y.l == 0.0f ? 0.0f : 1.0f / y.l;
    const float out[4] = {y.o[0] * inv, y.o[1] * inv, y.o[2] * inv, y.o[3] * inv};
    const int t = J.hb == 1 ? j / J.qpk : 0;
    store4<F32>(J.out, (int64_t)(c.tok + t) * J.ld_out + (int64_t)(c.head + j - t * J.qpk) * D + dim,
                J.vec & 2, out);
}

struct PagedPlan {
    int nr, rbr, grid, mixed, whole;
    size_t part, bytes;
};

// Units of 16 rows where no sequence has more, else of 32, or, where the work is large (a wave's
// share is 128 sub-tiles of 16 rows or more), of four waves' kMany tiles.  (bf16 of 32Q/4KV, d = 64, to
// 6001: 128 tokens of one sequence 36 us against 54, 64 x 8 52 against 57, 500 of one 89 against 79, 1500 x
// 4 480 against 289; d = 128, 8 kv heads: 48 x 8 59 against 74, 128 x 8 115 against 111, 1500 x 4 677 against
// 485.)
PagedPlan paged_plan(const eakvd_geom *g, const eakvd_pages *b, int n_q, int n_kv, bool bf16)
{
    PagedPlan p;
    const int qpk = n_q / n_kv;
    const int64_t rows = (int64_t)b->max_new * qpk;
    const int many = g->head_dim == 64 ? (bf16 ? kMany<64, false> : kMany<64, true>)
                                       : (bf16 ? kMany<128, false> : kMany<128, true>);
    p.mixed = rows > 32 && (double)b->n_new * n_q * b->max_len > 0x1p27;
    p.nr = rows <= 16 ? 1 : p.mixed ? many : 2;
    p.rbr = 16 * p.nr * (p.mixed ? kWaves : 1);
    const int rbr = p.rbr, tb = qpk < rbr ? rbr / qpk : 1, hb = (qpk + rbr - 1) / rbr;
    // units at most
    const int64_t units = (b->n_new / tb + (int64_t)(b->n_seqs < b->n_new ? b->n_seqs : b->n_new)) *
                          hb * n_kv;
    const int tile = p.mixed ? kRowsTile : kTile;
    const int64_t tiles = ((int64_t)b->max_len + (1 << tile) - 1) >> tile;
    // (two tiles stay together: the joining launch costs more)
    p.whole = !p.mixed && tiles <= 2;
    const int64_t most = units * (p.whole ? 1 : tiles > 1 ? tiles : 1), slots = (p.nr == 1 ? 3 : 2) * cu_count();
    p.grid = (int)(most < slots ? most : slots);
    p.part = ((size_t)p.grid * 2 * rbr * (g->head_dim + 2) * sizeof(float) + 255) & ~(size_t)255;
    p.bytes = p.whole ? 0 : p.part + (size_t)p.grid * sizeof(PagedCut);
    return p;
}

template <int D, bool F32, int NR, bool MIXED>
int launch(const eakvd_geom &g, PagedJob &J, const PagedPlan &p, hipStream_t st)
{
    constexpr size_t line0 = MIXED ? kRowsLds<D, F32> : Form<D, F32, MIXED ? 1 : NR>::kLine;
    static_assert(line0 + (EAKVD_PAGED_SEQS + 1) * 4 <= 160 * 1024, "LDS");
    void (*kern)(eakvd_geom, PagedJob);
    if constexpr (MIXED) kern = paged_rows_kernel<D, F32, NR>;
    else kern = paged_kernel<D, F32, NR>;
    static std::atomic<uint64_t> done;
    const int e = allow_lds((const void *)kern, line0 + (EAKVD_PAGED_SEQS + 1) * 4, done);
    if (e) return e;
    const size_t line = (J.b.n_seqs <= kFew ? 5 * kFew : J.b.n_seqs + 1) * 4;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.grid), dim3(64 * kWaves), line0 + line, st, g, J);
    if (!p.whole)
        hipLaunchKernelGGL((paged_join_kernel<D, F32>), dim3((unsigned)p.grid, (unsigned)(p.rbr / 16)), dim3(D * 4), 0,
                           st, J, p.grid);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" size_t eakvd_paged_work_bytes(const eakvd_geom *g, const eakvd_pages *b, int n_q, int n_kv, int bf16)
{
    return paged_plan(g, b, n_q, n_kv, bf16).bytes;
}

extern "C" int eakvd_paged_attend(const eakvd_geom *g, const uint8_t *base, const eakvd_pages *b,
                                  int layer, const void *q, int64_t ld_q, int bf16, int n_q, int n_kv,
                                  void *out, int64_t ld_out, void *work, void *stream)
{
    const PagedPlan p = paged_plan(g, b, n_q, n_kv, bf16);
    if (p.grid == 0) return 0;
    PagedJob J;
    memset(&J, 0, sizeof(J));
    J.b = *b;
    J.base = base;
    J.layer = layer;
    J.log2p = __builtin_ctz((unsigned)b->page_tokens);
    J.n_pages = g->max_seq_len >> J.log2p;
    J.n_q = n_q;
    J.n_kv = n_kv;
    J.qpk = n_q / n_kv;
    J.rbr = p.rbr;
    J.mixed = p.mixed;
    J.qinv = 65536 / J.qpk + 1;             // (r < 256, qpk <= 256)
    J.tb = J.qpk < J.rbr ? J.rbr / J.qpk : 1;
    J.hb = (J.qpk + J.rbr - 1) / J.rbr;
    J.whole = p.whole;
    J.q = q;
    J.out = out;
    J.ld_q = ld_q;
    J.ld_out = ld_out;
    J.ksc = EAKV_LOG2E / sqrtf((float)g->head_dim);
    // 16-byte loads of q, 16- or 8-byte stores of out
    const int64_t per = bf16 ? 8 : 4;
    J.vec = ((uintptr_t)q % 16 == 0 && ld_q % per == 0 ? 1 : 0) |
            ((uintptr_t)out % 16 == 0 && ld_out % per == 0 ? 2 : 0);
    J.part = (float *)work;
    J.cut = (PagedCut *)((uint8_t *)work + p.part);
    const hipStream_t st = (hipStream_t)stream;
    auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto by_type = [&](auto f32) {
            constexpr bool F = decltype(f32)::value;
            return p.mixed     ? launch<D, F, kMany<D, F>, true>(*g, J, p, st)
                   : p.nr == 1 ? launch<D, F, 1, false>(*g, J, p, st)
                               : launch<D, F, 2, false>(*g, J, p, st);
        };
        return bf16 ? by_type(std::false_type()) : by_type(std::true_type());
    };
    return g->head_dim == 64 ? run(std::integral_constant<int, 64>()) : run(std::integral_constant<int, 128>());
}
