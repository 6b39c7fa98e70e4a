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
// K's operands are n - z, exact in f16 (z: the nibble nearest the value 0; bf16
// queries of few rows: 0, the nibbles' own bits as subnormal f16, whose sums over a group are good
// to 2^-11 of a step times the largest of q, see nib_sub): score = sum over groups of
// s*(q.(n - z)) + c*sum(q), c = b + z*s, with s applied to the f32 dots and the c terms
// computed by one bf16 product of three pieces each (24 bits).
// Few rows: each wave makes the operands it needs in registers (window_draft.hip).
// Many: all are made once, in memory, and read from there (window_prompt.hip).
//
// Two arithmetics:
//   f32 queries   Q and the weights p*s are pairs of f16 (24 bits together),
//                 V's operands n - z; its c terms are f32 sums of p*c.
//   bf16 queries  Q (8 bits) is exact in f16.  V is dequantized to f16,
//                 (n - z)*s + c with s and c rounded to f16, and p is rounded
//                 to f16: 2^-12 relative each, against the output's 2^-9 (2e-4 of the
//                 outputs' norm before that rounding, 1.7e-3 after).
// f16's range: Q rows are scaled by a power of two to below 2^15, and each token of V by
// 2^-e of its own, e the exponent of its largest scale (f32) or value (bf16).  Its weight
// carries the 2^e: e is added to its scores by two spare terms of the c terms' product, so
// the softmax's reference point M bounds p*2^e of the tokens that a row sees, and nothing
// else has a part in it; weight operands stay below 2^15 and keep their precision down
// to 2^-29 of the largest.  (With one exponent for the 32 tokens of a sub-tile, one of
// them 10^8 times the others made rows 4e-3 off that did not even see it.)  bf16: the
// same product takes M off, so scores come out as exponents.
//
// Softmax in the log2 domain, f32: M moves only when a row's exponents pass it by
// kWinTop + kWinTau; sums, weighted sums and M are f32.  Tokens are split into chunks where
// rows alone do not fill the chip; partial (O, M, l) are merged by a second
// launch.  No atomics: results are the same bits on every call.
#include <string.h>

#include "window.h"

namespace {

// The chunks' (O, M, l) of a row (window token, q head) joined, d/4 lanes to a row of
// the sequences with chunks.  A chunk without visible tokens has l = 0 and no O.  A lane
// reads one chunk's M and l, so that the loads of O, 16 bytes each, wait for nothing but
// these.  Bound by HBM for many rows (37 MB of partials 12.8 us; a row to a wave, 4 bytes
// to a lane 23.6), else a dependent launch of 3 to 5 us.
template <int D, bool F32>
__global__ __launch_bounds__(256) void window_merge_kernel(WinJob job, const float *part,
                                                           void *out, int n_rows, int vec)
{
    constexpr int W = D / 4, RPW = 64 / W;           // lanes of a row, rows of a wave
    const int lane = threadIdx.x & 63, sub = lane % W;
    const int r0 = ((int)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane / W;
    const int r = min(r0, n_rows - 1), tok = r / job.n_q;
    int c = 0;
    for (int i = 1; i < job.n_seq; i++) c += tok >= job.lead[i] ? 1 : 0;
    const int mc = job.mc[c];
    int most = mc;                                   // of the wave's rows
#pragma unroll
    for (int o = W; o < 64; o *= 2) most = max(most, __shfl_xor(most, o, 64));
    if (most == 1) return;
    const int64_t per = (int64_t)job.ntok[c] * job.n_q;
    const int64_t local = r - (int64_t)job.lead[c] * job.n_q;
    // (a row of one chunk has no partial: it reads another's and writes nothing)
    const int64_t first = mc > 1 ? job.part[c] + local : 0;
    const float2 *ml = (const float2 *)(part + job.part_rows * D) + first;
    float m = kMInit;
    for (int k = sub; k < most; k += W) {
        const float2 x = ml[min(k, mc - 1) * per];
        if (x.y != 0.0f) m = fmaxf(m, x.x);
    }
#pragma unroll
    for (int o = 1; o < W; o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
    float l = 0.0f;
    v4f o4 = {0.0f, 0.0f, 0.0f, 0.0f};
    const float *po = part + first * D + sub * 4;
    for (int k0 = 0; k0 < most; k0 += W) {
        const float2 x = ml[min(k0 + sub, mc - 1) * per];
        // (-1: nothing there.  A factor that comes out 0 still takes its chunk's NaN along.)
        const float al = k0 + sub < mc && x.y != 0.0f ? __builtin_amdgcn_exp2f(x.x - m) : -1.0f;
        const float half = __builtin_amdgcn_exp2f(0.5f * (x.x - m));     // (as Soft::rescale)
        l = al < 0.0f ? l : fmaf(half * x.y, half, l);
        for (int k8 = k0; k8 < min(k0 + W, most); k8 += 8) {
            v4f v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = *(const v4f *)(po + min(k8 + k, mc - 1) * per * D);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float a = __shfl(al, lane - sub + k8 - k0 + k, 64);
#pragma unroll
                for (int e = 0; e < 4; e++) o4[e] = a < 0.0f ? o4[e] : fmaf(a, v[k][e], o4[e]);
            }
        }
    }
#pragma unroll
    for (int o = 1; o < W; o *= 2) l += __shfl_xor(l, o, 64);
    if (r0 >= n_rows || mc == 1) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float y[4] = {o4[0] * inv, o4[1] * inv, o4[2] * inv, o4[3] * inv};
    store4<F32>(out, ((int64_t)job.tok0[c] * job.n_q + local) * D + sub * 4, vec, y);
}

// The sequences of one launch: those of few rows (win_draft) or of many (win_prompt).
struct WinPart {
    WinJob job;
    int n_tok;              // window tokens of its sequences
    int64_t subtiles;       // win_prompt: expanded
    size_t part_bytes, bytes;
    double us;              // estimated
    bool merge;
};

struct WinPlan {
    WinPart few, many;
};

constexpr size_t kManyMost = (size_t)4 << 30;

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Tiles of a chunk, win_draft: an even share of the chip (4 tokens at 2048 of 32Q/8KV,
// 8 tiles: one each 16.6 us, two each 17.3, four each 19.9).  At most 2^25 tokens:
// offsets from a chunk's first token are 32 bits.
int64_t few_share(int64_t tiles, int cus)
{
    const int64_t s = (tiles + cus - 1) / cus, most = (1 << 25) / kDraftTile;
    return s < most ? s : most;
}

// Tiles of a chunk, win_prompt: the split of the longest context in k that ends first,
// by a model of a launch in tile times (256 rows x 32 tokens).  Blocks beyond the
// chip's slots run as slots come free, the longest first; partials are written and
// read at about 5 TB/s, the merge is a launch of its own.  us: of that split.
int64_t many_share(const WinJob &j, int64_t tiles, int cus, int head_dim, bool bf16, double *us)
{
    int64_t longest = 1, blocks = 0, rows = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t n_t = ((int64_t)j.start[i] + j.ntok[i] + 31) / 32;
        const int64_t r = (int64_t)j.ntok[i] * j.qpk;
        longest = n_t > longest ? n_t : longest;
        blocks += (r + 255) / 256 * j.n_kv;
        rows += r * j.n_kv;
    }
    const double tile_us = head_dim == 128 ? (bf16 ? 1.05 : 2.2) : (bf16 ? 0.68 : 1.3);
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
    *us = best * tile_us;
    return share;
}

// The sequences with in[i] as one launch, by way of the expanded operands or without.
// p->us: about what it takes.
void plan_part(const eakvd_geom *g, const eakvd_window *b, int n_q, int n_kv, bool bf16, bool many,
               const bool *in, WinPart *p)
{
    memset(p, 0, sizeof(*p));
    WinJob &j = p->job;
    const int qpk = n_q / n_kv;
    j.n_q = n_q;
    j.n_kv = n_kv;
    j.qpk = qpk;
    int tok0 = 0;
    for (int i = 0; i < b->n_seq; i++) {
        if (b->ntok[i] && in[i]) {
            const int k = j.n_seq++;
            j.base[k] = b->base[i];
            j.start[k] = b->start[i];
            j.ntok[k] = b->ntok[i];
            j.tok0[k] = tok0;
        }
        tok0 += b->ntok[i];
    }
    if (j.n_seq == 0) return;
    const int rbr = many ? 256 : 32, tile = many ? 32 : kDraftTile;
    // tiles of all blocks, were no sequence split (the mean of a sequence's first and last
    // row block; a tree's rows may all see the whole window, which is short)
    int64_t tiles = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t rows = (int64_t)j.ntok[i] * qpk, nrb = (rows + rbr - 1) / rbr;
        const int64_t first = (j.start[i] + (int64_t)(rows < rbr ? rows : rbr) / qpk + tile) / tile;
        const int64_t last = ((int64_t)j.start[i] + j.ntok[i] + tile - 1) / tile;
        tiles += (nrb * (first + last) + 1) / 2 * n_kv;
    }
    const int cus = cu_count();
    const int64_t share = many ? many_share(j, tiles, cus, g->head_dim, bf16, &p->us)
                               : few_share(tiles, cus);
    int64_t part = 0, longest = 0;
    for (int i = 0; i < j.n_seq; i++) {
        const int64_t rows = (int64_t)j.ntok[i] * qpk, nrb = (rows + rbr - 1) / rbr;
        const int64_t n_t = ((int64_t)j.start[i] + j.ntok[i] + tile - 1) / tile;
        // (two tiles stay together: at 500 tokens 13.0 us against 15.2 with the joining launch)
        int64_t mc = !many && n_t <= 2 ? 1 : (n_t + share - 1) / share;
        const int64_t per = (n_t + mc - 1) / mc;
        mc = (n_t + per - 1) / per;
        longest = per > longest ? per : longest;
        j.mc[i] = (int)mc;
        j.clen[i] = (int)(per * tile < INT32_MAX ? per * tile : INT32_MAX);
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
    if (many) {
        // the expansion: a launch, and both forms of K and V at about 4 TB/s
        const size_t img = win_prompt_bytes(g->head_dim, bf16, p->subtiles);
        p->bytes += align256(img);
        p->us += 8 + 1.3 * img / 4e6;
    } else {
        const bool wide = g->head_dim == 128;
        const double tile_us = wide ? (bf16 ? 1.75 : 2.7) : (bf16 ? 1.05 : 1.35), block_us = wide ? 9 : 6;
        const int64_t blocks = j.pre[j.n_seq];
        const double even = (tiles * tile_us + blocks * block_us) / cus + 0.25 * longest * tile_us;
        const double one = longest * tile_us + block_us;
        p->us = (blocks > cus && even > one ? even : one) +
                (p->merge ? 6 + 2.0 * part * (g->head_dim + 2) * 4 / 5e6 : 0);
    }
}

// Whether windows' K and V are expanded first: causal ones that no tree is allowed for,
// of more than 512 rows per kv head, if both estimates say so and the operands, 3.5 times
// the packed planes at d = 128, stay below kManyMost (2.3 GB for 131072 tokens of 32 kv
// heads).  What the estimates choose between, in us, expanded / not: 2000 tokens at 2000 of
// 32Q/32KV bf16 92 / 121, f32 156 / 164, of 8Q/8KV 49 / 36, 64 / 50; 3000 at 3000 of 40Q/8KV
// 138 / 259, 238 / 365; 4000 at 4000 of 12Q/12KV, d = 64, 80 / 89, 134 / 116; 8 of 600 at
// 600 of 32Q/8KV 76 / 187, 117 / 235; 512 at 8192 109 / 120, 177 / 188; 4 of 150 at 20000
// 480 / 395, 690 / 627.  They are wrong by up to 40 % for some 800 rows at very long
// contexts (70 tokens at 131072 of 64Q/8KV, not expanded: 729 / 817, 1084 / 1308).
void win_plan(const eakvd_geom *g, const eakvd_window *b, int n_q, int n_kv, bool bf16, WinPlan *p)
{
    bool few[EAKVD_MAX_BATCH], many[EAKVD_MAX_BATCH], any = false;
    for (int i = 0; i < b->n_seq; i++) {
        many[i] = b->ntok[i] > EAKVD_TREE_MAX && (int64_t)b->ntok[i] * (n_q / n_kv) > 512;
        few[i] = !many[i];
        any = any || many[i];
    }
    memset(&p->many, 0, sizeof(p->many));
    if (any) {
        plan_part(g, b, n_q, n_kv, bf16, false, many, &p->few);
        plan_part(g, b, n_q, n_kv, bf16, true, many, &p->many);
        if (p->few.us < p->many.us || p->many.bytes > kManyMost) {
            memset(&p->many, 0, sizeof(p->many));
            for (int i = 0; i < b->n_seq; i++) few[i] = true;
        }
    }
    plan_part(g, b, n_q, n_kv, bf16, false, few, &p->few);
}

int merge(const eakvd_geom *g, const WinPart &p, bool bf16, const float *part, void *out, bool vec,
          hipStream_t st)
{
    if (!p.merge) return 0;
    const int n_rows = p.n_tok * p.job.n_q, per = 4 * 256 / g->head_dim;
    auto *kern = g->head_dim == 64
                     ? (bf16 ? window_merge_kernel<64, false> : window_merge_kernel<64, true>)
                     : (bf16 ? window_merge_kernel<128, false> : window_merge_kernel<128, true>);
    hipLaunchKernelGGL(kern, dim3((unsigned)((n_rows + per - 1) / per)), dim3(256), 0, st, p.job,
                       part, out, n_rows, (int)vec);
    return (int)hipGetLastError();
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
        if (!e) e = merge(g, p.many, bf16, (const float *)w, out, vec, st);
        w += p.many.bytes;
    }
    if (!e && p.few.job.n_seq) {
        float *part = (float *)w;
        e = win_draft(*g, p.few.job, bf16, q, tree, out, part, vec, st);
        if (!e) e = merge(g, p.few, bf16, part, out, vec, st);
    }
    return e;
}
