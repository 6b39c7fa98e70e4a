// pages.hip — K and V of new tokens quantized into the pages that the sequences' tables
// name, both in one launch.  Rows are [token][kv head][dim], f32 or bf16, as a model's
// projections leave them; codes, scales and biases are bit for bit those of quantize.hip.
//
// A block takes 16 tokens (d = 64: 32) of some kv heads: a head's groups are contiguous in a page,
// where it writes, and 256 to 512 bytes a token where it reads.  While the first head's values
// are on their way its waves find each token's sequence and place, 64 row numbers at a time
// (two loads for up to 4096 sequences); 8 lanes quantize a group.  Bound by a launch's latency
// for a decode step (64 sequences, 8 heads, bf16: 4.6 us), by HBM for prompts (4000 tokens x 2, 32
// heads, f32: 59 us, 5.2 TB/s).
#include "pages.h"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kBlocks = 8192;

struct AppendJob {
    eakvd_pages b;
    uint8_t *base;
    int layer, n_pages, log2p;
    const void *src[2];
    int64_t ld;
    int heads, parts;       // heads (K's, then V's) of a block, blocks of a chunk of tokens
};

template <bool BF16, bool VEC>
__device__ __forceinline__ float4 load4(const void *src, int64_t at)
{
    if constexpr (BF16) {
        const uint16_t *p = (const uint16_t *)src + at;
        uint32_t x, y;
        if constexpr (VEC) {
            const uint2 v = *(const uint2 *)p;
            x = v.x;
            y = v.y;
        } else {
            x = p[0] | (uint32_t)p[1] << 16;
            y = p[2] | (uint32_t)p[3] << 16;
        }
        return make_float4(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u),
                           __uint_as_float(y << 16), __uint_as_float(y & 0xffff0000u));
    } else {
        const float *p = (const float *)src + at;
        if constexpr (VEC) {
            const v4f v = __builtin_nontemporal_load((const v4f *)p);
            return make_float4(v[0], v[1], v[2], v[3]);
        } else {
            return make_float4(p[0], p[1], p[2], p[3]);
        }
    }
}

template <int GPD, bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void append_kernel(eakvd_geom g, AppendJob J)
{
    constexpr int T = kThreads / 8 / GPD;            // tokens of a block
    __shared__ int place[T];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int chunk = (int)blockIdx.x / J.parts, part = (int)blockIdx.x - chunk * J.parts;
    const int r0 = chunk * T, n = J.b.n_seqs;
    const int l8 = tid & 7, gbase = lane & ~7, slot = tid >> 3;
    const int k8 = slot / GPD, gd = slot % GPD;
    const int y0 = part * J.heads, y1 = min(y0 + J.heads, 2 * g.n_kv_heads);
    // (rows behind the last are read as the last: the 8 lanes of a group, and the wave, go on together)
    const int64_t from = min(r0 + k8, J.b.n_new - 1) * J.ld + gd * 64 + l8 * 4;
    auto load = [&](int y, float4 &lo, float4 &hi) {
        const int kv = y >= g.n_kv_heads;
        const int64_t at = from + (int64_t)(y - kv * g.n_kv_heads) * g.head_dim;
        lo = load4<BF16, VEC>(J.src[kv], at);
        hi = load4<BF16, VEC>(J.src[kv], at + 32);
    };
    float4 lo, hi;
    load(y0, lo, hi);
    // the last sequence that does not begin behind row r
    auto begin = [&](int s) { return s < n ? seq_at(J.b, s).row : INT32_MAX; };
    const int coarse = n > 64 ? begin(lane * 64) : 0;
    for (int k = w; k < T; k += kThreads / 64) {
        const int r = r0 + k;
        if (r >= J.b.n_new) break;
        int s = n > 64 ? 64 * ((int)__popcll(__ballot(coarse <= r)) - 1) : 0;
        if (s < 0) s = 0;
        s += (int)__popcll(__ballot(begin(s + lane) <= r)) - 1;
        int at = -1;
        if (s >= 0) {
            const Seq q = seq_at(J.b, s);
            const int i = r - q.row, t = q.pos + i;
            if (i < q.n && t >= 0) at = place_of(J.b.tables + (int64_t)s * J.b.ld_table, t, J.log2p, J.n_pages);
        }
        if (lane == 0) place[k] = at;
    }
    __syncthreads();
    const int at = r0 + k8 < J.b.n_new ? place[k8] : -1;
    for (int y = y0; y < y1; y++) {
        float4 nlo = lo, nhi = hi;
        if (y + 1 < y1) load(y + 1, nlo, nhi);
        const QOut o = quantize_group8(lo, hi, gbase);
        if (at >= 0) {
            const int kv = y >= g.n_kv_heads;
            uint8_t *blk = J.base + (int64_t)(J.layer * 2 + kv) * g.block_bytes;
            const int64_t gi = (y - kv * g.n_kv_heads) * g.gph + (int64_t)at * GPD + gd;
            __builtin_nontemporal_store(o.word, (uint32_t *)(blk + gi * 32 + l8 * 4));
            if (l8 == 0) {
                __builtin_nontemporal_store(o.scale, (float *)(blk + g.s_off) + gi);
                __builtin_nontemporal_store(o.bias, (float *)(blk + g.b_off) + gi);
            }
        }
        lo = nlo;
        hi = nhi;
    }
}

int block_tokens(const eakvd_geom *g) { return kThreads / 8 / (int)g->gpd; }

}  // namespace

// (A launch has fewer than 2^32 threads; one of that many chunks gives a block all heads.)
extern "C" int64_t eakvd_paged_append_most(const eakvd_geom *g)
{
    return ((1ll << 32) / kThreads - 1) * block_tokens(g);
}

extern "C" int eakvd_paged_append(const eakvd_geom *g, uint8_t *base, const eakvd_pages *b, int layer,
                                  const void *k, const void *v, int64_t ld, int bf16, void *stream)
{
    if (b->n_new <= 0) return 0;
    AppendJob J;
    J.b = *b;
    J.base = base;
    J.layer = layer;
    J.log2p = __builtin_ctz((unsigned)b->page_tokens);
    J.n_pages = g->max_seq_len >> J.log2p;
    J.src[0] = k;
    J.src[1] = v;
    J.ld = ld;
    // 16-byte loads (bf16: 8)
    const uintptr_t odd = bf16 ? 7 : 15;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & odd) == 0 && ld % 4 == 0;
    const int t = block_tokens(g);
    // about kBlocks blocks, heads of the same tokens side by side
    const int64_t chunks = ((int64_t)b->n_new + t - 1) / t;
    const int all = 2 * g->n_kv_heads;
    int64_t parts = (kBlocks + chunks - 1) / chunks;
    if (parts > all) parts = all;
    J.heads = (int)((all + parts - 1) / parts);
    J.parts = (all + J.heads - 1) / J.heads;
    const dim3 grid((unsigned)(chunks * J.parts));
    auto run = [&](auto *kern) {
        hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, (hipStream_t)stream, *g, J);
        return (int)hipGetLastError();
    };
    if (g->gpd == 2) {
        if (bf16) return vec ? run(append_kernel<2, true, true>) : run(append_kernel<2, true, false>);
        return vec ? run(append_kernel<2, false, true>) : run(append_kernel<2, false, false>);
    }
    if (bf16) return vec ? run(append_kernel<1, true, true>) : run(append_kernel<1, true, false>);
    return vec ? run(append_kernel<1, false, true>) : run(append_kernel<1, false, false>);
}
