// pages.h — sequences in pages of a pool, as the kernels read them from the device
// (paged.hip, pages.hip).
#pragma once

#include "common.h"

namespace {

struct Seq {
    int row, n, pos;        // first row, new tokens, the first one's position
};

// Sequence s, every value held to the call's bounds.
__device__ __forceinline__ Seq seq_at(const eakvd_pages &b, int s)
{
    const int a = b.first ? b.first[s] : (int)min((int64_t)s * b.max_new, (int64_t)b.n_new);
    const int e = b.first ? b.first[s + 1] : (int)min((int64_t)a + b.max_new, (int64_t)b.n_new);
    Seq q;
    q.row = min(max(a, 0), b.n_new);
    q.n = min(min(max(e, q.row), b.n_new) - q.row, b.max_new);
    q.pos = min(max(b.lens[s], 0), b.max_len) - q.n;
    return q;
}

// A list of rows that falls after sequence s: rows would be several sequences', and all of these
// together more than the host counted on.
__device__ __forceinline__ bool falls_at(const eakvd_pages &b, int s) { return b.first && b.first[s + 1] < b.first[s]; }

// Where position t (0 <= t < max_len) of a sequence is in the pool, or -1.
__device__ __forceinline__ int place_of(const int32_t *table, int t, int log2p, int n_pages)
{
    const int p = table[t >> log2p];
    return p >= 0 && p < n_pages ? (p << log2p) + (t & ((1 << log2p) - 1)) : -1;
}

}  // namespace
