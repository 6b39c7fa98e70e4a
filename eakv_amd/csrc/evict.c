/* evict.c — eviction by attention weight (host C11): the weights that cached tokens get
 * (validation, ordering and workspace around eakvd_weights) and the choice of the tokens
 * that stay (on the HIP device current at the call). */
#include <string.h>

#include "internal.h"

size_t eakv_attention_weights_work_bytes(eakv_cache_t *const *caches, int n_caches, const int32_t *starts,
                                         const int32_t *n_tokens, int dtype, int n_q, int n_kv)
{
    eakvd_window b;
    int64_t total;
    if (eakvi_window_check(caches, n_caches, 0, starts, n_tokens, dtype, n_q, n_kv, 0, &b, &total)) return 0;
    int prev;
    if (eakvi_enter(caches[0], &prev)) return 0;
    const size_t need = eakvd_weights_work_bytes(&b, n_q, n_kv, dtype == EAKV_BF16);
    eakvi_leave(prev);
    return need;
}

int eakv_attention_weights_batch_device(eakv_cache_t *const *caches, int n_caches, int layer,
                                        const int32_t *starts, const int32_t *n_tokens, const void *d_q,
                                        int dtype, int n_q, int n_kv, float keep, float *d_weights,
                                        int64_t ld, void *d_work, size_t work_bytes, void *stream)
{
    eakvd_window b;
    int64_t total;
    int rc = eakvi_window_check(caches, n_caches, layer, starts, n_tokens, dtype, n_q, n_kv, 0, &b, &total);
    if (rc) return rc;
    int64_t most = 0;
    for (int i = 0; i < n_caches; i++) {
        const int64_t t = (int64_t)b.start[i] + b.ntok[i];
        if (!b.ntok[i]) continue;
        if (ld < t)
            return eakvi_set_error(EAKV_ERR_INVALID, "weights: rows of %lld for %lld tokens", (long long)ld,
                                   (long long)t);
        most = t > most ? t : most;
    }
    if (total == 0) return EAKV_OK;
    const uintptr_t odd = dtype == EAKV_F32 ? 3 : 1;
    if (!d_q || !d_weights || (uintptr_t)d_q & odd || (uintptr_t)d_weights & 3 || (uintptr_t)d_work & 15)
        return eakvi_set_error(EAKV_ERR_INVALID, "weights: NULL or misaligned buffer");
    eakv_cache_t *c0 = caches[0];
    int prev;
    rc = eakvi_enter(c0, &prev);
    if (rc) return rc;
    const size_t need = eakvd_weights_work_bytes(&b, n_q, n_kv, dtype == EAKV_BF16);
    const int own = !d_work;
    const eakvi_span q = {d_q, (size_t)total * n_q * c0->head_dim * (dtype == EAKV_F32 ? 4 : 2)},
                     out = {d_weights, eakvi_rows_bytes((int64_t)n_caches * n_kv, ld, most, 4)}, work = {d_work, need};
    int capturing = 0;
    if (d_work && work_bytes < need) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "weights: %zu bytes of workspace, %zu needed", work_bytes, need);
    } else if (eakvi_overlap(out, q) || eakvi_overlap(work, q) || eakvi_overlap(work, out)) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "weights: overlapping buffers");
    } else {
        int e = eakvd_stream_capturing(stream ? stream : c0->stream, &capturing);
        if (e) rc = eakvi_hip_fail(e, "weights");
        else if (capturing && own)
            rc = eakvi_set_error(EAKV_ERR_INVALID, "weights: a captured call needs a workspace of its own");
    }
    if (rc) {
        eakvi_leave(prev);
        return rc;
    }
    void *st = eakvi_batch_stream(caches, n_caches, stream);
    for (int i = 0; rc == EAKV_OK && !capturing && i < n_caches; i++) rc = eakvi_order_before(caches[i], st);
    if (rc == EAKV_OK && own) rc = eakvi_work_begin(c0, st, need);
    if (rc == EAKV_OK) {
        int e = eakvd_weights(&c0->geom, &b, layer, d_q, dtype == EAKV_BF16, n_q, n_kv, keep, d_weights, ld,
                              own ? c0->work : d_work, st);
        if (e) rc = eakvi_hip_fail(e, "weights launch");
        if (own) {
            int e2 = eakvi_work_end(c0, st);
            if (rc == EAKV_OK) rc = e2;
        }
    }
    eakvi_leave(prev);
    return rc;
}

/* the kernels' positions are 32 bits, with room for a block's behind the last */
#define MOST_TOKENS (1 << 30)

size_t eakv_evict_select_work_bytes(int n_seqs, const int32_t *n_tokens)
{
    int bad = n_seqs < 0 || n_seqs > EAKVD_MAX_BATCH || (n_seqs && !n_tokens);
    for (int i = 0; !bad && i < n_seqs; i++) bad = n_tokens[i] < 0 || n_tokens[i] > MOST_TOKENS;
    if (bad) {
        eakvi_set_error(EAKV_ERR_INVALID, "evict: invalid argument");
        return 0;
    }
    return eakvd_evict_work_bytes(n_seqs, n_tokens);
}

int eakv_evict_select_device(int n_seqs, int n_heads, const float *d_weights, int64_t ld,
                             const int32_t *n_tokens, int n_first, int n_recent, const int32_t *n_keep,
                             int32_t *d_index, float *d_kept, int64_t ld_kept, void *d_work,
                             size_t work_bytes, void *stream)
{
    if (n_seqs < 0 || n_seqs > EAKVD_MAX_BATCH || n_heads < 1 || n_heads > 65536 || n_first < 0 ||
        n_recent < 0 || (n_seqs && (!n_tokens || !n_keep)))
        return eakvi_set_error(EAKV_ERR_INVALID, "evict: invalid argument");
    eakvd_evict j;
    memset(&j, 0, sizeof(j));
    j.n_seq = n_seqs;
    j.n_heads = n_heads;
    j.n_first = n_first;
    j.n_recent = n_recent;
    int64_t total = 0, most = 0;
    for (int i = 0; i < n_seqs; i++) {
        const int64_t n = n_tokens[i], stay = (int64_t)n_first + n_recent;
        if (n < 0 || n > MOST_TOKENS || n_keep[i] < (stay < n ? stay : n) || n_keep[i] > n || ld < n ||
            (d_kept && ld_kept < n_keep[i]))
            return eakvi_set_error(EAKV_ERR_INVALID,
                                   "evict: %d of %lld tokens, %lld of them the first and last", n_keep[i],
                                   (long long)n, (long long)stay);
        j.n_tokens[i] = n_tokens[i];
        j.n_keep[i] = n_keep[i];
        j.first[i] = total;
        total += n_keep[i];
        most = n > most ? n : most;
    }
    if (n_seqs == 0 || (total == 0 && !d_kept)) return EAKV_OK;
    const size_t need = eakvd_evict_work_bytes(n_seqs, n_tokens);
    if (!d_weights || (total && !d_index) || (need && !d_work) ||
        ((uintptr_t)d_weights | (uintptr_t)d_index | (uintptr_t)d_kept | (uintptr_t)d_work) & 3)
        return eakvi_set_error(EAKV_ERR_INVALID, "evict: NULL or misaligned buffer");
    if (work_bytes < need)
        return eakvi_set_error(EAKV_ERR_INVALID, "evict: %zu bytes of workspace, %zu needed", work_bytes, need);
    const int64_t rows = (int64_t)n_seqs * n_heads;
    const eakvi_span in = {d_weights, eakvi_rows_bytes(rows, ld, most, 4)},
                     out[3] = {{d_index, (size_t)total * 4},
                               {d_kept, d_kept ? (size_t)rows * (size_t)ld_kept * 4 : 0},
                               {d_work, need}};
    for (int i = 0; i < 3; i++)
        if (eakvi_overlap(out[i], out[(i + 1) % 3]) || eakvi_overlap(out[i], in))
            return eakvi_set_error(EAKV_ERR_INVALID, "evict: overlapping buffers");
    int e = eakvd_evict_select(&j, d_weights, ld, d_index, d_kept, ld_kept, d_work, stream);
    return e ? eakvi_hip_fail(e, "evict launch") : EAKV_OK;
}
