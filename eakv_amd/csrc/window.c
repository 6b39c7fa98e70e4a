/* window.c — attention of several new tokens of each sequence (host C11):
 * validation, ordering and workspace around eakvd_window_attend; windows of one
 * f32 token take the decode launch (eakvd_fused). */
#include <string.h>

#include "internal.h"

int eakvi_window_check(eakv_cache_t *const *caches, int n, int layer, const int32_t *starts,
                       const int32_t *n_tokens, int dtype, int n_q, int n_kv, int tree,
                       eakvd_window *b, int64_t *total)
{
    if (!caches || n <= 0 || n > EAKVD_MAX_BATCH || !n_tokens)
        return eakvi_set_error(EAKV_ERR_INVALID, "window: invalid argument");
    if (dtype != EAKV_F32 && dtype != EAKV_BF16)
        return eakvi_set_error(EAKV_ERR_INVALID, "window: dtype %d not EAKV_F32 or EAKV_BF16",
                               dtype);
    int rc = eakvi_same_batch(caches, n, "window");
    if (rc == EAKV_OK) rc = eakvi_attn_check(caches[0], layer, n_q, n_kv);
    if (rc) return rc;
    memset(b, 0, sizeof(*b));
    b->n_seq = n;
    *total = 0;
    for (int i = 0; i < n; i++) {
        const eakv_cache_t *c = caches[i];
        const int32_t s = starts ? starts[i] : c->seq_len, m = n_tokens[i];
        if (m < 0 || s < 0 || s > c->seq_len || (int64_t)s + m > c->max_seq_len)
            return eakvi_set_error(EAKV_ERR_INVALID,
                                  "window: %d tokens at %d of a cache with %d tokens and room "
                                  "for %d", m, s, c->seq_len, c->max_seq_len);
        if (tree && m > EAKV_TREE_MAX)
            return eakvi_set_error(EAKV_ERR_INVALID, "window: a tree of %d tokens, at most %d",
                                  m, EAKV_TREE_MAX);
        b->base[i] = c->dev;
        b->start[i] = s;
        b->ntok[i] = m;
        *total += m;
    }
    if (*total * n_q > INT32_MAX / 2)
        return eakvi_set_error(EAKV_ERR_INVALID, "window: %lld rows in one call",
                              (long long)(*total * n_q));
    return EAKV_OK;
}

/* One f32 token of every sequence, without a tree, is a decode step. */
static int is_decode(const eakvd_window *b, int dtype, int tree, eakvd_batch *d)
{
    if (dtype != EAKV_F32 || tree) return 0;
    memset(d, 0, sizeof(*d));
    d->n_seq = b->n_seq;
    for (int i = 0; i < b->n_seq; i++) {
        if (b->ntok[i] != 1) return 0;
        d->base[i] = b->base[i];
        d->seq_len[i] = b->start[i] + 1;
    }
    return 1;
}

size_t eakv_attention_window_work_bytes(eakv_cache_t *const *caches, int n_caches,
                                        const int32_t *starts, const int32_t *n_tokens, int dtype,
                                        int n_q, int n_kv)
{
    eakvd_window b;
    eakvd_batch d;
    int64_t total;
    if (eakvi_window_check(caches, n_caches, 0, starts, n_tokens, dtype, n_q, n_kv, 0, &b, &total))
        return 0;
    int prev;
    if (eakvi_enter(caches[0], &prev)) return 0;
    size_t need = eakvd_window_work_bytes(&caches[0]->geom, &b, n_q, n_kv,
                                          dtype == EAKV_BF16);
    /* with a tree one token of each sequence is a window like others */
    if (is_decode(&b, dtype, 0, &d)) {
        const size_t dec = eakvd_fused_launch_bytes(&caches[0]->geom, &d, n_q, n_kv);
        if (dec > need) need = dec;
    }
    eakvi_leave(prev);
    return need;
}

int eakv_attention_window_batch_device(eakv_cache_t *const *caches, int n_caches, int layer,
                                       const int32_t *starts, const int32_t *n_tokens,
                                       const void *d_q, int dtype, int n_q, int n_kv,
                                       const uint64_t *d_tree, void *d_out, void *d_work,
                                       size_t work_bytes, void *stream)
{
    eakvd_window b;
    eakvd_batch d;
    int64_t total;
    int rc = eakvi_window_check(caches, n_caches, layer, starts, n_tokens, dtype, n_q, n_kv,
                                d_tree != NULL, &b, &total);
    if (rc) return rc;
    if (total == 0) return EAKV_OK;
    const uintptr_t odd = dtype == EAKV_F32 ? 3 : 1;
    if (!d_q || !d_out || ((uintptr_t)d_q | (uintptr_t)d_out) & odd || (uintptr_t)d_tree & 7 ||
        (uintptr_t)d_work & 15)
        return eakvi_set_error(EAKV_ERR_INVALID, "window: NULL or misaligned buffer");
    eakv_cache_t *c0 = caches[0];
    int prev;
    rc = eakvi_enter(c0, &prev);
    if (rc) return rc;
    const int decode = is_decode(&b, dtype, d_tree != NULL, &d);
    const size_t need = decode ? eakvd_fused_launch_bytes(&c0->geom, &d, n_q, n_kv)
                               : eakvd_window_work_bytes(&c0->geom, &b, n_q, n_kv,
                                                         dtype == EAKV_BF16);
    const int own = !d_work;
    int capturing = 0;
    const size_t rows = (size_t)total * n_q * c0->head_dim * (dtype == EAKV_F32 ? 4 : 2);
    const eakvi_span q = {d_q, rows}, out = {d_out, rows}, work_span = {d_work, need},
                     words = {d_tree, (size_t)total * 8};
    if (d_work && work_bytes < need) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "window: %zu bytes of workspace, %zu needed",
                             work_bytes, need);
    } else if (eakvi_overlap(out, words) || eakvi_overlap(work_span, q) ||
               eakvi_overlap(work_span, out) || eakvi_overlap(work_span, words)) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "window: overlapping buffers");
    } else {
        int e = eakvd_stream_capturing(stream ? stream : c0->stream, &capturing);
        if (e) rc = eakvi_hip_fail(e, "window");
        /* a graph would keep the address of a workspace that later calls
         * replace and share */
        else if (capturing && own && need)
            rc = eakvi_set_error(EAKV_ERR_INVALID,
                                 "window: a captured call needs a workspace of its own");
    }
    if (rc) {
        eakvi_leave(prev);
        return rc;
    }
    void *st = eakvi_batch_stream(caches, n_caches, stream);
    /* a caller's stream: after the work pending for each cache on the shared
     * stream.  A captured call cannot wait for work outside its graph: the
     * caller has the caches' work done before a replay. */
    for (int i = 0; rc == EAKV_OK && !capturing && i < n_caches; i++)
        rc = eakvi_order_before(caches[i], st);
    const int uses = own && need;
    if (rc == EAKV_OK && uses) rc = eakvi_work_begin(c0, st, need);
    if (rc == EAKV_OK) {
        void *work = own ? c0->work : d_work;
        /* the chunk counters belong to the cache's workspace */
        int e = decode ? eakvd_fused(&c0->geom, &d, layer, d_q, n_q, n_kv, d_out, work,
                                     uses ? c0->dev + c0->geom.ctr_off : NULL, st)
                       : eakvd_window_attend(&c0->geom, &b, layer, d_q, dtype == EAKV_BF16, n_q,
                                             n_kv, d_tree, d_out, work, st);
        if (e) rc = eakvi_hip_fail(e, "window launch");
        if (uses) {
            int e2 = eakvi_work_end(c0, st);
            if (rc == EAKV_OK) rc = e2;
        }
    }
    eakvi_leave(prev);
    return rc;
}
