/* paged.c — sequences in pages of a pool (host C11): K and V of new tokens quantized
 * into their pages, and attention over them.  Validation and ordering around
 * eakvd_paged_append and eakvd_paged_attend. */
#include <string.h>

#include "internal.h"

/* Positions and rows are 32 bits in the kernels, which look up to 64 sub-tiles behind a sequence's end
 * (and hold what they find there to it). */
#define MOST (INT32_MAX - 65535)

/* The batch against the pool: sizes, tables that hold the bound on lengths. */
static int batch_check(const eakv_cache_t *pool, const eakv_paged_batch_t *b, const char *what,
                       eakvd_pages *d)
{
    if (!pool || !b)
        return eakvi_set_error(EAKV_ERR_INVALID, "%s: invalid argument", what);
    if (pool->head_dim != 64 && pool->head_dim != 128)
        return eakvi_set_error(EAKV_ERR_INVALID, "%s: head_dim %d not 64 or 128", what, pool->head_dim);
    const int p = b->page_tokens;
    if (p < EAKV_PAGE_MIN || (p & (p - 1)) || p > pool->max_seq_len)
        return eakvi_set_error(EAKV_ERR_INVALID,
                               "%s: pages of %d tokens, a power of two from %d to the pool's %d wanted",
                               what, p, EAKV_PAGE_MIN, pool->max_seq_len);
    if (b->n_seqs < 0 || b->n_seqs > EAKV_PAGED_SEQS || b->n_new < 0 || b->max_new < 0 || b->max_len < 0)
        return eakvi_set_error(EAKV_ERR_INVALID, "%s: %d sequences, %d rows, at most %d new of %d tokens",
                               what, b->n_seqs, b->n_new, b->max_new, b->max_len);
    if (b->max_len > MOST || b->n_new > MOST)
        return eakvi_set_error(EAKV_ERR_INVALID, "%s: %d rows of up to %d tokens, %d at most", what, b->n_new,
                               b->max_len, MOST);
    /* the kernels' offsets from a kv head's first group are 32 bits */
    if ((int64_t)pool->geom.gph > INT32_MAX / 2)
        return eakvi_set_error(EAKV_ERR_INVALID, "%s: a pool of %d tokens", what, pool->max_seq_len);
    if (b->n_seqs && b->n_new) {
        if (!b->d_tables || !b->d_lens ||
            ((uintptr_t)b->d_tables | (uintptr_t)b->d_lens | (uintptr_t)b->d_first) & 3)
            return eakvi_set_error(EAKV_ERR_INVALID, "%s: NULL or misaligned table, lengths or rows", what);
        if (b->ld_table < ((int64_t)b->max_len + p - 1) / p)
            return eakvi_set_error(EAKV_ERR_INVALID, "%s: tables of %lld pages for %d tokens", what,
                                   (long long)b->ld_table, b->max_len);
    }
    d->n_seqs = b->n_seqs;
    d->page_tokens = p;
    d->n_new = b->n_new;
    d->max_new = b->max_new;
    d->max_len = b->max_len;
    d->tables = b->d_tables;
    d->lens = b->d_lens;
    d->first = b->d_first;
    d->ld_table = b->ld_table;
    return EAKV_OK;
}

static int nothing(const eakvd_pages *d) { return !d->n_seqs || !d->n_new || !d->max_new; }

/* The spans of a batch's own buffers. */
static void batch_spans(const eakvd_pages *d, eakvi_span *s)
{
    s[0] = (eakvi_span){d->tables, ((size_t)(d->n_seqs - 1) * (size_t)d->ld_table +
                                    (size_t)((d->max_len + (int64_t)d->page_tokens - 1) /
                                             d->page_tokens)) * 4};
    s[1] = (eakvi_span){d->lens, (size_t)d->n_seqs * 4};
    s[2] = (eakvi_span){d->first, d->first ? ((size_t)d->n_seqs + 1) * 4 : 0};
}

int eakv_append_paged_device(eakv_cache_t *pool, const eakv_paged_batch_t *b, int layer,
                             const void *d_k, const void *d_v, int dtype, int64_t ld, void *stream)
{
    eakvd_pages d;
    int rc = batch_check(pool, b, "append_paged", &d);
    if (rc) return rc;
    if (dtype != EAKV_F32 && dtype != EAKV_BF16)
        return eakvi_set_error(EAKV_ERR_INVALID, "append_paged: dtype %d not EAKV_F32 or EAKV_BF16", dtype);
    const int64_t width = (int64_t)pool->n_kv_heads * pool->head_dim;
    if (layer < 0 || layer >= pool->n_layers || ld < width)
        return eakvi_set_error(EAKV_ERR_INVALID, "append_paged: layer %d, %lld values from token to token",
                               layer, (long long)ld);
    if (nothing(&d)) return EAKV_OK;
    if (d.n_new > eakvd_paged_append_most(&pool->geom))
        return eakvi_set_error(EAKV_ERR_INVALID, "append_paged: %d rows, %lld at most", d.n_new,
                               (long long)eakvd_paged_append_most(&pool->geom));
    const uintptr_t odd = dtype == EAKV_F32 ? 3 : 1;
    if (!d_k || !d_v || ((uintptr_t)d_k | (uintptr_t)d_v) & odd)
        return eakvi_set_error(EAKV_ERR_INVALID, "append_paged: NULL or misaligned buffer");
    int prev;
    rc = eakvi_enter(pool, &prev);
    if (rc) return rc;
    int capturing = 0;
    int e = eakvd_stream_capturing(stream ? stream : pool->stream, &capturing);
    if (e) rc = eakvi_hip_fail(e, "append_paged");
    void *st = pool->stream;
    if (rc == EAKV_OK) {
        st = eakvi_stream_or_default(pool, stream);
        /* a captured call cannot wait for work outside its graph, nor later work for it */
        if (!capturing) rc = eakvi_order_before(pool, st);
    }
    if (rc == EAKV_OK) {
        e = eakvd_paged_append(&pool->geom, pool->dev, &d, layer, d_k, d_v, ld, dtype == EAKV_BF16, st);
        if (e) rc = eakvi_hip_fail(e, "append_paged launch");
    }
    if (rc == EAKV_OK && !capturing) rc = eakvi_order_after(&pool, 1, st);
    eakvi_leave(prev);
    return rc;
}

/* The head split, and that the work's line fits 32 bits. */
static int heads_check(const eakv_cache_t *pool, const eakvd_pages *d, int n_q, int n_kv, int dtype)
{
    if (dtype != EAKV_F32 && dtype != EAKV_BF16)
        return eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: dtype %d not EAKV_F32 or EAKV_BF16",
                               dtype);
    int rc = eakvi_attn_check(pool, 0, n_q, n_kv);
    if (rc) return rc;
    /* row blocks have 16 rows or more, but for a sequence's last; tiles 64 tokens */
    const int64_t seqs = d->n_seqs < d->n_new ? d->n_seqs : d->n_new;
    const int64_t units = (int64_t)d->n_new * n_q / 16 + seqs * n_q;
    const int64_t tiles = (int64_t)d->max_len / 64 + 1;
    if (units > INT32_MAX || units * tiles > INT32_MAX)
        return eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: %d rows of up to %d tokens in one call",
                               d->n_new, d->max_len);
    return EAKV_OK;
}

size_t eakv_attention_paged_work_bytes(const eakv_cache_t *pool, const eakv_paged_batch_t *b, int dtype,
                                       int n_q, int n_kv)
{
    eakvd_pages d;
    if (batch_check(pool, b, "attention_paged", &d) || heads_check(pool, &d, n_q, n_kv, dtype) ||
        nothing(&d))
        return 0;
    int prev;
    if (eakvi_enter(pool, &prev)) return 0;
    const size_t need = eakvd_paged_work_bytes(&pool->geom, &d, n_q, n_kv, dtype == EAKV_BF16);
    eakvi_leave(prev);
    return need;
}

int eakv_attention_paged_device(const eakv_cache_t *cpool, const eakv_paged_batch_t *b, int layer,
                                const void *d_q, int64_t ld_q, int dtype, int n_q, int n_kv, void *d_out,
                                int64_t ld_out, void *d_work, size_t work_bytes, void *stream)
{
    eakv_cache_t *pool = (eakv_cache_t *)cpool;
    eakvd_pages d;
    int rc = batch_check(pool, b, "attention_paged", &d);
    if (rc == EAKV_OK) rc = heads_check(pool, &d, n_q, n_kv, dtype);
    if (rc == EAKV_OK) rc = eakvi_attn_check(pool, layer, n_q, n_kv);
    if (rc) return rc;
    const int64_t width = (int64_t)n_q * pool->head_dim;
    if (ld_q < width || ld_out < width)
        return eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: %lld and %lld values from token to token",
                               (long long)ld_q, (long long)ld_out);
    if (nothing(&d)) return EAKV_OK;
    const uintptr_t odd = dtype == EAKV_F32 ? 3 : 1;
    if (!d_q || !d_out || ((uintptr_t)d_q | (uintptr_t)d_out) & odd || (uintptr_t)d_work & 15)
        return eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: NULL or misaligned buffer");
    int prev;
    rc = eakvi_enter(pool, &prev);
    if (rc) return rc;
    const size_t need = eakvd_paged_work_bytes(&pool->geom, &d, n_q, n_kv, dtype == EAKV_BF16);
    const size_t size = dtype == EAKV_F32 ? 4 : 2;
    const int own = !d_work && need;
    const eakvi_span q = {d_q, eakvi_rows_bytes(d.n_new, ld_q, width, size)},
                     out = {d_out, eakvi_rows_bytes(d.n_new, ld_out, width, size)}, work = {d_work, need};
    eakvi_span in[3];
    batch_spans(&d, in);
    /* a row is written when its own query has been read, others may not have been */
    int bad = eakvi_overlap(work, q) || eakvi_overlap(work, out) ||
              (eakvi_overlap(q, out) && (d_q != d_out || ld_q != ld_out));
    for (int i = 0; i < 3; i++) bad |= eakvi_overlap(in[i], out) || eakvi_overlap(in[i], work);
    int capturing = 0;
    if (d_work && work_bytes < need) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: %zu bytes of workspace, %zu needed",
                             work_bytes, need);
    } else if (bad) {
        rc = eakvi_set_error(EAKV_ERR_INVALID, "attention_paged: overlapping buffers");
    } else {
        int e = eakvd_stream_capturing(stream ? stream : pool->stream, &capturing);
        if (e) rc = eakvi_hip_fail(e, "attention_paged");
        else if (capturing && own)
            rc = eakvi_set_error(EAKV_ERR_INVALID,
                                 "attention_paged: a captured call needs a workspace of its own");
    }
    if (rc) {
        eakvi_leave(prev);
        return rc;
    }
    void *st = eakvi_batch_stream(&pool, 1, stream);
    if (!capturing) rc = eakvi_order_before(pool, st);
    if (rc == EAKV_OK && own) rc = eakvi_work_begin(pool, st, need);
    if (rc == EAKV_OK) {
        int e = eakvd_paged_attend(&pool->geom, pool->dev, &d, layer, d_q, ld_q, dtype == EAKV_BF16, n_q,
                                   n_kv, d_out, ld_out, own ? pool->work : d_work, st);
        if (e) rc = eakvi_hip_fail(e, "attention_paged launch");
        if (own) {
            int e2 = eakvi_work_end(pool, st);
            if (rc == EAKV_OK) rc = e2;
        }
    }
    eakvi_leave(prev);
    return rc;
}
