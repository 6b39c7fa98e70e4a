/* move.c — tokens moved between and within caches (host C11): copies of a range
 * into several caches, gathers of a list of tokens, and the synchronous forms
 * eakv_cache_fork and eakv_cache_compact. */
#include <string.h>

#include "internal.h"

static int like(const eakv_cache_t *a, const eakv_cache_t *b)
{
    return a->n_layers == b->n_layers && a->n_kv_heads == b->n_kv_heads &&
           a->head_dim == b->head_dim && a->device == b->device;
}

static int dim_ok(const eakv_cache_t *c) { return c->head_dim == 64 || c->head_dim == 128; }

/* These calls write caches, so their stream is ordered with the shared stream both
 * ways; that cannot be recorded in a graph. */
static int not_captured(const eakv_cache_t *c, void *stream, const char *what)
{
    int yes = 0;
    int e = eakvd_stream_capturing(stream ? stream : c->stream, &yes);
    if (e) return eakvi_hip_fail(e, what);
    return yes ? eakvi_set_error(EAKV_ERR_INVALID, "%s: the stream records a graph", what)
               : EAKV_OK;
}

int eakv_cache_copy_batch_device(const eakv_cache_t *src, int src_pos, eakv_cache_t *const *dsts,
                                 int n_dsts, int dst_pos, int n_tokens, void *stream)
{
    if (!src || !dsts || n_dsts <= 0 || n_dsts > EAKVD_MAX_BATCH || src_pos < 0 || dst_pos < 0 ||
        n_tokens < 0 || (int64_t)src_pos + n_tokens > src->max_seq_len)
        return eakvi_set_error(EAKV_ERR_INVALID, "copy: invalid argument");
    if (!dim_ok(src))
        return eakvi_set_error(EAKV_ERR_INVALID, "copy: head_dim %d not 64 or 128", src->head_dim);
    eakv_cache_t *all[EAKVD_MAX_BATCH + 1];
    uint8_t *dst[EAKVD_MAX_BATCH];
    for (int i = 0; i < n_dsts; i++) {
        eakv_cache_t *d = dsts[i];
        if (!d || !like(src, d) || d->max_seq_len != dsts[0]->max_seq_len)
            return eakvi_set_error(EAKV_ERR_INVALID, "copy: caches differ in shape");
        if (dst_pos > d->seq_len || (int64_t)dst_pos + n_tokens > d->max_seq_len)
            return eakvi_set_error(EAKV_ERR_INVALID,
                                  "copy: %d tokens to %d of a cache with %d tokens and room for %d",
                                  n_tokens, dst_pos, d->seq_len, d->max_seq_len);
        if (d == src && src_pos < dst_pos + n_tokens && dst_pos < src_pos + n_tokens)
            return eakvi_set_error(EAKV_ERR_INVALID, "copy: overlapping ranges of one cache");
        for (int k = 0; k < i; k++)
            if (dsts[k] == d)
                return eakvi_set_error(EAKV_ERR_INVALID, "copy: a destination named twice");
        all[i] = d;
        dst[i] = d->dev;
    }
    if (n_tokens == 0) return EAKV_OK;
    int rc = not_captured(src, stream, "copy");
    if (rc) return rc;
    int n_all = n_dsts;
    all[n_all++] = (eakv_cache_t *)src;
    int prev;
    rc = eakvi_enter(src, &prev);
    if (rc) return rc;
    void *st = eakvi_batch_stream(all, n_all, stream);
    for (int i = 0; rc == EAKV_OK && i < n_all; i++) rc = eakvi_order_before(all[i], st);
    if (rc == EAKV_OK) {
        int e = eakvd_copy_tokens(&src->geom, &dsts[0]->geom, src->dev, src_pos, dst, n_dsts,
                                  dst_pos, n_tokens, st);
        if (e) rc = eakvi_hip_fail(e, "copy launch");
    }
    /* later work on the shared stream and host-pointer calls on any of the
     * caches: after the copy (the source may be overwritten then) */
    if (rc == EAKV_OK) rc = eakvi_order_after(all, n_all, st);
    eakvi_leave(prev);
    return rc;
}

int eakv_cache_gather_batch_device(eakv_cache_t *const *srcs, eakv_cache_t *const *dsts,
                                   int n_caches, const int32_t *dst_pos, const int32_t *d_index,
                                   const int32_t *n_tokens, void *stream)
{
    if (!srcs || !dsts || n_caches <= 0 || n_caches > EAKVD_MAX_BATCH || !dst_pos || !n_tokens)
        return eakvi_set_error(EAKV_ERR_INVALID, "gather: invalid argument");
    eakv_cache_t *all[2 * EAKVD_MAX_BATCH];
    eakvd_gather job;
    memset(&job, 0, sizeof(job));
    int64_t total = 0;
    for (int i = 0; i < n_caches; i++) {
        eakv_cache_t *s = srcs[i], *d = dsts[i];
        if (!s || !d || !like(s, srcs[0]) || !like(d, s) ||
            s->max_seq_len != srcs[0]->max_seq_len || d->max_seq_len != dsts[0]->max_seq_len)
            return eakvi_set_error(EAKV_ERR_INVALID, "gather: caches differ in shape");
        if (dst_pos[i] < 0 || dst_pos[i] > d->seq_len || n_tokens[i] < 0 ||
            (int64_t)dst_pos[i] + n_tokens[i] > d->max_seq_len)
            return eakvi_set_error(EAKV_ERR_INVALID,
                                  "gather: %d tokens to %d of a cache with %d tokens and room for "
                                  "%d", n_tokens[i], dst_pos[i], d->seq_len, d->max_seq_len);
        job.src[i] = s->dev;
        job.dst[i] = d->dev;
        job.dst_pos[i] = dst_pos[i];
        job.n_tokens[i] = n_tokens[i];
        job.first[i] = total;
        total += n_tokens[i];
        all[i] = d;
        all[n_caches + i] = s;
    }
    /* a cache that is written is no other pair's source or destination */
    for (int i = 0; i < n_caches; i++)
        for (int k = 0; k < n_caches; k++)
            if (i != k && (dsts[i] == dsts[k] || dsts[i] == srcs[k]))
                return eakvi_set_error(EAKV_ERR_INVALID,
                                      "gather: a destination named by another pair");
    if (!dim_ok(srcs[0]))
        return eakvi_set_error(EAKV_ERR_INVALID, "gather: head_dim %d not 64 or 128",
                              srcs[0]->head_dim);
    if (total == 0) return EAKV_OK;
    if (!d_index || (uintptr_t)d_index & 3)
        return eakvi_set_error(EAKV_ERR_INVALID, "gather: NULL or misaligned index");
    int rc = not_captured(srcs[0], stream, "gather");
    if (rc) return rc;
    job.n_seq = n_caches;
    job.index = d_index;
    int prev;
    rc = eakvi_enter(srcs[0], &prev);
    if (rc) return rc;
    void *st = eakvi_batch_stream(all, 2 * n_caches, stream);
    for (int i = 0; rc == EAKV_OK && i < 2 * n_caches; i++) rc = eakvi_order_before(all[i], st);
    if (rc == EAKV_OK) {
        int e = eakvd_gather_tokens(&srcs[0]->geom, &dsts[0]->geom, &job, st);
        if (e) rc = eakvi_hip_fail(e, "gather launch");
    }
    if (rc == EAKV_OK) rc = eakvi_order_after(all, 2 * n_caches, st);
    eakvi_leave(prev);
    return rc;
}

eakv_cache_t *eakv_cache_fork(const eakv_cache_t *csrc, int n_tokens, int max_seq_len)
{
    eakv_cache_t *src = (eakv_cache_t *)csrc;
    if (!src || n_tokens < 0 || n_tokens > src->seq_len || n_tokens > max_seq_len) {
        eakvi_set_error(EAKV_ERR_INVALID, "fork: invalid argument");
        return NULL;
    }
    if (!dim_ok(src)) {
        eakvi_set_error(EAKV_ERR_INVALID, "fork: head_dim %d not 64 or 128", src->head_dim);
        return NULL;
    }
    int prev;
    if (eakvi_enter(src, &prev)) return NULL;
    eakv_cache_t *dst = eakv_cache_create(src->n_layers, src->n_kv_heads, src->head_dim,
                                          max_seq_len);
    if (dst && n_tokens) {
        int rc = eakvi_host_begin(src);
        if (rc == EAKV_OK) {
            int e = eakvd_copy_tokens(&src->geom, &dst->geom, src->dev, 0, &dst->dev, 1, 0,
                                      n_tokens, src->hstream);
            if (e) rc = eakvi_hip_fail(e, "fork launch");
        }
        rc = eakvi_host_end(src, rc, 0, "fork");
        if (rc) {
            eakv_cache_free(dst);
            dst = NULL;
        } else {
            dst->seq_len = n_tokens;
        }
    }
    eakvi_leave(prev);
    return dst;
}

int eakv_cache_compact(eakv_cache_t *c, int start, const int32_t *keep, int n_keep)
{
    if (!c || start < 0 || start > c->seq_len || n_keep < 0 || n_keep > c->seq_len - start ||
        (n_keep && !keep))
        return eakvi_set_error(EAKV_ERR_INVALID, "compact: invalid argument");
    if (!dim_ok(c))
        return eakvi_set_error(EAKV_ERR_INVALID, "compact: head_dim %d not 64 or 128", c->head_dim);
    for (int i = 0; i < n_keep; i++)
        if (keep[i] >= c->seq_len || keep[i] < start || (i && keep[i] <= keep[i - 1]))
            return eakvi_set_error(EAKV_ERR_INVALID,
                                  "compact: positions must ascend within the tokens from start on");
    /* the leading tokens that stay where they are */
    int same = 0;
    while (same < n_keep && keep[same] == start + same) same++;
    const int n = n_keep - same;
    int rc = EAKV_OK;
    if (n) {
        int prev;
        rc = eakvi_enter(c, &prev);
        if (rc) return rc;
        const size_t bytes = (size_t)n * 4;
        void *st = c->hstream;
        rc = eakvi_host_begin(c);
        if (rc == EAKV_OK) rc = eakvi_work_begin(c, st, bytes);
        const int began = rc == EAKV_OK;
        if (began) {
            eakvi_bounce bo;
            const void *list;
            eakvi_bounce_begin(c, bytes, 0, &bo);
            int e = eakvi_bounce_in(&bo, c->work, keep + same, bytes, 0, st, &list);
            if (!e) {
                eakvd_gather job;
                memset(&job, 0, sizeof(job));
                job.n_seq = 1;
                job.src[0] = c->dev;
                job.dst[0] = c->dev;
                job.dst_pos[0] = start + same;
                job.n_tokens[0] = n;
                job.index = list;
                e = eakvd_gather_tokens(&c->geom, &c->geom, &job, st);
            }
            if (e) rc = eakvi_hip_fail(e, "compact");
        }
        rc = eakvi_host_end(c, rc, began, "compact");
        eakvi_leave(prev);
    }
    if (rc == EAKV_OK) c->seq_len = start + n_keep;
    return rc;
}

int eakv_cache_planes_device(const eakv_cache_t *c, int layer, int kv_idx, uint8_t **weights,
                             float **scales, float **biases)
{
    if (!c || layer < 0 || layer >= c->n_layers || kv_idx < 0 || kv_idx > 1)
        return eakvi_set_error(EAKV_ERR_INVALID, "planes: invalid argument");
    uint8_t *blk = c->dev + (int64_t)(layer * 2 + kv_idx) * c->geom.block_bytes;
    if (weights) *weights = blk;
    if (scales) *scales = (float *)(blk + c->geom.s_off);
    if (biases) *biases = (float *)(blk + c->geom.b_off);
    return EAKV_OK;
}
