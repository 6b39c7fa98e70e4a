/* verify.c — drafted tokens against the target's probabilities (host C11), on the
 * HIP device current at the call and the given stream (NULL: the default stream). */
#include "internal.h"

/* Sequences of a call: one grid row each. */
#define kVerifySeqs 65535

static int sizes_ok(int n_seqs, int n_drafts, int vocab)
{
    return n_seqs >= 0 && n_seqs <= kVerifySeqs && n_drafts >= 0 && n_drafts < 65536 &&
           vocab >= 1 && vocab <= (1 << 30);
}

static size_t matrix(int64_t rows, int64_t ld, int cols)
{
    return rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)cols) * 4 : 0;
}

size_t eakv_verify_drafts_work_bytes(int n_seqs, int n_drafts, int vocab)
{
    if (!sizes_ok(n_seqs, n_drafts, vocab)) {
        eakvi_set_error(EAKV_ERR_INVALID, "verify: invalid size");
        return 0;
    }
    return eakvd_verify_work_bytes(n_seqs, vocab);
}

int eakv_verify_drafts_device(int n_seqs, int n_drafts, int vocab, const int32_t *d_counts,
                              const int32_t *d_tokens, const float *d_draft, int64_t ld_draft,
                              const float *d_target, int64_t ld_target, const float *d_uniform,
                              int32_t *d_accepted, int32_t *d_next, void *d_work,
                              size_t work_bytes, void *stream)
{
    if (!sizes_ok(n_seqs, n_drafts, vocab) || ld_target < vocab || (d_draft && ld_draft < vocab))
        return eakvi_set_error(EAKV_ERR_INVALID, "verify: invalid size");
    if (n_seqs == 0) return EAKV_OK;
    if (!d_target || !d_uniform || !d_accepted || !d_next || !d_work || (n_drafts && !d_tokens))
        return eakvi_set_error(EAKV_ERR_INVALID, "verify: NULL buffer");
    const uintptr_t any = (uintptr_t)d_counts | (uintptr_t)d_tokens | (uintptr_t)d_draft |
                          (uintptr_t)d_target | (uintptr_t)d_uniform | (uintptr_t)d_accepted |
                          (uintptr_t)d_next;
    if (any & 3 || (uintptr_t)d_work & 7)
        return eakvi_set_error(EAKV_ERR_INVALID, "verify: misaligned buffer");
    const size_t need = eakvd_verify_work_bytes(n_seqs, vocab);
    if (work_bytes < need)
        return eakvi_set_error(EAKV_ERR_INVALID, "verify: %zu bytes of workspace, %zu needed",
                              work_bytes, need);
    /* blocks write their results while others read */
    const int64_t n = n_seqs, k = n_drafts;
    const eakvi_span out[3] = {{d_accepted, (size_t)n * 4}, {d_next, (size_t)n * 4}, {d_work, need}};
    const eakvi_span in[5] = {{d_counts, (size_t)n * 4},
                        {d_tokens, (size_t)(n * k) * 4},
                        {d_uniform, (size_t)(n * (k + 1)) * 4},
                        {d_draft, matrix(n * k, ld_draft, vocab)},
                        {d_target, matrix(n * (k + 1), ld_target, vocab)}};
    for (int i = 0; i < 3; i++) {
        int bad = eakvi_overlap(out[i], out[(i + 1) % 3]);
        for (int j = 0; j < 5; j++) bad |= eakvi_overlap(out[i], in[j]);
        if (bad) return eakvi_set_error(EAKV_ERR_INVALID, "verify: overlapping buffers");
    }
    int e = eakvd_verify(n_seqs, n_drafts, vocab, d_counts, d_tokens, d_draft, ld_draft, d_target,
                         ld_target, d_uniform, d_accepted, d_next, d_work, stream);
    return e ? eakvi_hip_fail(e, "verify launch") : EAKV_OK;
}
