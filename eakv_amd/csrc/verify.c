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
    int e = eakvd_verify(n_seqs, n_drafts, vocab, d_counts, d_tokens, d_draft, ld_draft, d_target,
                         ld_target, d_uniform, d_accepted, d_next, d_work, stream);
    return e ? eakvi_hip_fail(e, "verify launch") : EAKV_OK;
}
