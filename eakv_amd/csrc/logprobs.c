/* logprobs.c — log probabilities of given tokens, entropies and alternatives (host C11), on
 * the HIP device current at the call and the given stream (NULL: the default stream). */
#include "internal.h"

static int sizes_ok(int n_rows, int vocab, int n_top)
{
    /* a block of 256 threads for each 16384 values of a row; a launch has fewer than 2^32 threads */
    return n_rows >= 0 && vocab >= 1 && vocab <= (1 << 30) && n_top >= 0 && n_top <= EAKV_TOP_MAX &&
           (int64_t)n_rows * ((int64_t)vocab / 16384 + 2) < 1 << 24;
}

size_t eakv_token_logprobs_work_bytes(int n_rows, int vocab, int n_top)
{
    if (!sizes_ok(n_rows, vocab, n_top)) {
        eakvi_set_error(EAKV_ERR_INVALID, "logprobs: invalid size");
        return 0;
    }
    return eakvd_logprobs_work_bytes(n_rows, vocab, n_top);
}

int eakv_token_logprobs_device(int n_rows, int vocab, const void *d_logits, int dtype, int64_t ld,
                               const int32_t *d_tokens, int n_top, float *d_logprobs, float *d_entropy,
                               int32_t *d_top_tokens, float *d_top_logprobs, void *d_work,
                               size_t work_bytes, void *stream)
{
    if (!sizes_ok(n_rows, vocab, n_top) || ld < vocab)
        return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: invalid size");
    if (dtype != EAKV_F32 && dtype != EAKV_BF16)
        return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: dtype %d not EAKV_F32 or EAKV_BF16", dtype);
    if (n_rows == 0 || (!d_logprobs && !d_entropy && n_top == 0)) return EAKV_OK;
    const size_t need = eakvd_logprobs_work_bytes(n_rows, vocab, n_top);
    if (!d_logits || (d_logprobs && !d_tokens) || (n_top && (!d_top_tokens || !d_top_logprobs)) ||
        (need && !d_work))
        return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: NULL buffer");
    const uintptr_t words = (uintptr_t)d_tokens | (uintptr_t)d_logprobs | (uintptr_t)d_entropy |
                            (uintptr_t)d_top_tokens | (uintptr_t)d_top_logprobs;
    if (words & 3 || (uintptr_t)d_logits & (dtype == EAKV_F32 ? 3 : 1) || (uintptr_t)d_work & 15)
        return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: misaligned buffer");
    if (work_bytes < need)
        return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: %zu bytes of workspace, %zu needed", work_bytes,
                               need);
    /* blocks write their results while others read */
    const size_t n = (size_t)n_rows, k = n * (size_t)n_top;
    const eakvi_span out[5] = {{d_logprobs, n * 4}, {d_entropy, n * 4}, {d_top_tokens, k * 4},
                               {d_top_logprobs, k * 4}, {d_work, need}};
    const eakvi_span in[2] = {{d_logits, ((n - 1) * (size_t)ld + (size_t)vocab) * (dtype == EAKV_F32 ? 4 : 2)},
                              {d_logprobs ? d_tokens : NULL, n * 4}};
    for (int i = 0; i < 5; i++) {
        int bad = eakvi_overlap(out[i], in[0]) || eakvi_overlap(out[i], in[1]);
        for (int j = 0; j < i; j++) bad |= eakvi_overlap(out[i], out[j]);
        if (bad) return eakvi_set_error(EAKV_ERR_INVALID, "logprobs: overlapping buffers");
    }
    int e = eakvd_logprobs(n_rows, vocab, d_logits, dtype == EAKV_BF16, ld, d_tokens, n_top, d_logprobs,
                           d_entropy, d_top_tokens, d_top_logprobs, d_work, stream);
    return e ? eakvi_hip_fail(e, "logprobs launch") : EAKV_OK;
}
