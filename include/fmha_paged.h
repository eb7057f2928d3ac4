/* fmha_paged.h -- head_dim-64 BF16 serving operators around the attention
 * forward of fmha_fwd.h, for B200 (sm_100a): rotary positions with up to four
 * axes, appending to a paged K/V cache with the rotation on the way, attention
 * of new tokens over the paged cache, and attention for a batch whose
 * sequences share one long prefix.
 *
 * Conventions shared by all entries
 *   - bf16 bits in uint16_t; head_dim 64 is innermost and contiguous.
 *   - Strides in elements, 64 bits; base pointers 16-byte aligned and strides
 *     multiples of 8 (16 bytes).
 *   - Tokens are dense ([batch, seqlen_q], seqstart_q == NULL) or packed
 *     ([total_q], seqstart_q = int32 [batch + 1] prefix sums on the device).
 *   - The cache: pages of page_size tokens (a power of two, 8 to 4096),
 *     addressed by (page, token in page, K/V head) strides.  page_table is
 *     int32 [batch, max_pages] on the device; only the entries that a
 *     sequence's length needs are read, and what pages hold past a sequence's
 *     end (NaN included) never reaches a result.
 *   - seqlens_k[b] is the sequence's length in the cache WITH the new tokens:
 *     new token i of a sequence with n new ones has place seqlens_k[b] - n + i.
 *   - Nothing is allocated, copied from the host or synchronised by a call
 *     (after the first on a device), so calls may be captured in CUDA graphs.
 *   - Limits: tokens * nhead_q and the 32-key units of batch * max_pages pages
 *     below 2^31; nhead_q at most 8192; strides below 2^39.
 *   - O is rounded to bf16 once.  Sequences of up to 16 rows (new tokens x query
 *     heads of a K/V head's group) carry the softmax weights to 2^-16 of
 *     themselves before that; for more rows, and for all keys of a shared
 *     prefix, they are rounded to bf16 as well.  The LSE is fp32 throughout.
 *   - seqstart_q should cover tokens 0 .. total_q - 1; a token outside every
 *     sequence is not worked on: append reports it and zeroes its row of q_out,
 *     the attention leaves its row of o unwritten.
 *   - Returns an FMHA_* status.  Bad values that only the device can see (a
 *     page id outside the cache, a length past the page table, a position
 *     outside the angle table, prefix sums that decrease or leave the tokens, more
 *     new tokens in a sequence than seqlen_q) access no memory out of range (rows
 *     of overlapping sequences may be left unwritten) and are reported once by
 *     fmha_fwd_d64_status as FMHA_ERR_INDEX.
 */
#ifndef FMHA_PAGED_H
#define FMHA_PAGED_H

#include "fmha_fwd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rotation of tokens' heads by their positions, and where they go. */
typedef struct FmhaRopeParams {
    const uint16_t* q;       /* [.., nhead_q, 64] or NULL */
    const uint16_t* k;       /* [.., nhead_k, 64] or NULL */
    const uint16_t* v;       /* append only */
    uint16_t* q_out;         /* may be q itself */
    uint16_t* k_out;         /* rope: may be k itself; append: the K cache */
    uint16_t* v_out;         /* append: the V cache */
    const float* cos_sin;    /* [max_pos, 2 * n_pairs]: cosines, then sines (NULL in append: no rotation) */
    const int32_t* positions;/* [axes, tokens] (NULL in append: the place in the cache) */
    const int32_t* seqstart_q;
    const int32_t* page_table;  /* append only */
    const int32_t* seqlens_k;   /* append only */
    long long stride_q, nhead_stride_q, batch_stride_q;
    long long stride_k, nhead_stride_k, batch_stride_k;
    long long stride_v, nhead_stride_v, batch_stride_v;
    long long stride_qo, nhead_stride_qo, batch_stride_qo;
    long long stride_ko, nhead_stride_ko, batch_stride_ko;  /* append: token in page, head, page */
    long long stride_vo, nhead_stride_vo, batch_stride_vo;  /* append: token in page, head, page */
    long long axis_stride;   /* elements between the axes' rows of positions */
    long long table_stride;  /* elements between the rows of page_table */
    int batch, seqlen_q;     /* dense: tokens = batch * seqlen_q */
    int total_q;             /* packed: tokens */
    int nhead_q, nhead_k;
    int max_pos, n_pairs;    /* n_pairs: 8, 16, 24 or 32 rotated pairs a head; the dims after them pass through */
    int interleaved;         /* 0: pairs (j, j + n_pairs); 1: pairs (2j, 2j + 1) */
    int inverse;             /* 1: rotate back (the gradient of the rotation) */
    int page_size, num_pages, max_pages;
    uint8_t axis_of[32];     /* axis whose position turns pair j */
} FmhaRopeParams;

/* q_out, k_out = rotated q, k.  q or k may be NULL.  A token whose position is
 * outside the angle table gets zero rows. */
int fmha_rope_d64_bf16(const FmhaRopeParams* params, struct CUstream_st* stream);

/* New K and V, K rotated, into the pages of the cache; q, if given, rotated
 * into q_out.  A token whose place is negative (a batch slot with fewer keys
 * than new tokens, such as an empty slot) is not stored, and its q_out row is
 * zero; so it is with one whose position is outside the angle table.  No two tokens of a call may name the same place. */
int fmha_paged_append_d64_bf16(const FmhaRopeParams* params, struct CUstream_st* stream);

typedef struct FmhaPagedParams {
    const uint16_t* q;       /* dense [batch, seqlen_q, nhead_q, 64] or packed [total_q, nhead_q, 64], any strides */
    const uint16_t* k_cache;
    const uint16_t* v_cache;
    uint16_t* o;
    float* lse;              /* natural log, or NULL: dense [batch, nhead_q, seqlen_q], packed [nhead_q, total_q] */
    const int32_t* seqstart_q;
    const int32_t* page_table;
    const int32_t* seqlens_k;
    const int32_t* prefix_pages;  /* prefix entry only: pages of the shared prefix */
    void* workspace;
    long long workspace_bytes;
    long long stride_q, nhead_stride_q, batch_stride_q;
    long long stride_o, nhead_stride_o, batch_stride_o;
    long long stride_k, nhead_stride_k, page_stride_k;  /* token in page, head, page */
    long long stride_v, nhead_stride_v, page_stride_v;
    long long table_stride;
    int batch, seqlen_q;     /* packed: seqlen_q bounds every sequence's new tokens */
    int total_q;
    int nhead_q, nhead_k;
    int page_size, num_pages, max_pages;
    int prefix_len;          /* prefix entry only */
    int causal;              /* bottom-right aligned: new token i sees the keys up to its own place */
    float scale;             /* softmax scale * log2(e), as in FmhaFwdParams; > 0 */
} FmhaPagedParams;

/* Device scratch that a call with these sizes needs (16-byte aligned, any
 * contents; calls that may overlap need one each); total_q 0 for dense tokens, prefix_len 0 for
 * fmha_paged_fwd_d64_bf16.  0 on invalid sizes. */
size_t fmha_paged_workspace_bytes(int batch, int seqlen_q, int total_q, int nhead_q, int nhead_k,
                                  int prefix_len);

/* O = softmax(scale * Q K^T + mask) V over each sequence's pages.  A row that
 * sees no key gets O = 0 and LSE = -inf; one with a score of NaN or +inf, which
 * has no softmax, O = LSE = NaN.  Values of keys that a row does not see never
 * reach it, NaN and infinities included. */
int fmha_paged_fwd_d64_bf16(const FmhaPagedParams* params, struct CUstream_st* stream);

/* The same where every sequence's keys are the prefix_len keys of
 * prefix_pages followed by its own seqlens_k[b] ones: the prefix is read once
 * for the whole batch.  prefix_len >= 1. */
int fmha_prefix_fwd_d64_bf16(const FmhaPagedParams* params, struct CUstream_st* stream);

#ifdef __cplusplus
}
#endif
#endif /* FMHA_PAGED_H */
