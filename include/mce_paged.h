/*
 * mce_paged.h — C ABI of the MI355X (gfx950) attention of one new token per sequence over a paged key/value cache
 * (libmce_attn.so): the single-token form of the masked attention of mce_attn.h.
 *
 * Sequence b has n = lengths[b] tokens in the cache, the new one among them. Its query head h of Hq reads key/value
 * head h / (Hq / Hkv); token j lies in page block_table[b * bt_sb + j / page] at slot j % page, and is seen when
 * window = 0, n - 1 - j < window or j < sinks:
 *   out_bh = sum_j p_j v_j,  p = softmax over the seen j of scale q_bh . k_j     (n <= 0: out = 0)
 * Lengths above max_pages * page count as that. A token in a page whose number is outside [0, pages) is not seen (a
 * cache may free the pages behind a window and leave their entries stale or -1); with no token left out = 0. Nothing of
 * a token that is not seen is used, whatever lies there.
 * Sums are fp32; p is rounded to the element type as operand of the second product, and the result is rounded once.
 *
 * Buffers: q [B, Hq, D] with element strides (batch, head); caches [pages, page, Hkv, D] with element strides (page,
 * slot, head), last dimensions contiguous, 16-byte aligned, strides multiples of 8; out contiguous [B, Hq, D]. D is a
 * multiple of 8 up to 128, page a multiple of 8; B Hq is at most 2^24, and B Hkv ceil(Hq / Hkv / 32) below it. Every call is asynchronous on `stream`, allocates nothing, and returns
 * 0 or an MCE_ATTN_E* code of mce_attn.h; arguments are checked before anything is launched.
 */
#ifndef MCE_PAGED_H
#define MCE_PAGED_H

#include "mce_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The parts of the sums of sequences whose cache is split over workgroups (0 where none is). The split depends on the
 * sizes alone, not on the lengths, which the host need not know. */
MCE_ATTN_API size_t mce_paged_ws_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages,
                                       int64_t window, int64_t sinks);
MCE_ATTN_API int mce_paged(const void* q, int64_t q_sb, int64_t q_sh, const void* k, int64_t k_sp, int64_t k_st,
                           int64_t k_sh, const void* v, int64_t v_sp, int64_t v_st, int64_t v_sh,
                           const int32_t* block_table, int64_t bt_sb, const int32_t* lengths, int64_t B, int64_t Hq,
                           int64_t Hkv, int64_t D, int64_t pages, int64_t page, int64_t max_pages, int64_t window,
                           int64_t sinks, float scale, int dtype, void* out, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MCE_PAGED_H */
