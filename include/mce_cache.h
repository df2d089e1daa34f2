/*
 * mce_cache.h — C ABI of the MI355X (gfx950) kernels over a paged key/value cache held in 8 bits (libmce_serve.so): writing
 * new tokens' keys and values into it, reading them back, and the attention of one new token per sequence over it.
 *
 * A cache holds the keys (or values) of all sequences as e4m3 codes (float8_e4m3fn: 3 bits behind the leading one, largest
 * value 448, no infinities, steps of 2^-9 at least), [pages, page, Hkv, D]. Token j of sequence b lies in page
 * block_table[b * bt_sb + j / page] at slot j % page. `block` neighbouring slots of a page share one fp32 scale for each
 * head, scales [pages, page / block, Hkv], contiguous: a value is its code times the scale.
 *
 * Writing. Sequence b gets the rows cu[b] .. cu[b + 1] - 1 of k and v (cu NULL: row b alone, N = B) as its last tokens:
 * they stand at the positions up to lengths[b] - 1, which counts them already. A block that gets tokens holds those of
 * its slots in front of the first new one as well; what lies behind the last new one is not looked at. With a the largest
 * finite magnitude of a block's new elements, its scale becomes the larger of
 *   2^e, the smallest power of two from 2^-100 on with a <= 448 2^e, and
 *   the scale that it had, if it holds earlier tokens;
 * earlier codes are rounded again where that is more than they had. A power of two costs a floating-point code none of its
 * precision, and rounding again costs only what falls below 2^-6 of the scale: whether tokens come one by one or at once
 * changes nothing else. Codes are rounded to nearest, ties to even; a NaN or an infinity is stored as a NaN. Tokens whose
 * page is outside [0, pages) or past max_pages are left out, as are rows outside every sequence. A page that gets tokens
 * must belong to one sequence of the call.
 *
 * Reading back. Rows cu[b] .. cu[b + 1] - 1 of the results get the first tokens of sequence b, code times scale rounded to
 * the element type (beyond fp16's largest value: that value). Rows outside every sequence and tokens outside the cache
 * give 0.
 *
 * Attention of one new token per sequence: mce_paged.h's, with the cache's values in the place of its elements:
 *   out_bh = sum_j p_j v_j,  p = softmax over the seen j of scale q_bh . k_j     (nothing seen: out = 0)
 * Codes are exact in the element type, so the first product's operands are exact; sums are fp32; exp(score) times the
 * value's scale is rounded to the element type as operand of the second product, and the result is rounded once. Scales
 * are positive, finite and between 2^-100 and 2^120; those of blocks without a seen token are not used. The denominator is
 * fp32 however far scales are apart, and scores may be of any finite size; what operands of the second product lose is what lies
 * below the type's range next to the largest exp(score) times scale (2^-25 of it in fp16).
 *
 * Buffers: k, v [N, Hkv, D] and q [B, Hq, D] in 16 bits with element strides (token, head; batch, head for q), 16-byte
 * aligned, strides multiples of 8; caches with strides (page, slot, head) in bytes, 16-byte aligned, strides multiples of
 * 16, slots at least D apart; the last dimension contiguous everywhere; results contiguous. D is a multiple of 16 up to
 * 128, page a multiple of 8 up to 65536, block a multiple of 8 up to 128 that divides page. Two elements of a cache that is
 * written must not share memory. cu as in mce_pack.h: numbers outside 0 .. N count as the nearest of the two; where they fall,
 * what is written is not defined, but lies inside the buffers. Launches hold fewer than 2^24 workgroups: a write takes
 * 2 Hkv (N / block + 2 B) below that (cu NULL: 2 Hkv B), a read (rows / 8 + B + 2) / 2, an attention B Hq below 2^24 - 2^20.
 * Calls are asynchronous on `stream`, allocate nothing and return 0 or an MCE_ATTN_E* code; arguments are checked before anything
 * is launched. Grids depend on sizes alone, so a captured call may be replayed with other lengths. Where the attention shares the
 * batch's tiles among workgroups evenly (small batches, and large ones of long caches), the places at which a sequence's sums are
 * cut depend on the lengths of all sequences: its last bits may change when a neighbour grows, and are the same for the same
 * lengths.
 */
#ifndef MCE_CACHE_H
#define MCE_CACHE_H

#include "mce_pack.h"

#ifdef __cplusplus
extern "C" {
#endif

MCE_SERVE_API int mce_cache_write(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                                  void* kc, int64_t kc_sp, int64_t kc_st, int64_t kc_sh, void* vc, int64_t vc_sp,
                                  int64_t vc_st, int64_t vc_sh, float* k_scale, float* v_scale,
                                  const int32_t* block_table, int64_t bt_sb, const int32_t* lengths, const int32_t* cu,
                                  int64_t B, int64_t N, int64_t Hkv, int64_t D, int64_t pages, int64_t page,
                                  int64_t block, int64_t max_pages, int dtype, void* stream);

/* k and v: contiguous [rows, Hkv, D] of the element type. */
MCE_SERVE_API int mce_cache_read(const void* kc, int64_t kc_sp, int64_t kc_st, int64_t kc_sh, const void* vc,
                                 int64_t vc_sp, int64_t vc_st, int64_t vc_sh, const float* k_scale,
                                 const float* v_scale, const int32_t* block_table, int64_t bt_sb, const int32_t* cu,
                                 int64_t B, int64_t rows, int64_t Hkv, int64_t D, int64_t pages, int64_t page,
                                 int64_t block, int64_t max_pages, int dtype, void* k, void* v, void* stream);

/* The parts of the sums of sequences whose cache is split over workgroups (0 where none is). */
MCE_SERVE_API size_t mce_cache_attn_ws_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page,
                                             int64_t max_pages, int64_t window, int64_t sinks);
MCE_SERVE_API int mce_cache_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* kc, int64_t kc_sp, int64_t kc_st,
                                 int64_t kc_sh, const void* vc, int64_t vc_sp, int64_t vc_st, int64_t vc_sh,
                                 const float* k_scale, const float* v_scale, const int32_t* block_table, int64_t bt_sb,
                                 const int32_t* lengths, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t pages,
                                 int64_t page, int64_t block, int64_t max_pages, int64_t window, int64_t sinks,
                                 float scale, int dtype, void* out, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MCE_CACHE_H */
