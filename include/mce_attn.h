/*
 * mce_attn.h — C ABI of the MI355X (gfx950) attention kernels (libmce_attn.so): causal attention over a sliding window
 * with first tokens that stay visible, forward and backward.
 *
 * memarch's blocks call torch's scaled_dot_product_attention or block-window helpers for this (lm.py:448-554,
 * full2.py:154-181).
 *
 * Query head h of Hq reads key/value head h / (Hq / Hkv). Position i of sequence b sees position j when
 *   j <= i  and  (window = 0  or  i - j < window  or  j < sinks)  and  i < lengths[b]
 *   s_ij = scale q_i . k_j;  p_i = softmax of s_ij over the j that i sees;  out_i = sum_j p_ij v_j
 * (window = 0: every earlier position; lengths NULL: T). A row that sees nothing (i >= lengths[b]) has out = 0, and the
 * gradients of such positions are 0; rows at or past lengths[b] are never read. Inside a sequence, masked pairs get a
 * weight of exactly 0: finite values there do not matter, a NaN or an infinity may reach rows that do not see it, up to 95
 * positions from one that does, and keys likewise (dk and dv of keys beside the first tokens, in the same 32, from any row).
 *   d_i = go_i . out_i;  ds_ij = p_ij (go_i . v_j - d_i)
 *   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij go_i  (dk, dv summed over the heads
 *   that share them)
 * Products take 16-bit operands and sum in fp32; softmax statistics are fp32; p and ds are rounded to the element type
 * as operands of the second products (half of dq's products take what the rounding of ds leaves over as well), results
 * are rounded once. In fp16, p (go v - d) has to stay in range, as the results have to. Scores may have any finite size for
 * out; the backward forms p from lse, an fp32 number of the scores' size, so that scores of S put p off by about S 2^-22 of
 * itself: gradients ask for scores below 2^20 or so, and from 2^27 on they may not be finite.
 *
 * Buffers: q [B, T, Hq, D], k and v [B, T, Hkv, D], go like q: element strides (batch, token, head) are given, the last
 * dimension is contiguous; 16-byte aligned, strides multiples of 8, the token stride at least D. D is a multiple of 8 up to 128. out, dq
 * [B, T, Hq, D] and dk, dv [B, T, Hkv, D] are contiguous. lse is [B, Hq, T] fp32. B Hq ceil(T / 128) is below 2^24 (what
 * one launch can hold). Every call is asynchronous on
 * `stream`, allocates nothing, and returns 0 or an MCE_ATTN_E* code; arguments are checked before anything is launched.
 */
#ifndef MCE_ATTN_H
#define MCE_ATTN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define MCE_ATTN_API __attribute__((visibility("default")))
#else
#define MCE_ATTN_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define MCE_ATTN_OK 0
#define MCE_ATTN_EINVAL 1     /* size, stride, head count, scale, element type or null pointer */
#define MCE_ATTN_EALIGN 2     /* a pointer that is not 16-byte aligned or a stride that is not a multiple of 8 */
#define MCE_ATTN_EWORKSPACE 3 /* workspace missing, too small or not 256-byte aligned */
#define MCE_ATTN_ELAUNCH 4    /* a HIP launch failed (mce_attn_last_hip_error) */

/* element types */
#define MCE_ATTN_BF16 1
#define MCE_ATTN_F16 2

/* Text of an MCE_ATTN_* code, and the hipError_t of the calling thread's last failed launch (0 if none). */
MCE_ATTN_API const char* mce_attn_error_string(int code);
MCE_ATTN_API int mce_attn_last_hip_error(void);

/* out, and for a backward (both may be NULL) lse, the log of the softmax's denominator in units of q . k, +inf on empty
 * rows, and res [B, T, Hq, D], what out's rounding left over: d_i = go_i . (out_i + res_i). Without res, d would carry
 * out's rounding into every ds of its row, where nothing averages it: at T = 4 that alone put dq off by 4e-3 of its norm
 * in bf16 (1.6e-3 is dq's own rounding). */
MCE_ATTN_API int mce_attn_fwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                              int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh,
                              const int32_t* lengths, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                              int64_t window, int64_t sinks, float scale, int dtype, void* out, void* res,
                              float* lse, void* stream);

/* dq, dk and dv from the forward's inputs, out, res and lse. The workspace holds -lse and -d (fp32 [B, Hq, 2, T]) and,
 * where the sums of dk and dv are shared by several workgroups, their fp32 parts. */
MCE_ATTN_API size_t mce_attn_bwd_ws_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                                          int64_t sinks);
MCE_ATTN_API int mce_attn_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                              int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh,
                              const void* go, int64_t go_sb, int64_t go_st, int64_t go_sh, const int32_t* lengths,
                              int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks,
                              float scale, int dtype, const void* out, const void* res, const float* lse, void* dq,
                              void* dk, void* dv, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MCE_ATTN_H */
