/*
 * mce_rope.h — C ABI of the MI355X (gfx950) kernels for norms and position rotation of query and key heads
 * (libmce_attn.so).
 *
 * memarch's blocks norm and rotate with torch operations before scaled_dot_product_attention (baseline.py:35-53).
 *
 * For each head vector x [D] of q and k, with the side's weight w [D] and the table rows c, s [R/2] of its position:
 *   n = x w / sqrt(mean(x^2) + eps)      (norm = 0: n = x)
 *   pairs (a, b) = (i, i + R/2), or (2i, 2i + 1) with interleaved != 0, for i < R/2:
 *     y_a = n_a c_i - n_b s_i,  y_b = n_b c_i + n_a s_i;   y_j = n_j for j >= R
 * and backward, dn being the inverse rotation of the upstream gradient g and r = 1 / sqrt(mean(x^2) + eps):
 *   dw = sum over tokens and heads of dn x r;   dx = r (dn w - x r^2 mean(dn w x))      (norm = 0: dx = dn)
 * (weights NULL, both: 1). All arithmetic is fp32, results are rounded once to the element type of q and k; weights, tables and dw are fp32.
 *
 * The position of token t of sequence b is positions[b * pos_sb + t * pos_st] (int64 with pos_i64 != 0, else int32), or
 * t with positions NULL. A position outside [0, P) gives NaN in that token's heads, in their gradients and in all of dw.
 *
 * Buffers: q [B, T, Hq, D] and k [B, T, Hkv, D] with element strides (batch, token, head) and a contiguous last
 * dimension, gradients g like them; cos and sin [P, R/2] contiguous; outputs contiguous. Any alignment and any even
 * R <= D <= 256: heads made of whole 16-byte pieces (of n = 8 elements, 4 in fp32: all pointers 16-byte aligned, strides
 * and D multiples of n, and R/2, or with interleaved pairs R) move as such, others element by element. Every call is asynchronous on `stream`, allocates nothing, and returns 0 or
 * an MCE_ROPE_E* code; arguments are checked before anything is launched.
 */
#ifndef MCE_ROPE_H
#define MCE_ROPE_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define MCE_ROPE_API __attribute__((visibility("default")))
#else
#define MCE_ROPE_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define MCE_ROPE_OK 0
#define MCE_ROPE_EINVAL 1     /* size, stride, element type or null pointer */
#define MCE_ROPE_EWORKSPACE 3 /* workspace missing, too small or not 256-byte aligned */
#define MCE_ROPE_ELAUNCH 4    /* a HIP launch failed (mce_attn_last_hip_error; the codes' texts: mce_attn_error_string) */

/* element types of q, k, their gradients and the outputs */
#define MCE_ROPE_F32 0
#define MCE_ROPE_BF16 1
#define MCE_ROPE_F16 2

MCE_ROPE_API int mce_rope_fwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                              int64_t k_st, int64_t k_sh, const float* cos, const float* sin, int64_t P,
                              const void* positions, int pos_i64, int64_t pos_sb, int64_t pos_st, const float* qw,
                              const float* kw, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t R,
                              int norm, float eps, int interleaved, int dtype, void* q_out, void* k_out, void* stream);

/* dq, dk and, with norm != 0 and both not NULL, dqw and dkw (fp32 [D]; the workspace holds their parts, summed in a fixed
 * order; it may be NULL without them). */
MCE_ROPE_API size_t mce_rope_bwd_ws_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int norm);
MCE_ROPE_API int mce_rope_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                              int64_t k_st, int64_t k_sh, const void* gq, int64_t gq_sb, int64_t gq_st, int64_t gq_sh,
                              const void* gk, int64_t gk_sb, int64_t gk_st, int64_t gk_sh, const float* cos,
                              const float* sin, int64_t P, const void* positions, int pos_i64, int64_t pos_sb,
                              int64_t pos_st, const float* qw, const float* kw, int64_t B, int64_t T, int64_t Hq,
                              int64_t Hkv, int64_t D, int64_t R, int norm, float eps, int interleaved, int dtype,
                              void* dq, void* dk, float* dqw, float* dkw, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MCE_ROPE_H */
