/*
 * mce_pack.h — C ABI of the MI355X (gfx950) attention over packed sequences, forward and backward (libmce_serve.so): the
 * mathematics of mce_attn.h for sequences of different lengths that lie behind each other without padding.
 *
 * Sequence s of nseq has the rows cu[s] .. cu[s + 1] - 1 of q and cu_k[s] .. cu_k[s + 1] - 1 of k and v (both arrays hold
 * nseq + 1 numbers that do not fall, in device memory; cu_k NULL: cu, with M = N). Its n rows of q are the last of its m
 * positions: row i stands at position i + m - n and sees position j of its sequence when
 *   j <= i + m - n  and  (window = 0  or  i + m - n - j < window  or  j < sinks)
 * A row that sees nothing (m < n: the first n - m rows), and rows outside every sequence (before cu[0] and from cu[nseq]
 * on) have out = 0 and dq = 0; rows of k outside every sequence have dk = dv = 0. Rows of one sequence are never used for
 * another's. Numbers in cu and cu_k outside 0 .. N (0 .. M) count as the nearest of the two; where one is smaller than the
 * one before it, what results hold is not defined (no address outside the buffers is touched).
 *
 * Buffers: q and go [N, Hq, D], k and v [M, Hkv, D] with element strides (token, head), the last dimension contiguous,
 * 16-byte aligned, strides multiples of 8, the token stride at least D; D a multiple of 8 up to 128; out, res, dq [N, Hq, D]
 * and dk, dv [M, Hkv, D] contiguous; lse [Hq, N] fp32. N and M are at most 2^27, Hq (N / 128 + nseq + 2) is below 2^24 and
 * Hkv (M / 128 + nseq + 2) below 2^23 - 2^11; with a window nseq sinks / 128 is below 2^31.
 * Roundings, ranges and the conventions of the calls are those of mce_attn.h: asynchronous on `stream`, no allocation,
 * arguments checked before anything is launched, MCE_ATTN_E* codes. The split of work depends on the sizes alone, so a
 * captured call may be replayed with other lengths.
 */
#ifndef MCE_PACK_H
#define MCE_PACK_H

#include "mce_attn.h"

#define MCE_SERVE_API MCE_ATTN_API

#ifdef __cplusplus
extern "C" {
#endif

/* Text of an MCE_ATTN_* code, and the hipError_t of the calling thread's last failed launch in this library. */
MCE_SERVE_API const char* mce_serve_error_string(int code);
MCE_SERVE_API int mce_serve_last_hip_error(void);

/* out, and for a backward (both may be NULL) res and lse, as in mce_attn_fwd. The plan, scratch memory of the forward, is the
 * order in which blocks of rows are taken, the longest first (0 bytes where their own order is as good); a backward takes the plan of
 * its forward, unchanged, which res asks for. The workspace holds parts of the sums of rows whose keys are shared by several
 * workgroups, as is done where there are few rows and many keys (else 0 bytes). */
MCE_SERVE_API size_t mce_pack_plan_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D,
                                         int64_t window, int64_t sinks);
MCE_SERVE_API size_t mce_pack_fwd_ws_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t window, int64_t sinks);
MCE_SERVE_API int mce_pack_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                               const void* v, int64_t v_st, int64_t v_sh, const int32_t* cu, const int32_t* cu_k,
                               int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                               int64_t sinks, float scale, int dtype, void* out, void* res, float* lse, void* plan,
                               size_t plan_bytes, void* ws, size_t ws_bytes, void* stream);

/* dq, dk and dv from the forward's inputs, out, res, lse and plan. The workspace holds -lse and -d (fp32 [Hq, 2, N]) and, where
 * sums may be shared by several workgroups, their fp32 parts. */
MCE_SERVE_API size_t mce_pack_bwd_ws_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t window, int64_t sinks);
MCE_SERVE_API int mce_pack_bwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                               const void* v, int64_t v_st, int64_t v_sh, const void* go, int64_t go_st, int64_t go_sh,
                               const int32_t* cu, const int32_t* cu_k, int64_t nseq, int64_t N, int64_t M, int64_t Hq,
                               int64_t Hkv, int64_t D, int64_t window, int64_t sinks, float scale, int dtype,
                               const void* out, const void* res, const float* lse, const void* plan, void* dq, void* dk,
                               void* dv, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MCE_PACK_H */
