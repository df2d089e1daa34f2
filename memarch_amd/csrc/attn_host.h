// attn_host.h — argument checks and error state shared by the host sides of the attention library.
#ifndef MEMARCH_ATTN_HOST_H
#define MEMARCH_ATTN_HOST_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_attn.h"

extern thread_local int mce_attn_hip_error;   // the calling thread's last failed launch (attn.hip)

namespace attn {

// Token strides up to 2^21 elements keep every offset inside a tile of at most 128 rows in 31 bits.
constexpr int64_t MAX_ST = int64_t(1) << 21;

// Workgroups of up to 256 threads that a launch can hold: HIP takes fewer than 2^32 threads.
constexpr int64_t MAX_GROUPS = (int64_t(1) << 24) - 1;

inline int finish() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    mce_attn_hip_error = (int)e;
    return MCE_ATTN_ELAUNCH;
  }
  return MCE_ATTN_OK;
}

// An operand whose rows (of D elements, st apart) are read in pieces of 16 bytes.
inline int check_strided(const void* p, int64_t sb, int64_t st, int64_t sh, int64_t D) {
  if (p == nullptr || sb < 0 || sh < 0 || st < D || st > MAX_ST) return MCE_ATTN_EINVAL;
  if ((reinterpret_cast<uintptr_t>(p) & 15) || (sb | st | sh) % 8) return MCE_ATTN_EALIGN;
  return MCE_ATTN_OK;
}

// Scales outside this range leave no room for the logarithms and products that are formed with them.
inline bool good_scale(float s) { return s >= 1e-30f && s <= 1e30f; }

inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace attn

#endif  // MEMARCH_ATTN_HOST_H
