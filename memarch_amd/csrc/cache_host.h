// cache_host.h — the paged 8-bit cache as the host sides and kernels of cache.hip and cache_attn.hip know it.
#ifndef MEMARCH_CACHE_HOST_H
#define MEMARCH_CACHE_HOST_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_host.h"

namespace attn {

// One cache (keys or values): codes with strides in bytes, and a scale per block and head.
struct Codes {
  uint8_t* p;
  int64_t sp, st, sh;
  float* scale;
};

// x / d for x d < 2^32: the high word of x * ceil(2^32 / d), and x itself for d = 1, without a branch.
struct Div {
  uint32_t m, one;
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return __umulhi(x, m) + (x & one); }
};
inline Div div_by(int64_t d) {
  return d == 1 ? Div{0, 0xFFFFFFFFu} : Div{(uint32_t)((uint64_t(1) << 32) / (uint64_t)d + 1), 0};
}

struct Paged {
  const int32_t* table;
  int64_t bt_sb;
  int pages, page, max_pages, Hkv, D;
  int per;                 // blocks per page
  Div page8, block8;       // by page / 8 and block / 8
  // the scale of the 8 slots from slot8 * 8 on of page pg
  __device__ __forceinline__ int64_t scale_at(int pg, uint32_t slot8, int h) const {
    return ((int64_t)pg * per + block8(slot8)) * Hkv + h;
  }
};

inline int check_paged_sizes(int64_t B, int64_t Hkv, int64_t D, int64_t pages, int64_t page, int64_t block,
                             int64_t max_pages, int64_t bt_sb) {
  if (B < 0 || Hkv < 1 || Hkv > 65536 || D < 16 || D > 128 || D % 16 || page < 8 || page % 8 || page > 65536 || block < 8 ||
      block % 8 || block > 128 || page % block || pages < 0 || pages > INT32_MAX || max_pages < 0 || bt_sb < 0 ||
      B > MAX_GROUPS)
    return MCE_ATTN_EINVAL;
  // positions in 30 bits, and exact divisions of an 8-slot group's number (below 2^38 / page / 8 times page / 8)
  if (max_pages > (int64_t(1) << 30) / page || max_pages * page > (int64_t(1) << 38) / page) return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

// Page strides in units of 16 bytes stay in 31 bits.
constexpr int64_t MAX_SP = int64_t(1) << 34;

inline int check_codes(const void* p, int64_t sp, int64_t st, int64_t sh, const void* scale, int64_t D) {
  if (p == nullptr || scale == nullptr || sp < 0 || sp > MAX_SP || sh < 0 || st < D || st > MAX_ST) return MCE_ATTN_EINVAL;
  if ((reinterpret_cast<uintptr_t>(p) & 15) || (sp | st | sh) % 16 || (reinterpret_cast<uintptr_t>(scale) & 3))
    return MCE_ATTN_EALIGN;
  return MCE_ATTN_OK;
}

inline Paged make_paged(const int32_t* table, int64_t bt_sb, int64_t Hkv, int64_t D, int64_t pages, int64_t page,
                        int64_t block, int64_t max_pages) {
  Paged g = {};
  g.table = table;
  g.bt_sb = bt_sb;
  g.pages = (int)pages;
  g.page = (int)page;
  g.max_pages = pages == 0 ? 0 : (int)max_pages;   // without pages nothing is in the cache
  g.Hkv = (int)Hkv;
  g.D = (int)D;
  g.per = (int)(page / block);
  g.page8 = div_by(page / 8);
  g.block8 = div_by(block / 8);
  return g;
}

}  // namespace attn

#endif  // MEMARCH_CACHE_HOST_H
