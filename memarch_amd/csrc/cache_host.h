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

struct Paged {
  const int32_t* table;
  int64_t bt_sb;
  int pages, page, max_pages, Hkv, D;
  int per;                 // blocks per page
  uint32_t mpage, mblock;  // of the divisions by page / 8 and block / 8 (0: by 1)
  __device__ __forceinline__ static uint32_t div(uint32_t x, uint32_t magic) { return magic ? __umulhi(x, magic) : x; }
  // the scale of the 8 slots from slot8 * 8 on of page pg
  __device__ __forceinline__ int64_t scale_at(int pg, uint32_t slot8, int h) const {
    return ((int64_t)pg * per + div(slot8, mblock)) * Hkv + h;
  }
};

// x / d = the high word of x * magic_of(d) while x d < 2^32 (d = 1: 0)
inline uint32_t magic_of(int64_t d) { return d == 1 ? 0 : (uint32_t)((uint64_t(1) << 32) / (uint64_t)d + 1); }

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

inline int check_codes(const void* p, int64_t sp, int64_t st, int64_t sh, const void* scale, int64_t D) {
  if (p == nullptr || scale == nullptr || sp < 0 || sh < 0 || st < D || st > MAX_ST) return MCE_ATTN_EINVAL;
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
  g.mpage = magic_of(page / 8);
  g.mblock = magic_of(block / 8);
  return g;
}

}  // namespace attn

#endif  // MEMARCH_CACHE_HOST_H
