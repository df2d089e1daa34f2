// cache.hip — keys and values into a paged cache of e4m3 codes, and back, for MI355X (gfx950). The C ABI and the rules of
// scales are in include/mce_cache.h.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_cache.h"
#include "attn_tile.h"
#include "cache_host.h"
#include "seq_find.h"

namespace {

using namespace attn;

constexpr int WAVES = 4;   // waves per workgroup
constexpr int THREADS = 64 * WAVES;
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Rows16 {
  const uint16_t* p;
  int64_t st, sh;
};

// ------------------------------------------------------------------------------------------------------------- write

struct WriteArgs {
  Rows16 x[2];        // keys, values
  Codes c[2];
  Paged g;
  const int32_t *lengths, *cu;
  int B, N, block;
  int64_t waves;
};

// The elements' magnitudes are ordered as their bits are: the largest of a block comes from 16-bit integer maxima.
template <typename T>
constexpr uint32_t inf_bits() { return sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7C00u : 0x7F80u; }

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// The smallest power of two s >= 2^-100 with a <= 448 s, a finite: 448 = 1.75 2^8, and a = m 2^k with m in [1, 2).
__device__ __forceinline__ float scale_for(float a) {
  const uint32_t u = __builtin_bit_cast(uint32_t, a);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = e < -100 ? -100 : e;
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// Two products as codes in the low or high half of w; infinities become NaN (x - x is NaN for them and 0 otherwise).
template <bool HI>
__device__ __forceinline__ int codes2(float x, float y, float f, int w) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_fmaf(x, f, x - x), __builtin_fmaf(y, f, y - y), w, HI);
}

// A wave takes the new tokens of one block, one head, of the keys or the values: they stay in registers between the
// largest magnitude and the rounding (NL loads of 64 pieces of 8 elements), so that memory is passed once. Large blocks
// are shared by a workgroup's waves (SPLIT): as one wave each they left the GPU short of waves (20011 tokens, 2 heads of
// 96, blocks of 128: 12.1 us, 10.1 so). Earlier codes are read only when the scale grows. Sequence b's blocks are the units
// from floor(cu[b] / block) + 2 b on: n tokens touch at most floor(n / block) + 2 blocks.
// Bound by HBM: 65536 tokens, 8 heads of 128, blocks of 32, 403 MB: 67 us, 6.0 TB/s.
// ONCE: the new rows are read past the caches.
template <typename T, int DP, int NL, bool SPLIT, bool ONCE>
__global__ __launch_bounds__(THREADS, 4) void k_cache_write(WriteArgs a) {
  constexpr int CH = DP / 8, RPI = 64 / CH;   // pieces per row, rows per load
  __shared__ uint32_t most[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w64 = SPLIT ? blockIdx.x : (int64_t)blockIdx.x * WAVES + wave;
  if (w64 >= a.waves) return;
  const uint32_t w = (uint32_t)w64;
  const Paged& g = a.g;
  const int h = w % g.Hkv, which = w / g.Hkv & 1, u = w / g.Hkv >> 1;
  int b = u, first = u, fresh = 1, i = 0;
  if (a.cu != nullptr) {
    b = last_from(a.B, u, [&](int s) { return s == 0 ? 0 : start_in(a.cu, s, a.N) / a.block + 2 * s; });
    first = start_in(a.cu, b, a.N);
    fresh = start_in(a.cu, b + 1, a.N) - first;
    i = u - (b == 0 ? 0 : first / a.block + 2 * b);
  }
  const int64_t cap = (int64_t)g.max_pages * g.page;
  const int64_t n = a.lengths[b], p0 = n - fresh, from = p0 < 0 ? 0 : p0;   // positions of the new tokens: p0 .. n - 1
  const int64_t at = (from / a.block + i) * a.block;                        // of the block's first slot
  if (fresh <= 0 || i < 0 || at >= cap || at >= n) return;
  const int lo = (int)(at > from ? at : from), hi = (int)(at + a.block < n ? at + a.block : n);
  if (lo >= hi) return;
  const int pi = (int)at / g.page, pg = g.table[b * g.bt_sb + pi];
  if (pg < 0 || pg >= g.pages) return;
  const int slot = (int)at - pi * g.page, had = lo - (int)at, cnt = hi - lo;
  const Rows16& x = which ? a.x[1] : a.x[0];
  const Codes& c = which ? a.c[1] : a.c[0];
  float* const scale = c.scale + g.scale_at(pg, slot >> 3, h);
  const float old = had > 0 ? *scale : 0.f;
  const int row = lane / CH, col = lane % CH * 8, j0 = SPLIT ? wave * NL : 0;
  const bool ok = col < g.D;
  const i32x4 r = make_rsrc(x.p + (first + (int64_t)(lo - p0)) * x.st + h * x.sh, (int)((cnt - 1) * x.st + g.D) * 2);
  u32x4 v[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    v[j] = u32x4{};
    const int o = ok ? ((j0 + j) * RPI + row) * (int)x.st * 2 + col * 2 : OOB;
    if ((j0 + j) * RPI < cnt) v[j] = __builtin_bit_cast(u32x4, attn_buffer_load16(r, o, 0, ONCE ? 2 : 0));
  }
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < NL; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max2(m, v[j][e] & 0x7FFF7FFFu);
  // over the wave's lanes, and the waves that share the block
  auto share = [&](uint32_t x) {
    for (int o = 32; o > 0; o >>= 1) x = max2(x, __shfl_xor(x, o));
    x = max2(x, x >> 16) & 0xFFFFu;
    if constexpr (SPLIT) {
      most[wave] = x;
      __syncthreads();
      x = max2(max2(most[0], most[1]), max2(most[2], most[3]));
      __syncthreads();
    }
    return x;
  };
  m = share(m);
  if (m >= inf_bits<T>()) {   // some element is not finite: the others' largest
    m = 0;
#pragma unroll
    for (int j = 0; j < NL; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t l = v[j][e] & 0x7FFFu, t = v[j][e] >> 16 & 0x7FFFu;
        m = l < inf_bits<T>() && l > m ? l : m;
        m = t < inf_bits<T>() && t > m ? t : m;
      }
    m = share(m);
  }
  const float s = fmaxf(scale_for(lo_f32<T>(m)), old), f = 1.f / s;
  uint8_t* const out = c.p + (int64_t)pg * c.sp + (int64_t)slot * c.st + h * c.sh;
  if (old > 0.f && s > old) {   // (a scale that is no positive number has codes that mean nothing)
    const float again = old / s;
    for (int j = SPLIT ? wave * RPI : 0; j < had; j += SPLIT ? WAVES * RPI : RPI) {
      if (j + row >= had || !ok) continue;
      u32x2* const p = reinterpret_cast<u32x2*>(out + (int64_t)(j + row) * c.st + col);
      u32x2 o = *p;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x2 lo2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)o[e], false);
        const f32x2 hi2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)o[e], true);
        const int t = __builtin_amdgcn_cvt_pk_fp8_f32(lo2[0] * again, lo2[1] * again, 0, false);
        o[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi2[0] * again, hi2[1] * again, t, true);
      }
      *p = o;
    }
  }
  if (lane == 0 && j0 == 0) *scale = s;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    if ((j0 + j) * RPI + row >= cnt || !ok) continue;
    u32x2 o;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t p = v[j][2 * e], q = v[j][2 * e + 1];
      o[e] = (uint32_t)codes2<true>(lo_f32<T>(q), hi_f32<T>(q), f, codes2<false>(lo_f32<T>(p), hi_f32<T>(p), f, 0));
    }
    *reinterpret_cast<u32x2*>(out + (int64_t)(had + (j0 + j) * RPI + row) * c.st + col) = o;
  }
}

// -------------------------------------------------------------------------------------------------------------- read

struct ReadArgs {
  Codes c[2];
  Paged g;
  const int32_t* cu;
  uint16_t* out[2];
  int B, rows, hs;   // hs: waves that share a group's heads
  int64_t waves;
};

constexpr int HEADS = 4;   // loads of 16 bytes per lane under way at once

// A wave takes 8 neighbouring tokens (which lie in one page) of the keys or the values, and some of the heads: 16 codes per
// lane and load, whole 128-byte lines on both sides. Rows before the first sequence and behind the last are taken as
// sequences without pages, so every row is written. Bound by HBM: 98304 tokens, 8 heads of 128, 604 MB: 135 us, 4.5 TB/s, two
// thirds of it writes. Sequence s's groups are the units from floor(start / 8) + s on.
// ONCE: the results are written past the caches.
template <typename T, int DP, bool ONCE>
__global__ __launch_bounds__(THREADS) void k_cache_read(ReadArgs a) {
  constexpr int CH = DP / 16, HPL = 64 / (8 * CH);   // pieces per head, heads per load
  const int lane = threadIdx.x & 63;
  const int64_t w64 = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
  if (w64 >= a.waves) return;
  const uint32_t w = __builtin_amdgcn_readfirstlane((uint32_t)w64);
  const Paged& g = a.g;
  const int hp = w % a.hs, which = w / a.hs & 1, u = w / a.hs >> 1;
  auto start = [&](int s) { return s == 0 ? 0 : (s > a.B + 1 ? a.rows : start_in(a.cu, s - 1, a.rows)); };
  const int s = last_from(a.B + 2, u, [&](int x) { return start(x) / 8 + x; });
  const int first = start(s), n = start(s + 1) - first, j0 = (u - first / 8 - s) * 8;
  if (j0 < 0 || j0 >= n) return;
  const Codes& c = which ? a.c[1] : a.c[0];
  uint16_t* const out = which ? a.out[1] : a.out[0];
  int pg = -1;
  uint32_t slot = 0;
  if (s > 0 && s <= a.B && j0 < (int64_t)g.max_pages * g.page) {
    const uint32_t pi = g.page8((uint32_t)j0 >> 3);
    slot = j0 - pi * g.page;
    pg = g.table[(s - 1) * g.bt_sb + pi];
    if (pg >= g.pages) pg = -1;
  }
  const int t = lane / CH % 8, col = lane % CH * 16, hl = lane / (8 * CH);
  const bool ok = col < g.D && j0 + t < n;
  for (int h0 = hp * HEADS * HPL + hl; h0 - hl < g.Hkv; h0 += a.hs * HEADS * HPL) {
    u32x4 v[HEADS];
    float f[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = h0 + i * HPL;
      v[i] = u32x4{};
      f[i] = 0.f;
      if (ok && h < g.Hkv && pg >= 0) {
        v[i] = *reinterpret_cast<const u32x4*>(c.p + (int64_t)pg * c.sp + (int64_t)(slot + t) * c.st + h * c.sh + col);
        f[i] = c.scale[g.scale_at(pg, slot >> 3, h)];
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = h0 + i * HPL;
      if (!ok || h >= g.Hkv) continue;
      u32x4 o[2];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c4 = (int)v[i][e];
          const f32x2 x = k ? __builtin_amdgcn_cvt_pk_f32_fp8(c4, true) : __builtin_amdgcn_cvt_pk_f32_fp8(c4, false);
          float y = x[0] * f[i], z = x[1] * f[i];
          if (__is_same(T, _Float16)) {   // (a NaN stays one)
            y = y > 65504.f ? 65504.f : (y < -65504.f ? -65504.f : y);
            z = z > 65504.f ? 65504.f : (z < -65504.f ? -65504.f : z);
          }
          o[e / 2][e % 2 * 2 + k] = pack2<T>(y, z);
        }
      u32x4* const to = reinterpret_cast<u32x4*>(out + ((int64_t)(first + j0 + t) * g.Hkv + h) * g.D + col);
      if constexpr (ONCE) {
        __builtin_nontemporal_store(o[0], to);
        __builtin_nontemporal_store(o[1], to + 1);
      } else {
        to[0] = o[0];
        to[1] = o[1];
      }
    }
  }
}

// --------------------------------------------------------------------------------------------------------- host side

// So many bytes of new rows are read, and of results written, past the caches (loads and stores of the non-temporal kind).
// 65536 tokens written and 98304 read back, 8 heads of 128: 227 us without, 214 with the results past them, 217 with the
// rows, 201 with both; 20011 and 120014, 2 heads of 96: 53 and 42 (the results). Both are passes with nobody who reads the results
// behind them: what such a kernel loses where the last cache (256 MiB) would have held them is not measured.
constexpr int64_t LARGE_BYTES = int64_t(1) << 26;

template <typename T, int DP, bool ONCE>
void start_write(const WriteArgs& a, hipStream_t st) {
  constexpr int RPI = 512 / DP;
  // one new token per sequence needs one load, whatever the block
  const int rows = a.cu == nullptr ? 1 : a.block, nl = (rows + RPI - 1) / RPI;
  const dim3 grid((unsigned)((a.waves + WAVES - 1) / WAVES)), threads(THREADS), each((unsigned)a.waves);
  if (nl <= 1) hipLaunchKernelGGL((k_cache_write<T, DP, 1, false, ONCE>), grid, threads, 0, st, a);
  else if (nl <= 2) hipLaunchKernelGGL((k_cache_write<T, DP, 2, false, ONCE>), grid, threads, 0, st, a);
  else if (nl <= 4) hipLaunchKernelGGL((k_cache_write<T, DP, 4, false, ONCE>), grid, threads, 0, st, a);
  else if (nl <= 8) hipLaunchKernelGGL((k_cache_write<T, DP, 8, false, ONCE>), grid, threads, 0, st, a);
  else if (nl <= 16) hipLaunchKernelGGL((k_cache_write<T, DP, 4, true, ONCE>), each, threads, 0, st, a);
  else if constexpr (DP == 128) hipLaunchKernelGGL((k_cache_write<T, 128, 8, true, ONCE>), each, threads, 0, st, a);
}

template <typename T, int DP>
int launch_write(const WriteArgs& a, hipStream_t st) {
  if ((int64_t)4 * a.N * a.g.Hkv * a.g.D >= LARGE_BYTES) start_write<T, DP, true>(a, st);
  else start_write<T, DP, false>(a, st);
  return finish();
}

template <typename T, int DP>
int launch_read(const ReadArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.waves + WAVES - 1) / WAVES)), threads(THREADS);
  if ((int64_t)4 * a.rows * a.g.Hkv * a.g.D >= LARGE_BYTES)
    hipLaunchKernelGGL((k_cache_read<T, DP, true>), grid, threads, 0, st, a);
  else
    hipLaunchKernelGGL((k_cache_read<T, DP, false>), grid, threads, 0, st, a);
  return finish();
}

bool good_dtype(int dtype) { return dtype == MCE_ATTN_BF16 || dtype == MCE_ATTN_F16; }

}  // namespace

extern "C" {

int mce_cache_write(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, void* kc,
                    int64_t kc_sp, int64_t kc_st, int64_t kc_sh, void* vc, int64_t vc_sp, int64_t vc_st, int64_t vc_sh,
                    float* k_scale, float* v_scale, const int32_t* block_table, int64_t bt_sb, const int32_t* lengths,
                    const int32_t* cu, int64_t B, int64_t N, int64_t Hkv, int64_t D, int64_t pages, int64_t page,
                    int64_t block, int64_t max_pages, int dtype, void* stream) {
  int rc = check_paged_sizes(B, Hkv, D, pages, page, block, max_pages, bt_sb);
  if (rc) return rc;
  if (N < 0 || N > (int64_t(1) << 27) || (cu == nullptr && N != B) || !good_dtype(dtype)) return MCE_ATTN_EINVAL;
  const int64_t units = cu == nullptr ? B : N / block + 2 * B, waves = units * 2 * Hkv;
  if (waves > MAX_GROUPS) return MCE_ATTN_EINVAL;
  if (B == 0 || N == 0 || pages == 0 || max_pages == 0) return MCE_ATTN_OK;
  if (lengths == nullptr || block_table == nullptr) return MCE_ATTN_EINVAL;
  if ((rc = check_strided(k, 0, k_st, k_sh, D)) || (rc = check_strided(v, 0, v_st, v_sh, D)) ||
      (rc = check_codes(kc, kc_sp, kc_st, kc_sh, k_scale, D)) || (rc = check_codes(vc, vc_sp, vc_st, vc_sh, v_scale, D)))
    return rc;
  WriteArgs a = {};
  a.x[0] = {static_cast<const uint16_t*>(k), k_st, k_sh};
  a.x[1] = {static_cast<const uint16_t*>(v), v_st, v_sh};
  a.c[0] = {static_cast<uint8_t*>(kc), kc_sp, kc_st, kc_sh, k_scale};
  a.c[1] = {static_cast<uint8_t*>(vc), vc_sp, vc_st, vc_sh, v_scale};
  a.g = make_paged(block_table, bt_sb, Hkv, D, pages, page, block, max_pages);
  a.lengths = lengths;
  a.cu = cu;
  a.B = (int)B;
  a.N = (int)N;
  a.block = (int)block;
  a.waves = waves;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_write<__bf16, 64>(a, st) : launch_write<__bf16, 128>(a, st);
  return D <= 64 ? launch_write<_Float16, 64>(a, st) : launch_write<_Float16, 128>(a, st);
}

int mce_cache_read(const void* kc, int64_t kc_sp, int64_t kc_st, int64_t kc_sh, const void* vc, int64_t vc_sp,
                   int64_t vc_st, int64_t vc_sh, const float* k_scale, const float* v_scale, const int32_t* block_table,
                   int64_t bt_sb, const int32_t* cu, int64_t B, int64_t rows, int64_t Hkv, int64_t D, int64_t pages,
                   int64_t page, int64_t block, int64_t max_pages, int dtype, void* k, void* v, void* stream) {
  int rc = check_paged_sizes(B, Hkv, D, pages, page, block, max_pages, bt_sb);
  if (rc) return rc;
  if (rows < 0 || rows > (int64_t(1) << 27) || !good_dtype(dtype)) return MCE_ATTN_EINVAL;
  // few tokens: their heads over several waves, so that no wave has more than one round of loads
  const int64_t round = HEADS * (D <= 64 ? 2 : 1), all = (Hkv + round - 1) / round, units = rows / 8 + B + 2;
  const int64_t hs = units * 2 * all <= 16384 ? all : 1, waves = units * 2 * hs;
  if (waves > MAX_GROUPS * WAVES) return MCE_ATTN_EINVAL;
  if (rows == 0) return MCE_ATTN_OK;
  if (cu == nullptr || k == nullptr || v == nullptr || (block_table == nullptr && B > 0 && pages > 0 && max_pages > 0))
    return MCE_ATTN_EINVAL;
  if (pages > 0 && ((rc = check_codes(kc, kc_sp, kc_st, kc_sh, k_scale, D)) ||
                    (rc = check_codes(vc, vc_sp, vc_st, vc_sh, v_scale, D))))
    return rc;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return MCE_ATTN_EALIGN;
  ReadArgs a = {};
  a.c[0] = {static_cast<uint8_t*>(const_cast<void*>(kc)), kc_sp, kc_st, kc_sh, const_cast<float*>(k_scale)};
  a.c[1] = {static_cast<uint8_t*>(const_cast<void*>(vc)), vc_sp, vc_st, vc_sh, const_cast<float*>(v_scale)};
  a.g = make_paged(block_table, bt_sb, Hkv, D, pages, page, block, max_pages);
  a.cu = cu;
  a.out[0] = static_cast<uint16_t*>(k);
  a.out[1] = static_cast<uint16_t*>(v);
  a.B = (int)B;
  a.rows = (int)rows;
  a.hs = (int)hs;
  a.waves = waves;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_read<__bf16, 64>(a, st) : launch_read<__bf16, 128>(a, st);
  return D <= 64 ? launch_read<_Float16, 64>(a, st) : launch_read<_Float16, 128>(a, st);
}

}  // extern "C"
