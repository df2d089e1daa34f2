// attn_tile.h — LDS tiles and MFMA fragments shared by the attention kernels (gfx950).
//
// A tile is ROWS x DP elements of 16 bits (DP = 64 or 128, the head dimension rounded up) with rows of DP * 2 bytes
// made of DP/8 chunks of 16 bytes. Chunk c of row r lies at r * DP*2 + ((c ^ swz(r)) << 4). Two kinds of fragments of
// v_mfma_f32_32x32x16 are read from it:
//   rows   lane l holds 8 consecutive columns of row l%32 (ds_read_b128): the operand whose summed index is the column;
//   tr     lane l holds 8 rows of column l%32 (two ds_read_b64_tr_b16): the operand whose summed index is the row.
// The accumulator of a 32x32 product holds, in lane l, column l%32 and the rows 8*(e/4) + 4*(l/32) + e%4 (e = 0..15).
// The elements 8s .. 8s+7 of it are therefore the fragment of a following product over those rows, once the other
// operand's tr fragment takes its 8 rows in the same order: 16s + 4(l/32) + {0..3} and 16s + 8 + 4(l/32) + {0..3}.
// No value crosses lanes between the two products.
#ifndef MEMARCH_ATTN_TILE_H
#define MEMARCH_ATTN_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef int32_t attn_i32x4 __attribute__((ext_vector_type(4)));
// The LLVM intrinsic behind buffer_load_dwordx4: (resource, per-lane offset, scalar offset, cache policy).
__device__ attn_i32x4 attn_buffer_load16(attn_i32x4 rsrc, int voffset, int soffset, int aux) __asm(
    "llvm.amdgcn.raw.buffer.load.v4i32");

namespace attn {

#define LDS_AS __attribute__((address_space(3)))

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef attn_i32x4 i32x4;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// Where a maximum's product m c (c = scale log2 e) is larger, the scores have m taken off before they are multiplied by c:
// s c - m c would carry the rounding of m c, which makes the exponential of the maximum itself 0 or infinite from about 2^30
// on. The difference is exact next to m; below the limit (a rounding of 2^-7 at most) one instruction does both.
constexpr float LARGE = 131072.f;
constexpr int OOB = 0x7FFFFFFF;          // a byte offset past every resource's records
constexpr int BUF_DWORD3 = 0x00020000;   // gfx9 buffer resource word 3 (raw, 32-bit data format)

template <typename T>
__device__ __forceinline__ f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c);
template <>
__device__ __forceinline__ f32x16 mfma<__bf16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
template <>
__device__ __forceinline__ f32x16 mfma<_Float16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two fp32 values rounded to nearest even into one register.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T T2 __attribute__((ext_vector_type(2)));
  T2 v;
  v[0] = (T)a;
  v[1] = (T)b;
  return __builtin_bit_cast(uint32_t, v);
}
template <typename T>
__device__ __forceinline__ float lo_f32(uint32_t x) { return (float)__builtin_bit_cast(T, (uint16_t)(x & 0xFFFFu)); }
template <typename T>
__device__ __forceinline__ float hi_f32(uint32_t x) { return (float)__builtin_bit_cast(T, (uint16_t)(x >> 16)); }

// s_waitcnt vmcnt(N) (the other counters left alone). gfx9 encoding: vmcnt[3:0], and vmcnt[5:4] at bits 15:14.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// A buffer resource of `records` bytes at a wave-uniform address: loads past the records return zeros and touch no
// memory.
__device__ __forceinline__ i32x4 make_rsrc(const void* p, int records) {
  const uint64_t addr = reinterpret_cast<uint64_t>(p);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)addr);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(addr >> 32) & 0xFFFFu));
  r[2] = __builtin_amdgcn_readfirstlane(records);
  r[3] = BUF_DWORD3;
  return r;
}

__device__ __forceinline__ u32x4 load16(const i32x4& rsrc, int voff) {
  return __builtin_bit_cast(u32x4, attn_buffer_load16(rsrc, voff, 0, 0));
}

// 16 bytes per lane from a resource straight into LDS at lds + dst + 16 * lane (M0, which the compiler sets). Written as an
// instruction of its own because the compiler waits for every pending load of a kind it knows before each transposing LDS
// read; the kernels order these loads themselves (wait_vmcnt, then a barrier, before the tile's first read). A vector memory
// instruction may read a scalar register only five states after a vector instruction (readfirstlane) has written it, and the
// compiler does not look for that inside an asm block: the block waits them itself, whatever stands in front.
__device__ __forceinline__ void dma16(const i32x4& rsrc, const char* lds, int dst, int voff) {
  const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(LDS_AS const char*)lds + (uint32_t)dst);
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "{m0}"(a), "v"(voff), "s"(rsrc) : "memory");
}

// The same with 4 bytes per lane, at lds + dst + 4 * lane.
__device__ __forceinline__ void dma4(const i32x4& rsrc, const char* lds, int dst, int voff) {
  const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(LDS_AS const char*)lds + (uint32_t)dst);
  asm volatile("s_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" : : "{m0}"(a), "v"(voff), "s"(rsrc) : "memory");
}

// The swizzle: 8 consecutive rows at one chunk fall on the 8 different 16-byte bank groups of 128 bytes and 16 on the
// 16 of 256 bytes (ds_read_b128), and the 4 rows x 32 bytes (16 lanes) or x 64 bytes (32 lanes) of a transposing read
// likewise, so both kinds of reads are free of bank conflicts whichever width the LDS serves at once.
template <int DP>
__device__ __forceinline__ int swz(int r) {
  const int r0 = r & 1, r1 = (r >> 1) & 1, r2 = (r >> 2) & 1, r3 = (r >> 3) & 1;
  if constexpr (DP == 128) return ((r1 ^ r3) << 3) | (r0 << 2) | (r1 << 1) | r2;
  else return (r1 << 2) | ((r0 ^ r3) << 1) | r2;
}

// Loads of a tile of ROWS rows by NW waves: instruction i moves 1 KiB of the image; wave w issues i = w, w + NW, ... A
// wave's instructions are a multiple of 16 rows apart, so they have one swizzle, and one offset per lane serves them all
// (a lane without a column stays past every resource's records).
template <int DP, int ROWS, int NW>
struct TileLoad {
  static constexpr int ROWB = DP * 2;
  static constexpr int BYTES = ROWS * ROWB;
  static constexpr int RPI = 1024 / ROWB;            // rows per instruction
  static constexpr int N = BYTES / 1024 / NW;        // instructions per wave
  static_assert(BYTES % (1024 * NW) == 0 && NW * RPI % 16 == 0, "whole instructions per wave, 16 rows apart");
  int voff, step;
  // ldb: bytes between rows; d: columns that exist (a multiple of 8): the others read zeros
  __device__ __forceinline__ void init(int ldb, int d, int wave, int lane) {
    const int row = wave * RPI + lane / (DP / 8);
    const int c = (lane % (DP / 8)) ^ swz<DP>(row);
    voff = c * 8 < d ? row * ldb + c * 16 : OOB;
    step = NW * RPI * ldb;
  }
  __device__ __forceinline__ void issue(const i32x4& rsrc, const char* lds, int img, int wave) const {
    int v = voff;
    asm volatile("" : "+v"(v));                      // the sums below are made again each time: registers are scarce
#pragma unroll
    for (int j = 0; j < N; ++j) {
      dma16(rsrc, lds, img + (j * NW + wave) * 1024, v);
      v += step;
    }
  }
};

// The resource of the tile of rows row0 .. row0 + ROWS - 1 (of `rows` that exist) at p: rows past the last read zeros.
template <int ROWS>
__device__ __forceinline__ i32x4 tile_rsrc(const uint16_t* p, int64_t ld, int row0, int rows, int d) {
  int left = rows - row0;
  left = left < 0 ? 0 : (left > ROWS ? ROWS : left);
  return make_rsrc(p + (int64_t)row0 * ld, left == 0 ? 0 : (int)((left - 1) * ld + d) * 2);
}

// Per-lane byte offsets of the fragments inside a tile. A column slice (16 columns, ks) or block (32 columns, dt) is some
// bits of the chunk number, which the swizzle leaves where they are, so the offset of any is the first one's with those
// bits flipped.
template <int DP>
struct FragAddr {
  uint32_t row;     // rows fragment of column slice 0, row block 0
  uint32_t tr[2];   // tr fragment of column block 0, row slice 0: rows 0..7 and 8..15
  __device__ __forceinline__ void init(int lane) {
    const int r = lane & 31, h = lane >> 5;
    row = r * DP * 2 + ((h ^ swz<DP>(r)) << 4);
    const int g = (lane >> 4) & 1, j = (lane >> 2) & 3, q = lane & 3;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int rr = 8 * t + 4 * h + j;
      tr[t] = rr * DP * 2 + (((2 * g + (q >> 1)) ^ swz<DP>(rr)) << 4) + 8 * (q & 1);
    }
  }
  // Forbids keeping the flipped offsets in registers past this point (a kernel short of registers calls it once per
  // tile; the flips are then made again, one instruction each).
  __device__ __forceinline__ void refresh() { asm volatile("" : "+v"(row), "+v"(tr[0]), "+v"(tr[1])); }
};

// rows fragment: rows rb*32 .. +31, columns 16 ks .. +15 (rb and img are compile-time or scalar: immediates)
template <int DP>
__device__ __forceinline__ u32x4 frag_rows(const char* lds, const FragAddr<DP>& ad, int img, int rb, int ks) {
  return *reinterpret_cast<const u32x4*>(lds + (ad.row ^ (ks << 5)) + img + rb * 32 * DP * 2);
}
// tr fragment: columns 32 dt .. +31, rows of slice kk (16 rows) in the accumulator's order. With DP = 128 the swizzle of
// a row 8 further differs in the chunk's highest bit, as the column blocks dt and dt ^ 2 do: the second half needs no
// offset of its own.
template <int DP>
__device__ __forceinline__ u32x4 frag_tr(const char* lds, const FragAddr<DP>& ad, int img, int dt, int kk) {
  const int off = img + kk * 16 * DP * 2;
  const uint32_t first = ad.tr[0] ^ (dt << 6);
  const uint32_t second = DP == 128 ? (ad.tr[0] ^ ((dt ^ 2) << 6)) + 8 * DP * 2 : ad.tr[1] ^ (dt << 6);
  const u32x2 a = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)(const_cast<char*>(lds) + first + off)));
  const u32x2 b = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)(const_cast<char*>(lds) + second + off)));
  u32x4 r;
  r[0] = a[0];
  r[1] = a[1];
  r[2] = b[0];
  r[3] = b[1];
  return r;
}
// 8 accumulator values as the fragment of the following product
template <typename T>
__device__ __forceinline__ u32x4 frag_acc(const f32x16& p, int s) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = pack2<T>(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
  return r;
}

// Reductions over the two lanes that hold one accumulator column: the swap exchanges the first value's high half with
// the second's low half, so of the same value it gives the low half's and the high half's.
// (The elements are taken into scalars first: a bit_cast of one element of the pair loses its index in this compiler.)
__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float sum_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// Stores the accumulators acc[dt] (rows = columns 32 dt + ... of the result, accumulator column = its row l%32) scaled
// by f: row `row` of p, DP/32 x 16 bytes x 2 per lane. The halves exchange 4 columns of every 16, so that each lane
// stores 16 bytes. Only rows with ok and columns below d are written, those that are not live as zeros (whatever acc
// holds: 0 * NaN is no 0). RES: the values stored are what the rounding of the same call without RES leaves over, rounded
// in their turn.
template <typename T, int DP, bool RES = false>
__device__ __forceinline__ void store_acc(const f32x16 (&acc)[DP / 32], float f, uint16_t* p, int d, bool ok, bool live,
                                          int h) {
  const uint32_t keep = live ? 0xFFFFFFFFu : 0u;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // lane half h holds columns 16 s + 4 h + {0..3} (lo) and 16 s + 8 + 4 h + {0..3} (hi)
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = acc[dt][8 * s + 2 * e] * f, y = acc[dt][8 * s + 2 * e + 1] * f;
        w[e] = (RES ? pack2<T>(x - (float)(T)x, y - (float)(T)y) : pack2<T>(x, y)) & keep;
      }
      // swap(w[2], w[0])'s halves: low lanes end with columns 16 s + 0..7, high lanes with 16 s + 8..15
      const auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      const int col = 32 * dt + 16 * s + 8 * h;
      u32x4 v;
      v[0] = r0[0];
      v[1] = r1[0];
      v[2] = r0[1];
      v[3] = r1[1];
      if (ok && col < d) *reinterpret_cast<u32x4*>(p + col) = v;
    }
}

// The same as fp32, unscaled: 16 bytes per lane and group of 4 columns.
template <int DP>
__device__ __forceinline__ void store_f32(const f32x16 (&acc)[DP / 32], float* p, int d, bool ok, bool live, int h) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int col = 32 * dt + 8 * e4 + 4 * h;
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = live ? acc[dt][4 * e4 + e] : 0.f;
      if (ok && col < d) *reinterpret_cast<f32x4*>(p + col) = x;
    }
}

}  // namespace attn

#endif  // MEMARCH_ATTN_TILE_H
