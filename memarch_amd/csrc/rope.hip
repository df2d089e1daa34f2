// rope.hip — norms and position rotation of query and key heads in one pass, forward and backward, for MI355X (gfx950).
// The C ABI and the formulas are in include/mce_rope.h.
//
// Both passes are HBM streams (2 element accesses per element forward, 3 backward), so the layout serves the loads: a
// head vector belongs to a group of G lanes (a power of two), each lane moving two 16-byte pieces of it (two pairs of
// them in fp32). In the half layout the two pieces are the two halves of 8 rotation pairs, interleaved they lie side by
// side; either way a lane rotates what it loaded with 8 consecutive table entries, and the norm's sum is the only value
// that crosses lanes. A group takes UNR heads of one token at once: their loads are issued together and share the
// token's table entries.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_rope.h"
#include "attn_host.h"

namespace {

constexpr int THREADS = 256;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 8 consecutive elements as fp32
template <typename T>
struct Piece {
  __device__ static __forceinline__ void load(const T* p, float (&v)[8]) {
    const u32x4 a = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = a[e];
      v[2 * e] = (float)__builtin_bit_cast(T, (uint16_t)(w & 0xFFFFu));
      v[2 * e + 1] = (float)__builtin_bit_cast(T, (uint16_t)(w >> 16));
    }
  }
  __device__ static __forceinline__ void store(T* p, const float (&v)[8]) {
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      a[e] = (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e + 1]) << 16);
    __builtin_nontemporal_store(a, reinterpret_cast<u32x4*>(p));
  }
};
template <>
struct Piece<float> {
  __device__ static __forceinline__ void load(const float* p, float (&v)[8]) {
    const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)),
                b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  }
  __device__ static __forceinline__ void store(float* p, const float (&v)[8]) {
    f32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = v[e];
      b[e] = v[4 + e];
    }
    __builtin_nontemporal_store(a, reinterpret_cast<f32x4*>(p));
    __builtin_nontemporal_store(b, reinterpret_cast<f32x4*>(p + 4));
  }
};
__device__ __forceinline__ void load_f32(const float* p, float (&v)[8]) {   // table entries and weights: kept in caches
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = a[e];
    v[4 + e] = b[e];
  }
}

struct Side {
  const void* x;
  int64_t xb, xt, xh;
  const void* g;           // upstream gradient (backward)
  int64_t gb, gt, gh;
  void* y;                 // output, or the gradient of x
  const float* w;
  float* part;             // [blocks, D] parts of the weight's gradient
  int H;
};
struct Args {
  Side side[2];            // q, k
  const float *cos, *sin;
  const void* pos;
  int64_t pos_sb, pos_st, P;
  int pos_i64;
  uint32_t tokens, T;
  uint32_t blocks_q;       // workgroups of q (the others are k's)
  int D, R, G;             // G: lanes per head vector
  float eps;
};

// table row of a token, or -1 when its position is outside the table
__device__ __forceinline__ int64_t table_row(const Args& a, uint32_t b, uint32_t t) {
  int64_t p = t;
  if (a.pos != nullptr) {
    const int64_t o = b * a.pos_sb + t * a.pos_st;
    p = a.pos_i64 ? static_cast<const int64_t*>(a.pos)[o] : (int64_t)static_cast<const int32_t*>(a.pos)[o];
  }
  return p >= 0 && p < a.P ? p : -1;
}

__device__ __forceinline__ float group_sum(float x, int G) {
  for (int o = G >> 1; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// A lane's two pieces and its table entries: lane p of the group.
struct Lane {
  int c0, c1;      // element offsets of the pieces
  bool on0, on1;   // whether they exist
  bool turns;      // whether they are rotated, by table entries 8p .. 8p+7
  __device__ __forceinline__ Lane(const Args& a, int p, bool il) {
    const int half = a.R / 2;
    turns = 8 * p < half;
    if (turns) {
      c0 = il ? 16 * p : 8 * p;
      c1 = il ? c0 + 8 : c0 + half;
    } else {
      c0 = a.R + 16 * (p - half / 8);
      c1 = c0 + 8;
    }
    on0 = c0 < a.D;
    on1 = c1 < a.D;
  }
};

// the rotation by (c, s); the inverse one with the sine's sign turned
template <bool IL>
__device__ __forceinline__ void rotate(float (&u)[8], float (&v)[8], const float (&c)[8], const float (&s)[8]) {
  if constexpr (IL) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = u[2 * e], b = u[2 * e + 1], x = v[2 * e], y = v[2 * e + 1];
      u[2 * e] = a * c[e] - b * s[e];
      u[2 * e + 1] = b * c[e] + a * s[e];
      v[2 * e] = x * c[4 + e] - y * s[4 + e];
      v[2 * e + 1] = y * c[4 + e] + x * s[4 + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = u[e], b = v[e];
      u[e] = a * c[e] - b * s[e];
      v[e] = b * c[e] + a * s[e];
    }
  }
}

// A workgroup's share of one side: groups of a.G lanes over units of UNR heads of one token.
template <typename T, bool NORM, bool IL, bool BWD, int UNR>
__global__ __launch_bounds__(THREADS) void k_rope(Args a) {
  const bool kside = blockIdx.x >= a.blocks_q;
  const Side& sd = a.side[kside];
  const uint32_t block = kside ? blockIdx.x - a.blocks_q : blockIdx.x;
  const uint32_t blocks = kside ? gridDim.x - a.blocks_q : a.blocks_q;
  const int G = a.G, p = threadIdx.x & (G - 1);
  const uint32_t groups = THREADS / G, group = threadIdx.x / G;
  const uint32_t hu = (sd.H + UNR - 1) / UNR, units = a.tokens * hu;
  const Lane ln(a, p, IL);
  float w0[8] = {}, w1[8] = {}, dw0[8] = {}, dw1[8] = {};
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w0[e] = w1[e] = 1.f;
    if (ln.on0 && sd.w != nullptr) load_f32(sd.w + ln.c0, w0);
    if (ln.on1 && sd.w != nullptr) load_f32(sd.w + ln.c1, w1);
  }
  const float inv_d = 1.f / a.D;
  for (uint32_t unit = block * groups + group; unit < units; unit += blocks * groups) {
    const uint32_t tok = unit / hu, h0 = (unit - tok * hu) * UNR, b = tok / a.T, t = tok - b * a.T;
    const T* const xp = static_cast<const T*>(sd.x) + b * sd.xb + t * sd.xt;
    const T* const gp = BWD ? static_cast<const T*>(sd.g) + b * sd.gb + t * sd.gt : nullptr;
    T* const yp = static_cast<T*>(sd.y) + (int64_t)tok * sd.H * a.D;
    float x0[UNR][8], x1[UNR][8], g0[UNR][8], g1[UNR][8];
#pragma unroll
    for (int j = 0; j < UNR; ++j) {
      const bool on = h0 + j < (uint32_t)sd.H;
#pragma unroll
      for (int e = 0; e < 8; ++e) x0[j][e] = x1[j][e] = g0[j][e] = g1[j][e] = 0.f;
      if constexpr (!BWD || NORM) {
        if (on && ln.on0) Piece<T>::load(xp + (h0 + j) * sd.xh + ln.c0, x0[j]);
        if (on && ln.on1) Piece<T>::load(xp + (h0 + j) * sd.xh + ln.c1, x1[j]);
      }
      if constexpr (BWD) {
        if (on && ln.on0) Piece<T>::load(gp + (h0 + j) * sd.gh + ln.c0, g0[j]);
        if (on && ln.on1) Piece<T>::load(gp + (h0 + j) * sd.gh + ln.c1, g1[j]);
      }
    }
    const int64_t row = table_row(a, b, t);
    float c[8] = {}, s[8] = {};
    if (ln.turns && row >= 0) {
      load_f32(a.cos + row * (a.R / 2) + 8 * p, c);
      load_f32(a.sin + row * (a.R / 2) + 8 * p, s);
    }
    if constexpr (BWD) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = -s[e];
    }
    const float bad = row >= 0 ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < UNR; ++j) {
      float r = 1.f;
      if constexpr (NORM) {
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) q += x0[j][e] * x0[j][e] + x1[j][e] * x1[j][e];
        r = 1.f / sqrtf(group_sum(q, G) * inv_d + a.eps);
      }
      float(&u)[8] = BWD ? g0[j] : x0[j];
      float(&v)[8] = BWD ? g1[j] : x1[j];
      if constexpr (NORM && !BWD) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[e] = u[e] * r * w0[e];
          v[e] = v[e] * r * w1[e];
        }
      }
      if (ln.turns) rotate<IL>(u, v, c, s);
      if constexpr (NORM && BWD) {   // u, v: dn
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a0 = x0[j][e] * r, a1 = x1[j][e] * r;
          if (h0 + j < (uint32_t)sd.H) {
            dw0[e] += u[e] * a0;
            dw1[e] += v[e] * a1;
          }
          x0[j][e] = a0;
          x1[j][e] = a1;
          u[e] *= w0[e];
          v[e] *= w1[e];
          dot += u[e] * a0 + v[e] * a1;
        }
        dot = group_sum(dot, G) * inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[e] = r * (u[e] - x0[j][e] * dot);
          v[e] = r * (v[e] - x1[j][e] * dot);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] += bad;
        v[e] += bad;
      }
      if (h0 + j < (uint32_t)sd.H) {
        if (ln.on0) Piece<T>::store(yp + (int64_t)(h0 + j) * a.D + ln.c0, u);
        if (ln.on1) Piece<T>::store(yp + (int64_t)(h0 + j) * a.D + ln.c1, v);
      }
    }
    if constexpr (NORM && BWD) {
      if (row < 0) dw0[0] += bad;   // one NaN is enough to show
    }
  }
  if constexpr (NORM && BWD) {
    __shared__ float red[THREADS / 64][256];
    // lanes of one wave with the same place in their groups, then the waves
#pragma unroll
    for (int e = 0; e < 8; ++e)
      for (int o = 32; o >= G; o >>= 1) {
        dw0[e] += __shfl_xor(dw0[e], o);
        dw1[e] += __shfl_xor(dw1[e], o);
      }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < G) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (ln.on0) red[wave][ln.c0 + e] = dw0[e];
        if (ln.on1) red[wave][ln.c1 + e] = dw1[e];
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < a.D && sd.part != nullptr) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < THREADS / 64; ++i) v += red[i][threadIdx.x];
      sd.part[(int64_t)block * a.D + threadIdx.x] = v;
    }
  }
}

// Any alignment, any even R: one wave per head vector, lane e the elements e, e + 64, ...; a rotation pair's other
// element is read again (from the cache).
template <typename T, bool NORM, bool IL, bool BWD>
__global__ __launch_bounds__(THREADS) void k_rope_any(Args a) {
  constexpr int E = 4;   // elements per lane: D <= 256
  const bool kside = blockIdx.x >= a.blocks_q;
  const Side& sd = a.side[kside];
  const uint32_t block = kside ? blockIdx.x - a.blocks_q : blockIdx.x;
  const uint32_t blocks = kside ? gridDim.x - a.blocks_q : a.blocks_q;
  const int lane = threadIdx.x & 63;
  const uint32_t wave = threadIdx.x >> 6, units = a.tokens * sd.H;
  float dw[E] = {};
  for (uint32_t unit = block * (THREADS / 64) + wave; unit < units; unit += blocks * (THREADS / 64)) {
    const uint32_t tok = unit / sd.H, h = unit - tok * sd.H, b = tok / a.T, t = tok - b * a.T;
    const T* const xp = static_cast<const T*>(sd.x) + b * sd.xb + t * sd.xt + h * sd.xh;
    const T* const gp = BWD ? static_cast<const T*>(sd.g) + b * sd.gb + t * sd.gt + h * sd.gh : nullptr;
    T* const yp = static_cast<T*>(sd.y) + ((int64_t)tok * sd.H + h) * a.D;
    const int64_t row = table_row(a, b, t);
    float q = 0.f, dot = 0.f, x[E], n[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = lane + 64 * i;
      x[i] = e < a.D && (NORM || !BWD) ? (float)xp[e] : 0.f;
      q += x[i] * x[i];
    }
    const float r = NORM ? 1.f / sqrtf(group_sum(q, 64) / a.D + a.eps) : 1.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = lane + 64 * i;
      n[i] = 0.f;
      if (e >= a.D) continue;
      // element e of the (inverse) rotation of src, and its partner
      const bool turns = e < a.R, second = turns && (IL ? (e & 1) : e >= a.R / 2);
      const int o = !turns ? e : IL ? e ^ 1 : second ? e - a.R / 2 : e + a.R / 2;
      const int i2 = IL ? e >> 1 : second ? e - a.R / 2 : e;
      float own, other;
      if (BWD) {
        own = (float)gp[e];
        other = (float)gp[o];
      } else {
        own = x[i];
        other = (float)xp[o];
        if (NORM) {
          own = own * r * (sd.w != nullptr ? sd.w[e] : 1.f);
          other = other * r * (sd.w != nullptr ? sd.w[o] : 1.f);
        }
      }
      if (turns) {
        const float c = row >= 0 ? a.cos[row * (a.R / 2) + i2] : 0.f;
        float s = row >= 0 ? a.sin[row * (a.R / 2) + i2] : 0.f;
        if (BWD) s = -s;
        own = second ? own * c + other * s : own * c - other * s;
      }
      if (row < 0) own = __builtin_nanf("");
      if (NORM && BWD) {
        dw[i] += own * x[i] * r;
        own *= sd.w != nullptr ? sd.w[e] : 1.f;
        dot += own * x[i] * r;
      }
      n[i] = own;
    }
    if (NORM && BWD) dot = group_sum(dot, 64) / a.D;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = lane + 64 * i;
      if (e < a.D) yp[e] = (T)(NORM && BWD ? r * (n[i] - x[i] * r * dot) : n[i]);
    }
  }
  if constexpr (NORM && BWD) {
    __shared__ float red[THREADS / 64][256];
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (lane + 64 * i < a.D) red[wave][lane + 64 * i] = dw[i];
    __syncthreads();
    if ((int)threadIdx.x < a.D && sd.part != nullptr) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < THREADS / 64; ++i) v += red[i][threadIdx.x];
      sd.part[(int64_t)block * a.D + threadIdx.x] = v;
    }
  }
}

// dw[c] = sum of the parts of column c, 64 rows apart per lane in a fixed order: one wave per column of a side.
__global__ __launch_bounds__(64) void k_rope_dw(const float* part_q, int nq, const float* part_k, int nk, float* dqw,
                                                float* dkw, int D) {
  const bool kside = (int)blockIdx.x >= D;
  const int c = kside ? blockIdx.x - D : blockIdx.x, n = kside ? nk : nq;
  const float* const p = kside ? part_k : part_q;
  float v = 0.f;
  for (int i = threadIdx.x; i < n; i += 64) v += p[(int64_t)i * D + c];
  v = group_sum(v, 64);
  if (threadIdx.x == 0) (kside ? dkw : dqw)[c] = v;
}

// -------------------------------------------------------------------------------------------------------- host side

int64_t lanes_of(int64_t D, int64_t R) { return R / 16 + (D - R + 15) / 16; }
int group_of(int64_t lanes) {
  int g = 1;
  while (g < lanes) g *= 2;
  return g;
}

// Workgroups of the backward's two sides: in proportion to their heads, at most MAX_BLOCKS together.
constexpr int64_t MAX_BLOCKS = 1024;
void bwd_blocks(int64_t tokens, int64_t Hq, int64_t Hkv, int64_t& nq, int64_t& nk) {
  const int64_t per = 16;   // head vectors below which another workgroup does not pay
  nq = (tokens * Hq + per - 1) / per;
  nk = (tokens * Hkv + per - 1) / per;
  if (nq + nk > MAX_BLOCKS) {
    nq = MAX_BLOCKS * Hq / (Hq + Hkv);
    if (nq < 1) nq = 1;
    if (nq > MAX_BLOCKS - 1) nq = MAX_BLOCKS - 1;
    nk = MAX_BLOCKS - nq;
  }
}

bool bad_sizes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  return B < 0 || T < 0 || Hq < 1 || Hkv < 1 || D < 2 || D > 256 || Hq > 65536 || Hkv > 65536 ||
         B > (int64_t(1) << 31) || T > (int64_t(1) << 31) || (B > 0 && T > (int64_t(1) << 31) / B) ||
         B * T * (Hq > Hkv ? Hq : Hkv) >= (int64_t(1) << 31);
}

bool whole_pieces(const void* p, int64_t sb, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (sb | st | sh) % 8 == 0;
}

using attn::finish;

template <typename T, bool NORM, bool IL, bool BWD>
void launch(Args& a, bool pieces, int64_t nq, int64_t nk, hipStream_t st) {
  if (BWD) {
    a.blocks_q = (uint32_t)nq;
    if (pieces)
      hipLaunchKernelGGL((k_rope<T, NORM, IL, BWD, 2>), dim3((unsigned)(nq + nk)), dim3(THREADS), 0, st, a);
    else
      hipLaunchKernelGGL((k_rope_any<T, NORM, IL, BWD>), dim3((unsigned)(nq + nk)), dim3(THREADS), 0, st, a);
    return;
  }
  if (!pieces) {
    auto blocks = [&](int H) { return (uint32_t)(((int64_t)a.tokens * H + THREADS / 64 - 1) / (THREADS / 64)); };
    a.blocks_q = blocks(a.side[0].H);
    hipLaunchKernelGGL((k_rope_any<T, NORM, IL, BWD>), dim3(a.blocks_q + blocks(a.side[1].H)), dim3(THREADS), 0, st, a);
    return;
  }
  auto blocks = [&](int H, int unr) {
    return (uint32_t)(((int64_t)a.tokens * ((H + unr - 1) / unr) * a.G + THREADS - 1) / THREADS);
  };
  a.blocks_q = blocks(a.side[0].H, 4);
  hipLaunchKernelGGL((k_rope<T, NORM, IL, BWD, 4>), dim3(a.blocks_q + blocks(a.side[1].H, 4)), dim3(THREADS), 0, st, a);
}

template <bool BWD>
int run(Args& a, int norm, int interleaved, int dtype, bool pieces, int64_t nq, int64_t nk, hipStream_t st) {
#define MCE_ROPE_CASE(T)                                                  \
  if (norm) {                                                             \
    if (interleaved) launch<T, true, true, BWD>(a, pieces, nq, nk, st);   \
    else launch<T, true, false, BWD>(a, pieces, nq, nk, st);              \
  } else {                                                                \
    if (interleaved) launch<T, false, true, BWD>(a, pieces, nq, nk, st);  \
    else launch<T, false, false, BWD>(a, pieces, nq, nk, st);             \
  }
  switch (dtype) {
    case MCE_ROPE_F32: MCE_ROPE_CASE(float); break;
    case MCE_ROPE_BF16: MCE_ROPE_CASE(__bf16); break;
    default: MCE_ROPE_CASE(_Float16); break;
  }
#undef MCE_ROPE_CASE
  return finish();
}

int check(const void* q, const void* k, const float* cos, const float* sin, int64_t P, const void* positions,
          const float* qw, const float* kw, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t R,
          int norm, float eps, int dtype, const void* yq, const void* yk) {
  if (bad_sizes(B, T, Hq, Hkv, D) || R < 2 || R > D || R % 2 || P < 0 || dtype < 0 || dtype > 2 || !(eps >= 0.f))
    return MCE_ROPE_EINVAL;
  if (positions == nullptr && T > P) return MCE_ROPE_EINVAL;
  if (B == 0 || T == 0) return MCE_ROPE_OK;
  if (q == nullptr || k == nullptr || yq == nullptr || yk == nullptr || ((cos == nullptr || sin == nullptr) && P > 0) ||
      (norm && (qw == nullptr) != (kw == nullptr)))
    return MCE_ROPE_EINVAL;
  return MCE_ROPE_OK;
}

}  // namespace

extern "C" {

int mce_rope_fwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                 int64_t k_sh, const float* cos, const float* sin, int64_t P, const void* positions, int pos_i64,
                 int64_t pos_sb, int64_t pos_st, const float* qw, const float* kw, int64_t B, int64_t T, int64_t Hq,
                 int64_t Hkv, int64_t D, int64_t R, int norm, float eps, int interleaved, int dtype, void* q_out,
                 void* k_out, void* stream) {
  const int rc = check(q, k, cos, sin, P, positions, qw, kw, B, T, Hq, Hkv, D, R, norm, eps, dtype, q_out, k_out);
  if (rc || B == 0 || T == 0) return rc;
  Args a = {};
  a.side[0] = {q, q_sb, q_st, q_sh, nullptr, 0, 0, 0, q_out, qw, nullptr, (int)Hq};
  a.side[1] = {k, k_sb, k_st, k_sh, nullptr, 0, 0, 0, k_out, kw, nullptr, (int)Hkv};
  a.cos = cos;
  a.sin = sin;
  a.pos = positions;
  a.pos_sb = pos_sb;
  a.pos_st = pos_st;
  a.P = P;
  a.pos_i64 = pos_i64;
  a.tokens = (uint32_t)(B * T);
  a.T = (uint32_t)T;
  a.D = (int)D;
  a.R = (int)R;
  a.eps = eps;
  const bool pieces = D % 8 == 0 && R % 16 == 0 && whole_pieces(q, q_sb, q_st, q_sh) &&
                      whole_pieces(k, k_sb, k_st, k_sh) && whole_pieces(q_out, 0, 0, 0) &&
                      whole_pieces(k_out, 0, 0, 0) && whole_pieces(cos, 0, 0, 0) && whole_pieces(sin, 0, 0, 0) &&
                      whole_pieces(qw, 0, 0, 0) && whole_pieces(kw, 0, 0, 0);
  a.G = group_of(lanes_of(D, R));
  return run<false>(a, norm, interleaved, dtype, pieces, 0, 0, reinterpret_cast<hipStream_t>(stream));
}

size_t mce_rope_bwd_ws_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int norm) {
  if (bad_sizes(B, T, Hq, Hkv, D) || !norm) return 0;
  int64_t nq, nk;
  bwd_blocks(B * T, Hq, Hkv, nq, nk);
  return (size_t)((nq + nk) * D * 4 + 255) / 256 * 256;
}

int mce_rope_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                 int64_t k_sh, const void* gq, int64_t gq_sb, int64_t gq_st, int64_t gq_sh, const void* gk,
                 int64_t gk_sb, int64_t gk_st, int64_t gk_sh, const float* cos, const float* sin, int64_t P,
                 const void* positions, int pos_i64, int64_t pos_sb, int64_t pos_st, const float* qw, const float* kw,
                 int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t R, int norm, float eps,
                 int interleaved, int dtype, void* dq, void* dk, float* dqw, float* dkw, void* ws, size_t ws_bytes,
                 void* stream) {
  const int rc = check(q, k, cos, sin, P, positions, qw, kw, B, T, Hq, Hkv, D, R, norm, eps, dtype, dq, dk);
  if (rc) return rc;
  const bool weights = norm && dqw != nullptr;
  if (norm && (dqw == nullptr) != (dkw == nullptr)) return MCE_ROPE_EINVAL;
  const bool empty = B == 0 || T == 0;
  if (!empty && (gq == nullptr || gk == nullptr)) return MCE_ROPE_EINVAL;
  if (weights && !empty &&
      (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < mce_rope_bwd_ws_bytes(B, T, Hq, Hkv, D, norm)))
    return MCE_ROPE_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  int64_t nq = 0, nk = 0;
  float* const part = static_cast<float*>(ws);
  if (!empty) {
    bwd_blocks(B * T, Hq, Hkv, nq, nk);
    Args a = {};
    a.side[0] = {q, q_sb, q_st, q_sh, gq, gq_sb, gq_st, gq_sh, dq, qw, weights ? part : nullptr, (int)Hq};
    a.side[1] = {k, k_sb, k_st, k_sh, gk, gk_sb, gk_st, gk_sh, dk, kw, weights ? part + nq * D : nullptr, (int)Hkv};
    a.cos = cos;
    a.sin = sin;
    a.pos = positions;
    a.pos_sb = pos_sb;
    a.pos_st = pos_st;
    a.P = P;
    a.pos_i64 = pos_i64;
    a.tokens = (uint32_t)(B * T);
    a.T = (uint32_t)T;
    a.D = (int)D;
    a.R = (int)R;
    a.eps = eps;
    const bool pieces = D % 8 == 0 && R % 16 == 0 && whole_pieces(q, q_sb, q_st, q_sh) &&
                        whole_pieces(k, k_sb, k_st, k_sh) && whole_pieces(gq, gq_sb, gq_st, gq_sh) &&
                        whole_pieces(gk, gk_sb, gk_st, gk_sh) && whole_pieces(dq, 0, 0, 0) &&
                        whole_pieces(dk, 0, 0, 0) && whole_pieces(cos, 0, 0, 0) && whole_pieces(sin, 0, 0, 0) &&
                        whole_pieces(qw, 0, 0, 0) && whole_pieces(kw, 0, 0, 0);
    a.G = group_of(lanes_of(D, R));
    const int e = run<true>(a, norm, interleaved, dtype, pieces, nq, nk, st);
    if (e) return e;
  }
  if (weights) {
    hipLaunchKernelGGL(k_rope_dw, dim3((unsigned)(2 * D)), dim3(64), 0, st, part, (int)nq, part + nq * D, (int)nk, dqw,
                       dkw, (int)D);
    return finish();
  }
  return MCE_ROPE_OK;
}

}  // extern "C"
