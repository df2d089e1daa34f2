// rope.hip — norms and position rotation of query and key heads in one pass, forward and backward, for MI355X (gfx950).
// The C ABI and the formulas are in include/mce_rope.h.
//
// Both passes are HBM streams (2 element accesses per element forward, 3 backward), so the layout serves the loads: a
// head vector belongs to a group of G lanes (a power of two), each lane moving two 16-byte pieces of it, neighbouring
// lanes neighbouring pieces. In the half layout a lane's two pieces are the two sides of its rotation pairs, interleaved
// pairs lie inside a piece; either way the norm's sum is the only value that crosses lanes. A group takes UNR heads of one
// token at once: their loads are issued together, kept as loaded until each is used, and share the token's table entries.
// Measured (32 x 1024 tokens of 16 + 16 heads of 128, bf16, norm): forward 96 us, 5.6 TB/s; backward 149 us, 5.4 TB/s, and 5 us
// for the weights' gradients (a large copy reaches 4.9 TB/s).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_rope.h"
#include "attn_host.h"

namespace {

constexpr int THREADS = 256;
constexpr int UNR_F = 2, UNR_B = 1;   // heads per group at once, forward and backward

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A 16-byte piece: N elements of T
template <typename T>
struct Piece {
  static constexpr int N = 8;
  __device__ static __forceinline__ void unpack(const u32x4& a, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = a[e];
      v[2 * e] = (float)__builtin_bit_cast(T, (uint16_t)(w & 0xFFFFu));
      v[2 * e + 1] = (float)__builtin_bit_cast(T, (uint16_t)(w >> 16));
    }
  }
  __device__ static __forceinline__ u32x4 pack(const float (&v)[8]) {
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      a[e] = (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e + 1]) << 16);
    return a;
  }
};
template <>
struct Piece<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void unpack(const u32x4& a, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = a[e];
      v[e] = __builtin_bit_cast(float, w);
    }
  }
  __device__ static __forceinline__ u32x4 pack(const float (&v)[4]) {
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = __builtin_bit_cast(uint32_t, v[e]);
    return a;
  }
};
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const u32x4& a) {
  __builtin_nontemporal_store(a, reinterpret_cast<u32x4*>(p));
}
// N fp32 table entries or weights (multiples of 2, 8-byte aligned at least): kept in the caches
template <int N>
__device__ __forceinline__ void load_f32(const float* p, float* v) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = a[e];
    }
  } else {
    v[0] = p[0];
    v[1] = p[1];
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

// A lane's two pieces of a head vector of D elements, N to a piece: their first elements, whether they exist and whether
// they are rotated.
template <int N, bool IL>
struct Lane {
  int c0, c1;
  bool on0, on1, turn0, turn1;
  __device__ __forceinline__ Lane(const Args& a, int p) {
    if constexpr (IL) {   // piece p and the one half the pieces further
      c0 = N * p;
      c1 = c0 + N * ((a.D / N + 1) / 2);
      on0 = p < (a.D / N + 1) / 2;
      on1 = on0 && c1 < a.D;
      turn0 = on0 && c0 < a.R;
      turn1 = on1 && c1 < a.R;
    } else {              // the two sides of N pairs; behind the rotated part as above
      const int half = a.R / 2, rest = (a.D - a.R) / N, q = p - half / N;
      turn0 = turn1 = q < 0;
      c0 = turn0 ? N * p : a.R + N * q;
      c1 = turn0 ? c0 + half : c0 + N * ((rest + 1) / 2);
      on0 = turn0 || q < (rest + 1) / 2;
      on1 = turn0 || (on0 && c1 < a.D);
    }
  }
};

// the rotation by the lane's table entries (c, s): N pairs across its pieces, or N/2 inside each
template <int N, bool IL>
__device__ __forceinline__ void rotate(float (&u)[N], float (&v)[N], const float (&c)[N], const float (&s)[N]) {
  if constexpr (IL) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float a = u[2 * e], b = u[2 * e + 1], x = v[2 * e], y = v[2 * e + 1];
      u[2 * e] = a * c[e] - b * s[e];
      u[2 * e + 1] = b * c[e] + a * s[e];
      v[2 * e] = x * c[N / 2 + e] - y * s[N / 2 + e];
      v[2 * e + 1] = y * c[N / 2 + e] + x * s[N / 2 + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float a = u[e], b = v[e];
      u[e] = a * c[e] - b * s[e];
      v[e] = b * c[e] + a * s[e];
    }
  }
}

// A workgroup's share of one side: groups of a.G lanes over units of UNR heads of one token.
template <typename T, bool NORM, bool IL, bool BWD, int UNR>
__global__ __launch_bounds__(THREADS, 4) void k_rope(Args a) {
  using P = Piece<T>;
  constexpr int N = P::N;
  const bool kside = blockIdx.x >= a.blocks_q;
  const Side sd = kside ? a.side[1] : a.side[0];
  const uint32_t block = kside ? blockIdx.x - a.blocks_q : blockIdx.x;
  const uint32_t blocks = kside ? gridDim.x - a.blocks_q : a.blocks_q;
  const int G = a.G, p = threadIdx.x & (G - 1);
  const uint32_t groups = THREADS / G, group = threadIdx.x / G;
  const uint32_t hu = (sd.H + UNR - 1) / UNR, units = a.tokens * hu;
  const Lane<N, IL> ln(a, p);
  float w0[N], w1[N], dw0[N] = {}, dw1[N] = {};
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < N; ++e) w0[e] = w1[e] = 1.f;
    if (ln.on0 && sd.w != nullptr) load_f32<N>(sd.w + ln.c0, w0);
    if (ln.on1 && sd.w != nullptr) load_f32<N>(sd.w + ln.c1, w1);
  }
  const float inv_d = 1.f / a.D;
  for (uint32_t unit = block * groups + group; unit < units; unit += blocks * groups) {
    const uint32_t tok = unit / hu, h0 = (unit - tok * hu) * UNR, b = tok / a.T, t = tok - b * a.T;
    const T* const xp = static_cast<const T*>(sd.x) + b * sd.xb + t * sd.xt;
    const T* const gp = BWD ? static_cast<const T*>(sd.g) + b * sd.gb + t * sd.gt : nullptr;
    T* const yp = static_cast<T*>(sd.y) + (int64_t)tok * sd.H * a.D;
    u32x4 xr0[UNR], xr1[UNR], gr0[UNR], gr1[UNR];
#pragma unroll
    for (int j = 0; j < UNR; ++j) {
      const bool on = h0 + j < (uint32_t)sd.H;
      xr0[j] = xr1[j] = gr0[j] = gr1[j] = u32x4{};
      if constexpr (!BWD || NORM) {
        if (on && ln.on0) xr0[j] = load_piece(xp + (h0 + j) * sd.xh + ln.c0);
        if (on && ln.on1) xr1[j] = load_piece(xp + (h0 + j) * sd.xh + ln.c1);
      }
      if constexpr (BWD) {
        if (on && ln.on0) gr0[j] = load_piece(gp + (h0 + j) * sd.gh + ln.c0);
        if (on && ln.on1) gr1[j] = load_piece(gp + (h0 + j) * sd.gh + ln.c1);
      }
    }
    // table entries; where nothing turns the identity
    const int64_t row = table_row(a, b, t);
    float c[N], s[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    if (row >= 0) {
      const int64_t o = row * (a.R / 2);
      if constexpr (IL) {
        if (ln.turn0) {
          load_f32<N / 2>(a.cos + o + ln.c0 / 2, c);
          load_f32<N / 2>(a.sin + o + ln.c0 / 2, s);
        }
        if (ln.turn1) {
          load_f32<N / 2>(a.cos + o + ln.c1 / 2, c + N / 2);
          load_f32<N / 2>(a.sin + o + ln.c1 / 2, s + N / 2);
        }
      } else if (ln.turn0) {
        load_f32<N>(a.cos + o + ln.c0, c);
        load_f32<N>(a.sin + o + ln.c0, s);
      }
    }
    if constexpr (BWD) {   // the inverse rotation
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = -s[e];
    }
#pragma unroll
    for (int j = 0; j < UNR; ++j) {
      float x0[N], x1[N], u[N], v[N];
      float r = 1.f;
      if constexpr (!BWD || NORM) {
        P::unpack(xr0[j], x0);
        P::unpack(xr1[j], x1);
      }
      if constexpr (NORM) {
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) q += x0[e] * x0[e] + x1[e] * x1[e];
        r = 1.f / sqrtf(group_sum(q, G) * inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          x0[e] *= r;
          x1[e] *= r;
        }
      }
      if constexpr (BWD) {
        P::unpack(gr0[j], u);
        P::unpack(gr1[j], v);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          u[e] = NORM ? x0[e] * w0[e] : x0[e];
          v[e] = NORM ? x1[e] * w1[e] : x1[e];
        }
      }
      // (a lane in which only one or none of its pieces turns has the identity in the other's place; half layout: both)
      if (ln.turn0) rotate<N, IL>(u, v, c, s);
      if (row < 0) {   // NaN in the head, and through it in its gradient and the weights'
#pragma unroll
        for (int e = 0; e < N; ++e) u[e] = v[e] = __builtin_nanf("");
      }
      if constexpr (NORM && BWD) {   // u, v: dn; heads past the last have zeros
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          dw0[e] += u[e] * x0[e];
          dw1[e] += v[e] * x1[e];
          u[e] *= w0[e];
          v[e] *= w1[e];
          dot += u[e] * x0[e] + v[e] * x1[e];
        }
        dot = group_sum(dot, G) * inv_d;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          u[e] = r * (u[e] - x0[e] * dot);
          v[e] = r * (v[e] - x1[e] * dot);
        }
      }
      if (h0 + j < (uint32_t)sd.H) {
        if (ln.on0) store_piece(yp + (int64_t)(h0 + j) * a.D + ln.c0, P::pack(u));
        if (ln.on1) store_piece(yp + (int64_t)(h0 + j) * a.D + ln.c1, P::pack(v));
      }
    }
  }
  if constexpr (NORM && BWD) {
    __shared__ float red[THREADS / 64][256];
    // lanes of one wave with the same place in their groups, then the waves
#pragma unroll
    for (int e = 0; e < N; ++e)
      for (int o = 32; o >= G; o >>= 1) {
        dw0[e] += __shfl_xor(dw0[e], o);
        dw1[e] += __shfl_xor(dw1[e], o);
      }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < G) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
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
// element is read again (from the cache). A step of 32 x 1024 tokens of 16 + 16 heads in bf16, norm, takes 1.06 ms with
// D = 80, R = 40 and 1.09 ms with D = 96, R = 24, where R = D in whole pieces takes 0.23 and 0.25.
template <typename T, bool NORM, bool IL, bool BWD>
__global__ __launch_bounds__(THREADS) void k_rope_any(Args a) {
  constexpr int E = 4;   // elements per lane: D <= 256
  const bool kside = blockIdx.x >= a.blocks_q;
  const Side sd = kside ? a.side[1] : a.side[0];
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

// dw[c] = sum of the parts of column c, in fp64, 64 rows apart per lane in a fixed order: one wave per column of a side.
__global__ __launch_bounds__(64) void k_rope_dw(const float* part_q, int nq, const float* part_k, int nk, float* dqw,
                                                float* dkw, int D) {
  const bool kside = (int)blockIdx.x >= D;
  const int c = kside ? blockIdx.x - D : blockIdx.x, n = kside ? nk : nq;
  const float* const p = kside ? part_k : part_q;
  double v = 0.;
  for (int i = threadIdx.x; i < n; i += 64) v += p[(int64_t)i * D + c];
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if (threadIdx.x == 0) (kside ? dkw : dqw)[c] = (float)v;
}

// -------------------------------------------------------------------------------------------------------- host side

// Lanes per head vector: two pieces of n elements each.
int group_of(int64_t D, int64_t R, int64_t n, bool interleaved) {
  const int64_t lanes = interleaved ? (D / n + 1) / 2 : R / 2 / n + ((D - R) / n + 1) / 2;
  int g = 1;
  while (g < lanes) g *= 2;
  return g;
}

// Workgroups of the backward's two sides: in proportion to their heads, at most MAX_BLOCKS (4 per CU) together.
constexpr int64_t MAX_BLOCKS = 1024;
// Workgroups of one side of the forward, at most.
constexpr int64_t MAX_BLOCKS_F = int64_t(1) << 22;
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

bool whole_pieces(const void* p, int64_t sb, int64_t st, int64_t sh, int64_t n) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (sb | st | sh) % n == 0;
}

// Whether head vectors and tables can be moved in pieces of n elements: rotation pairs across whole pieces (half layout)
// or inside them, table entries in fours (or twos: fp32, interleaved).
bool whole_layout(int64_t D, int64_t R, int64_t n, bool interleaved, const void* cos, const void* sin, const void* qw,
                  const void* kw) {
  return D % n == 0 && (interleaved ? R : R / 2) % n == 0 && (R / 2) % (interleaved ? n / 2 : n) == 0 &&
         whole_pieces(cos, 0, 0, 0, n) && whole_pieces(sin, 0, 0, 0, n) && whole_pieces(qw, 0, 0, 0, n) &&
         whole_pieces(kw, 0, 0, 0, n);
}

using attn::finish;

template <typename T, bool NORM, bool IL, bool BWD>
void launch(Args& a, bool pieces, int64_t nq, int64_t nk, hipStream_t st) {
  if constexpr (BWD) {
    a.blocks_q = (uint32_t)nq;
    if (pieces)
      hipLaunchKernelGGL((k_rope<T, NORM, IL, BWD, UNR_B>), dim3((unsigned)(nq + nk)), dim3(THREADS), 0, st, a);
    else
      hipLaunchKernelGGL((k_rope_any<T, NORM, IL, BWD>), dim3((unsigned)(nq + nk)), dim3(THREADS), 0, st, a);
  } else {
    // lanes per head vector or per UNR_F of them; a launch holds fewer than 2^32 threads, the kernels stride over the rest
    auto blocks = [&](int64_t H) {
      const int64_t threads = pieces ? a.tokens * ((H + UNR_F - 1) / UNR_F) * a.G : a.tokens * H * 64;
      const int64_t n = (threads + THREADS - 1) / THREADS;
      return (uint32_t)(n < MAX_BLOCKS_F ? n : MAX_BLOCKS_F);
    };
    a.blocks_q = blocks(a.side[0].H);
    const dim3 grid(a.blocks_q + blocks(a.side[1].H));
    if (pieces) hipLaunchKernelGGL((k_rope<T, NORM, IL, BWD, UNR_F>), grid, dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((k_rope_any<T, NORM, IL, BWD>), grid, dim3(THREADS), 0, st, a);
  }
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
  const int64_t n = dtype == MCE_ROPE_F32 ? 4 : 8;
  const bool pieces = whole_layout(D, R, n, interleaved, cos, sin, qw, kw) && whole_pieces(q, q_sb, q_st, q_sh, n) &&
                      whole_pieces(k, k_sb, k_st, k_sh, n) && whole_pieces(q_out, 0, 0, 0, n) &&
                      whole_pieces(k_out, 0, 0, 0, n);
  a.G = group_of(D, R, n, interleaved);
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
    const int64_t n = dtype == MCE_ROPE_F32 ? 4 : 8;
    const bool pieces = whole_layout(D, R, n, interleaved, cos, sin, qw, kw) && whole_pieces(q, q_sb, q_st, q_sh, n) &&
                        whole_pieces(k, k_sb, k_st, k_sh, n) && whole_pieces(gq, gq_sb, gq_st, gq_sh, n) &&
                        whole_pieces(gk, gk_sb, gk_st, gk_sh, n) && whole_pieces(dq, 0, 0, 0, n) &&
                        whole_pieces(dk, 0, 0, 0, n);
    a.G = group_of(D, R, n, interleaved);
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
