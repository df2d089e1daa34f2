// cache_attn.hip — attention of one new token per sequence over a paged cache of e4m3 codes, for MI355X (gfx950). The C ABI
// is in include/mce_cache.h.
//
// Every code that a sequence sees is read once, straight into the registers of the lanes that feed it to the matrix core,
// converted there (exactly) and used for the query heads that share it: the pass is bound by HBM and by the bytes in
// flight. Products are v_mfma_f32_16x16x32 with 16 query heads as columns, over tiles of 32 keys per wave:
//   scores  rows are keys: lane l loads the key 8 ((l%16)/4) + 4 k + (l%16)%4 of the k-th product, 16 bytes at 16 (l/16)
//           of every 64. The summed index is the same permutation of the head's columns for the query fragments. Lane l's
//           results are then the keys 8 (l/16) + 0..7 under the query head l%16: 8 neighbouring tokens, which lie in one
//           page and share one scale.
//   values  rows are columns of the head: lane l loads DP/16 neighbouring columns of the same 8 keys, so that exp(score)
//           is the other operand where it is; bytes of two keys are put side by side (one permutation per 4 bytes) and
//           converted in pairs. Product i gives the columns (DP/16) row + i.
// No value crosses lanes or goes through LDS in the loop. A value's scale goes into its probability's exponent:
// w_j = exp(s_j) scale_j is what multiplies the codes, and the denominator adds up w_j / scale_j.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_cache.h"
#include "attn_tile.h"
#include "cache_host.h"
#include "seq_find.h"

namespace {

using namespace attn;

constexpr int BK = 32;             // keys per tile of a wave
constexpr int HC = 16;             // query heads per column block
constexpr int NW = 4;              // waves per workgroup
constexpr int THREADS = 64 * NW;
constexpr int MIN_TILES = 4 * NW;  // tiles below which a sequence is not split further
constexpr int TARGET = 1024;       // workgroups that fill the GPU
constexpr float LAZY = 8.f;        // growth of a maximum (log2) up to which its old value is kept

struct Args {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  Codes k, v;
  Paged g;
  const int32_t* lengths;
  uint16_t* out;
  float *part, *ml;        // parts of the sums [B Hq, S, D]; their maxima and denominators [B Hq, S, 2]
  int Hq, Hkv, grp, ng, D; // ng: workgroups that share a key/value head's query heads
  int page, max_pages, window, sinks, S;
  float scale;
};


template <typename T, bool HI>
__device__ __forceinline__ uint32_t from_codes(uint32_t w) {   // two codes as a pair of T, exactly
  if constexpr (__is_same(T, __bf16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
}

template <typename T>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// What a wave holds of a tile while its loads are under way. VW: dwords of a value row per lane.
template <int DP>
struct Tile {
  static constexpr int VW = DP / 64;
  u32x4 k[2][DP / 64];
  uint32_t v[8][VW];
  float ks, vs;
  bool ok;               // the lane's 8 tokens lie in a page, and one of them at least is seen
};

// CB: column blocks of 16 query heads per workgroup.
template <typename T, int DP, int CB>
__global__ __launch_bounds__(THREADS, DP * CB > 128 ? 1 : 2) void k_cache_attn(Args a) {
  constexpr int VB = DP / 16, VW = DP / 64;             // value columns per lane, their dwords
  __shared__ __attribute__((aligned(16))) float sums[NW][CB * HC][DP];
  __shared__ float stat[NW][2][CB * HC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, quad = lane >> 4;
  const int s = blockIdx.x % a.S, unit = blockIdx.x / a.S;
  const int gi = unit % a.ng, hk = unit / a.ng % a.Hkv, b = unit / a.ng / a.Hkv;
  const Seen<BK> sn(a, b);
  const int run = sn.run<NW>(a.S, MIN_TILES), t0 = s * run;
  int t1 = t0 + run;
  t1 = t1 < sn.tiles ? t1 : sn.tiles;
  if (t0 >= sn.tiles && a.S > 1) return;                // the joining launch does not read this part
  const int h0 = hk * a.grp + gi * CB * HC;             // first query head
  int heads = a.grp - gi * CB * HC;
  heads = heads < CB * HC ? heads : CB * HC;
  const Paged& g = a.g;
  // query fragments: column r16, the columns of the head that the lane's codes have
  u32x4 qf[CB][DP / 32];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks) {
      const int col = 64 * (ks / 2) + 16 * quad + 8 * (ks % 2), hd = cb * HC + r16;
      qf[cb][ks] = u32x4{};
      if (col < a.D && hd < heads)
        qf[cb][ks] = *reinterpret_cast<const u32x4*>(a.q + b * a.q_sb + (h0 + hd) * a.q_sh + col);
    }
  f32x4 acc[CB][VB] = {};
  float m[CB], l[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = -INFINITY;
    l[cb] = 0.f;
  }
  const float c = a.scale * LOG2E;
  const uint8_t* const kp = a.k.p + hk * a.k.sh + 16 * quad;
  const uint8_t* const vp = a.v.p + hk * a.v.sh + (r16 * VB < a.D ? r16 * VB : 0);
  const int32_t* const table = g.table + b * g.bt_sb;
  const int kg = r16 >> 2, kr = r16 & 3;                // the 8 tokens whose keys the lane loads, and its row of 4
  // the page (or -1) of the 8 tokens `grp8` of tile it: asked for one tile before their codes
  auto page_of = [&](int it, int grp8) {
    const int pos = sn.key0(it) + 8 * grp8;
    const bool want = it < t1 && pos < sn.n && (pos + 7 >= sn.lo || pos < a.sinks);
    int pg = -1;
    if (want) pg = table[Paged::div((uint32_t)pos >> 3, g.mpage)];
    return pg;
  };
  auto issue = [&](Tile<DP>& t, int it, int pk, int pv) {
    const int k0 = sn.key0(it);
    const uint32_t gk = (uint32_t)(k0 >> 3) + kg, gv = (uint32_t)(k0 >> 3) + quad;
    const uint32_t sk = gk * 8 - Paged::div(gk, g.mpage) * a.page, sv = gv * 8 - Paged::div(gv, g.mpage) * a.page;
    const bool okk = pk >= 0 && pk < g.pages;
    t.ok = pv >= 0 && pv < g.pages;
    // what is not seen is read from the first page instead, and not used
    const uint8_t* const kb = kp + (okk ? (int64_t)pk * a.k.sp + (int64_t)(sk + kr) * a.k.st : 0);
    const uint8_t* const vb = vp + (t.ok ? (int64_t)pv * a.v.sp + (int64_t)sv * a.v.st : 0);
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
      const int o = 64 * i + 16 * quad < a.D ? 64 * i : -16 * quad;
      t.k[0][i] = *reinterpret_cast<const u32x4*>(kb + o);
      t.k[1][i] = *reinterpret_cast<const u32x4*>(kb + (okk ? 4 * a.k.st : 0) + o);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (VW == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(vb + j * a.v.st);
        t.v[j][0] = x[0];
        t.v[j][1] = x[1];
      } else {
        t.v[j][0] = *reinterpret_cast<const uint32_t*>(vb + j * a.v.st);
      }
    }
    const int64_t at = t.ok ? g.scale_at(pv, sv >> 3, hk) : 0;
    t.ks = a.k.scale[at];
    t.vs = a.v.scale[at];
  };
  auto use = [&](Tile<DP>& t, int it) {
    const int k0 = sn.key0(it);
    const int pos = k0 + 8 * quad;                      // the lane's first token
    const bool edge = __builtin_amdgcn_ballot_w64(!t.ok) != 0 || k0 + BK > sn.n || k0 < sn.lo;
    if (a.D < DP) {
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) {
        const bool in = 64 * i + 16 * quad < a.D;       // columns that the query has as zeros must not be NaN
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          t.k[0][i][e] = in ? t.k[0][i][e] : 0;
          t.k[1][i][e] = in ? t.k[1][i][e] : 0;
        }
      }
    }
    uint32_t see = 0xFF;
    if (edge) {
      see = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool y = t.ok && pos + j < sn.n && (pos + j >= sn.lo || pos + j < a.sinks);
        see |= y ? 1u << j : 0;
#pragma unroll
        for (int e = 0; e < VW; ++e) t.v[j][e] = y ? t.v[j][e] : 0;
      }
      t.ks = see ? t.ks : 1.f;
      t.vs = see ? t.vs : 1.f;
    }
    f32x4 sc[CB][2] = {};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int ks = 0; ks < DP / 32; ++ks) {
        u32x4 f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = t.k[kb][ks / 2][2 * (ks % 2) + e];
          f[2 * e] = from_codes<T, false>(w);
          f[2 * e + 1] = from_codes<T, true>(w);
        }
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) sc[cb][kb] = mfma16<T>(f, qf[cb][ks], sc[cb][kb]);
      }
    const float kc = t.ks * c, lv = __builtin_amdgcn_logf(t.vs), rv = __builtin_amdgcn_rcpf(t.vs);
    u32x4 pf[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float x[8], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_fmaf(sc[cb][e / 4][e % 4], kc, lv);
        if (edge) x[e] = (see >> e & 1) ? x[e] : -INFINITY;
        mx = fmaxf(mx, x[e]);
      }
      // the sums are rescaled only when some head's maximum has grown by more than LAZY since the last time
      if (__builtin_amdgcn_ballot_w64(mx - m[cb] > LAZY) != 0) {
        mx = fmaxf(mx, m[cb]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = max_halves(mx);
        const float al = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[cb] - mx);
        m[cb] = mx;
        l[cb] *= al;
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[cb][i] *= al;
      }
      const float mu = m[cb] == -INFINITY ? 0.f : m[cb];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_amdgcn_exp2f(x[e] - mu);
        sum += x[e];
      }
      l[cb] = __builtin_fmaf(sum, rv, l[cb]);
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[cb][e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    }
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {                  // bytes 2 hf and 2 hf + 1 of each dword
        u32x4 f[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t p = __builtin_amdgcn_perm(t.v[2 * j + 1][w], t.v[2 * j][w], hf ? 0x07030602u : 0x05010400u);
          f[0][j] = from_codes<T, false>(p);
          f[1][j] = from_codes<T, true>(p);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            const int i = 4 * w + 2 * hf + y;
            acc[cb][i] = mfma16<T>(f[y], pf[cb], acc[cb][i]);
          }
      }
  };
  Tile<DP> ta, tb;
  int it = t0 + wave;
  if (it < t1) {
    int pk = page_of(it, kg), pv = page_of(it, quad);
    issue(ta, it, pk, pv);
    pk = page_of(it + NW, kg);
    pv = page_of(it + NW, quad);
    while (true) {
      if (it + NW >= t1) {
        use(ta, it);
        break;
      }
      issue(tb, it + NW, pk, pv);
      pk = page_of(it + 2 * NW, kg);
      pv = page_of(it + 2 * NW, quad);
      __builtin_amdgcn_sched_barrier(0);
      use(ta, it);
      it += NW;
      if (it + NW >= t1) {
        use(tb, it);
        break;
      }
      issue(ta, it + NW, pk, pv);
      pk = page_of(it + 2 * NW, kg);
      pv = page_of(it + 2 * NW, quad);
      __builtin_amdgcn_sched_barrier(0);
      use(tb, it);
      it += NW;
    }
  }
  // join the waves: each leaves its sums [head][D] and its state
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    l[cb] += __shfl_xor(l[cb], 16);
    l[cb] = sum_halves(l[cb]);
    if (quad == 0) {
      stat[wave][0][cb * HC + r16] = m[cb];
      stat[wave][1][cb * HC + r16] = l[cb];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i4 = 0; i4 < VB; i4 += 4) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[cb][i4 + i][e];
        *reinterpret_cast<f32x4*>(&sums[wave][cb * HC + r16][(4 * quad + e) * VB + i4]) = x;
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (DP / 4); i += THREADS) {
    const int hd = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= a.D) continue;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, stat[w][0][hd]);
    const float mu = mm == -INFINITY ? 0.f : mm;
    f32x4 o = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(stat[w][0][hd] - mu);
      ll = __builtin_fmaf(stat[w][1][hd], f, ll);
      o += *reinterpret_cast<const f32x4*>(&sums[w][hd][d]) * f;
    }
    const int64_t row = (int64_t)b * a.Hq + h0 + hd;
    if (a.S == 1) {
      const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);   // nothing seen: 0; NaN stays
      u32x2 w;
      w[0] = pack2<T>(o[0] * inv, o[1] * inv);
      w[1] = pack2<T>(o[2] * inv, o[3] * inv);
      *reinterpret_cast<u32x2*>(a.out + row * a.D + d) = w;
    } else {
      *reinterpret_cast<f32x4*>(a.part + (row * a.S + s) * a.D + d) = o;
      if (d == 0) {
        a.ml[(row * a.S + s) * 2] = mm;
        a.ml[(row * a.S + s) * 2 + 1] = ll;
      }
    }
  }
}

// out = the parts of one query head joined: one wave per head, 2 columns per lane. The parts' states are read by all
// lanes at once and their factors shared through LDS, so that the sums' loads depend on nothing.
template <typename T>
__global__ __launch_bounds__(64) void k_cache_join(Args a) {
  __shared__ float f[TARGET];
  const int64_t row = blockIdx.x;
  const Seen<BK> sn(a, (int)(row / a.Hq));
  const int run = sn.run<NW>(a.S, MIN_TILES), n = (sn.tiles + run - 1) / run, lane = threadIdx.x, d = lane * 2;
  const float* const ml = a.ml + row * a.S * 2;
  float mm = -INFINITY;
  for (int s = lane; s < n; s += 64) mm = fmaxf(mm, ml[2 * s]);
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
  const float mu = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  for (int s = lane; s < n; s += 64) {
    f[s] = __builtin_amdgcn_exp2f(ml[2 * s] - mu);
    ll = __builtin_fmaf(ml[2 * s + 1], f[s], ll);
  }
  for (int o = 32; o > 0; o >>= 1) ll += __shfl_xor(ll, o);
  __syncthreads();
  if (d < a.D) {
    const float* const p = a.part + row * a.S * a.D + d;
    float x = 0.f, y = 0.f;
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float2 v = *reinterpret_cast<const float2*>(p + (int64_t)s * a.D);
      x = __builtin_fmaf(v.x, f[s], x);
      y = __builtin_fmaf(v.y, f[s], y);
    }
    const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);   // nothing seen: 0; NaN stays
    *reinterpret_cast<uint32_t*>(a.out + row * a.D + d) = pack2<T>(x * inv, y * inv);
  }
}

// --------------------------------------------------------------------------------------------------------- host side

int64_t heads_of(int64_t grp) { return grp <= HC ? HC : 2 * HC; }

// Workgroups per key/value head of a sequence.
int64_t splits(int64_t B, int64_t Hq, int64_t Hkv, int64_t page, int64_t max_pages, int64_t window, int64_t sinks) {
  int64_t n = page * max_pages;
  if (window > 0 && window + sinks < n) n = window + sinks;
  const int64_t grp = Hq / Hkv, tiles = (n + BK - 1) / BK + 2, units = B * Hkv * ((grp + heads_of(grp) - 1) / heads_of(grp));
  if (units >= TARGET / 2) return 1;
  int64_t s = (TARGET + units - 1) / units;
  const int64_t most = (tiles + MIN_TILES - 1) / MIN_TILES;
  s = s < most ? s : most;
  return s < 1 ? 1 : s;
}

int check_attn(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages, int64_t window,
               int64_t sinks) {
  const int rc = check_paged_sizes(B, Hkv, D, 0, page, 8, max_pages, 0);
  if (rc) return rc;
  if (Hq < 1 || Hq > 65536 || Hq % Hkv || window < 0 || sinks < 0 || B * Hq > MAX_GROUPS) return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

size_t ws_bytes_of(int64_t B, int64_t Hq, int64_t D, int64_t S) {
  return S == 1 ? 0 : (size_t)(align256(B * Hq * S * D * 4) + align256(B * Hq * S * 8));
}

template <typename T, int DP>
int launch(const Args& a, int64_t B, hipStream_t st) {
  const dim3 grid((unsigned)(B * a.Hkv * a.ng * a.S)), threads(THREADS);
  if (a.grp <= HC) hipLaunchKernelGGL((k_cache_attn<T, DP, 1>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((k_cache_attn<T, DP, 2>), grid, threads, 0, st, a);
  if (a.S > 1) hipLaunchKernelGGL((k_cache_join<T>), dim3((unsigned)(B * a.Hq)), dim3(64), 0, st, a);
  return finish();
}

}  // namespace

extern "C" {

size_t mce_cache_attn_ws_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages,
                               int64_t window, int64_t sinks) {
  if (check_attn(B, Hq, Hkv, D, page, max_pages, window, sinks) || B == 0) return 0;
  return ws_bytes_of(B, Hq, D, splits(B, Hq, Hkv, page, max_pages, window, sinks));
}

int mce_cache_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* kc, int64_t kc_sp, int64_t kc_st,
                   int64_t kc_sh, const void* vc, int64_t vc_sp, int64_t vc_st, int64_t vc_sh, const float* k_scale,
                   const float* v_scale, const int32_t* block_table, int64_t bt_sb, const int32_t* lengths, int64_t B,
                   int64_t Hq, int64_t Hkv, int64_t D, int64_t pages, int64_t page, int64_t block, int64_t max_pages,
                   int64_t window, int64_t sinks, float scale, int dtype, void* out, void* ws, size_t ws_bytes,
                   void* stream) {
  int rc = check_attn(B, Hq, Hkv, D, page, max_pages, window, sinks);
  if (rc || (rc = check_paged_sizes(B, Hkv, D, pages, page, block, max_pages, bt_sb))) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16)) return MCE_ATTN_EINVAL;
  if (B == 0) return MCE_ATTN_OK;
  if (out == nullptr || lengths == nullptr || (block_table == nullptr && max_pages > 0)) return MCE_ATTN_EINVAL;
  if ((rc = check_strided(q, q_sb, q_sh, 0, D))) return rc;
  if (pages > 0 && ((rc = check_codes(kc, kc_sp, kc_st, kc_sh, k_scale, D)) ||
                    (rc = check_codes(vc, vc_sp, vc_st, vc_sh, v_scale, D))))
    return rc;
  if (reinterpret_cast<uintptr_t>(out) & 15) return MCE_ATTN_EALIGN;
  const int64_t S = splits(B, Hq, Hkv, page, max_pages, window, sinks), need = (int64_t)ws_bytes_of(B, Hq, D, S);
  if (need > 0 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < (size_t)need))
    return MCE_ATTN_EWORKSPACE;
  Args a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.k = {static_cast<uint8_t*>(const_cast<void*>(kc)), kc_sp, kc_st, kc_sh, const_cast<float*>(k_scale)};
  a.v = {static_cast<uint8_t*>(const_cast<void*>(vc)), vc_sp, vc_st, vc_sh, const_cast<float*>(v_scale)};
  a.g = make_paged(block_table, bt_sb, Hkv, D, pages, page, block, max_pages);
  a.lengths = lengths;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(static_cast<char*>(ws) + align256(B * Hq * S * D * 4));
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.ng = (int)((a.grp + heads_of(a.grp) - 1) / heads_of(a.grp));
  a.D = (int)D;
  a.page = (int)page;
  a.max_pages = a.g.max_pages;
  a.window = window == 0 || window > INT32_MAX ? INT32_MAX : (int)window;
  a.sinks = a.window == INT32_MAX ? 0 : (int)(sinks < (1 << 30) ? sinks : 1 << 30);
  a.S = (int)S;
  a.scale = scale;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch<__bf16, 64>(a, B, st) : launch<__bf16, 128>(a, B, st);
  return D <= 64 ? launch<_Float16, 64>(a, B, st) : launch<_Float16, 128>(a, B, st);
}

}  // extern "C"
