// paged.hip — attention of one new token per sequence over a paged key/value cache, for MI355X (gfx950). The C ABI is
// in include/mce_paged.h; tiles and fragments are in attn_tile.h.
//
// Every cached element that a sequence sees is read once and used for the few query heads that share it, so the pass is
// bound by HBM and by the bytes in flight. A workgroup takes one sequence's key/value head (with up to 32 query heads as
// the columns of the products) and a run of 32-key tiles; each of its waves walks its own tiles with its own softmax
// state and its own double-buffered LDS images, without barriers, so that the loads of one tile are under way while the
// previous one is used. The waves' states are joined through LDS at the end, the workgroups' through fp32 parts and a
// second launch. Measured (bf16, D = 128, bytes of the keys seen): 64 sequences of up to 8192 tokens, 138 us, 4.9 TB/s;
// 8 of up to 131072, 273 us, 5.6 TB/s (a large copy, half of it writes, reaches 4.9); one of 1000 tokens 9 us, latency. The
// joining launch takes 4 to 8.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_paged.h"
#include "attn_host.h"
#include "attn_tile.h"
#include "seq_find.h"

namespace {

using namespace attn;

constexpr int NW = 4;              // waves per workgroup
constexpr int THREADS = 64 * NW;
constexpr int BK = 32;             // keys per tile of a wave
constexpr int HC = 32;             // query heads per workgroup: the columns of the products
constexpr int MIN_TILES = 2 * NW;  // tiles below which a sequence is not split further
constexpr int TARGET = 1024;       // workgroups that fill the GPU, some of them with shorter sequences

struct Args {
  const uint16_t *q, *k, *v;
  int64_t q_sb, q_sh, k_sp, k_st, k_sh, v_sp, v_st, v_sh, bt_sb;
  const int32_t *table, *lengths;
  uint16_t* out;
  float *part, *ml;        // parts of the sums [B Hq, S, D]; their maxima and denominators [B Hq, S, 2]
  int Hq, Hkv, grp, ng, D; // ng: workgroups that share a key/value head's query heads
  int pages, page, max_pages, window, sinks, S;
  uint32_t magic;          // of the division by page / 8 (0: page = 8)
  float scale;
};

template <typename T, int DP>
__global__ __launch_bounds__(THREADS, DP == 64 ? 2 : 1) void k_paged(Args a) {
  constexpr int IMG = BK * DP * 2, WAVE = 4 * IMG;     // a wave's LDS: K and V, two tiles each
  constexpr int RPI = 1024 / (DP * 2), NI = BK / RPI;  // rows per load instruction, instructions per image
  __shared__ __attribute__((aligned(1024))) char lds[NW * WAVE];
  __shared__ float stat[NW][2][HC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int s = blockIdx.x % a.S, unit = blockIdx.x / a.S;
  const int gi = unit % a.ng, hk = unit / a.ng % a.Hkv, b = unit / a.ng / a.Hkv;
  const Seen<BK> sn(a, b);
  const int run = sn.run<NW>(a.S, MIN_TILES), t0 = s * run;
  int t1 = t0 + run;
  t1 = t1 < sn.tiles ? t1 : sn.tiles;
  if (t0 >= sn.tiles && a.S > 1) return;               // the joining launch does not read this part
  const int h0 = hk * a.grp + gi * HC;                 // first query head
  int heads = a.grp - gi * HC;
  heads = heads < HC ? heads : HC;
  const int img = wave * WAVE;
  FragAddr<DP> ad;
  ad.init(lane);
  int ko[NI], vo[NI], kr[NI];                          // offsets in a group of 8 rows, and the tile's row
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int row = j * RPI + lane / (DP / 8), c = (lane % (DP / 8)) ^ swz<DP>(row);
    kr[j] = row;
    ko[j] = c * 8 < a.D ? (row & 7) * (int)a.k_st * 2 + c * 16 : OOB;
    vo[j] = c * 8 < a.D ? (row & 7) * (int)a.v_st * 2 + c * 16 : OOB;
  }
  u32x4 qf[DP / 16];
  const i32x4 qr = make_rsrc(a.q + b * a.q_sb + h0 * a.q_sh, (int)((heads - 1) * a.q_sh + a.D) * 2);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int col = 16 * ks + 8 * h;
    qf[ks] = load16(qr, col < a.D && (lane & 31) < heads ? (lane & 31) * (int)a.q_sh * 2 + col * 2 : OOB);
  }
  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * LOG2E;
  const uint16_t* const kp = a.k + hk * a.k_sh;
  const uint16_t* const vp = a.v + hk * a.v_sh;
  // lane i holds the page (or -1) and slot of 8-row group i % 4 of the wave's tile i / 4 of the next 16
  int pid = -1, slot = 0;
  auto look_up = [&](int it) {
    const int ti = it + (lane >> 2) * NW;
    pid = -1;
    if (ti < t1) {
      const uint32_t g8 = (uint32_t)(sn.key0(ti) >> 3) + (lane & 3);
      const uint32_t pg = a.magic ? __umulhi(g8, a.magic) : g8;
      slot = (int)(g8 * 8 - pg * a.page);
      if ((int)g8 * 8 < sn.n) pid = a.table[b * a.bt_sb + pg];
      if (pid < 0 || pid >= a.pages) pid = -1;
    }
  };
  // issues the loads of tile `it`, the wave's i-th; returns which of its 4 groups are in a page
  auto issue = [&](int it, int i) {
    const int buf = img + (i & 1) * 2 * IMG, k0 = sn.key0(it);
    const bool edge = k0 < sn.lo;                      // some rows lie before the window: those are not read
    int good = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int p = __builtin_amdgcn_readlane(pid, (i & 15) * 4 + g), sl = __builtin_amdgcn_readlane(slot, (i & 15) * 4 + g);
      good |= (p >= 0) << g;
      int left = sn.n - (k0 + 8 * g);
      left = left > 8 ? 8 : left;
      const bool any = p >= 0 && left > 0;
      const i32x4 rk = make_rsrc(kp + (int64_t)(any ? p : 0) * a.k_sp + (any ? sl : 0) * a.k_st,
                                 any ? (int)((left - 1) * a.k_st + a.D) * 2 : 0);
      const i32x4 rv = make_rsrc(vp + (int64_t)(any ? p : 0) * a.v_sp + (any ? sl : 0) * a.v_st,
                                 any ? (int)((left - 1) * a.v_st + a.D) * 2 : 0);
#pragma unroll
      for (int j = g * NI / 4; j < (g + 1) * NI / 4; ++j) {
        const bool cut = edge && k0 + kr[j] < sn.lo && k0 + kr[j] >= a.sinks;
        dma16(rk, lds, buf + j * 1024, cut ? OOB : ko[j]);
        dma16(rv, lds, buf + IMG + j * 1024, cut ? OOB : vo[j]);
      }
    }
    return good;
  };
  int good = 0;
  const bool work = t0 + wave < t1;
  if (work) look_up(t0 + wave);
  // The query fragments are here before the first tile's loads go out: a wait for them that the compiler put among the
  // loop's products would be a wait for the next tile too, as loads return in order.
  wait_vmcnt<0>();
  if (work) good = issue(t0 + wave, 0);
  for (int it = t0 + wave, i = 0; it < t1; it += NW, ++i) {
    int next = 0;
    if (it + NW < t1) {
      if ((i & 15) == 15) look_up(it + NW);
      next = issue(it + NW, i + 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int buf = img + (i & 1) * 2 * IMG, k0 = sn.key0(it);
    f32x16 sc = {};
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) sc = mfma<T>(frag_rows<DP>(lds, ad, buf, 0, ks), qf[ks], sc);
    if (good != 15 || k0 < sn.lo || k0 + BK > sn.n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = k0 + 8 * (e / 4) + 4 * h + e % 4;
        const bool see = ((good >> (e / 4)) & 1) && j < sn.n && (j >= sn.lo || j < a.sinks);
        sc[e] = see ? sc[e] : -INFINITY;
      }
    }
    float mx = m;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
    mx = max_halves(mx);
    const float mu = mx == -INFINITY ? 0.f : mx, al = __builtin_amdgcn_exp2f((m - mu) * c);
    float mc = mu * c;
    m = mx;
    l *= al;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= al;
    if (__builtin_amdgcn_ballot_w64(fabsf(mc) > LARGE) != 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] -= mu;
      mc = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      sc[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -mc));
      l += sc[e];
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const u32x4 pf = frag_acc<T>(sc, kk);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = mfma<T>(frag_tr<DP>(lds, ad, buf + IMG, dt, kk), pf, acc[dt]);
    }
    good = next;
    // the images just read are loaded into next: every read has returned
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // join the waves: each leaves its sums [head][D] and its state
  l = sum_halves(l);
  float* const mine = reinterpret_cast<float*>(lds + img);   // 32 heads x DP floats: as large as the wave's images
  __syncthreads();
  if (h == 0) {
    stat[wave][0][lane] = m;
    stat[wave][1][lane] = l;
  }
  if ((lane & 31) < heads) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[dt][4 * e4 + e];
        *reinterpret_cast<f32x4*>(mine + (lane & 31) * DP + 32 * dt + 8 * e4 + 4 * h) = x;
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
      const float f = __builtin_amdgcn_exp2f((stat[w][0][hd] - mu) * c);
      ll = __builtin_fmaf(stat[w][1][hd], f, ll);
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * WAVE) + hd * DP + d) * f;
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
__global__ __launch_bounds__(64) void k_paged_join(Args a) {
  __shared__ float f[TARGET];
  const int64_t row = blockIdx.x;
  const Seen<BK> sn(a, (int)(row / a.Hq));
  const int run = sn.run<NW>(a.S, MIN_TILES), n = (sn.tiles + run - 1) / run, lane = threadIdx.x, d = lane * 2;
  const float c = a.scale * LOG2E;
  const float* const ml = a.ml + row * a.S * 2;
  float mm = -INFINITY;
  for (int s = lane; s < n; s += 64) mm = fmaxf(mm, ml[2 * s]);
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
  const float mu = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  for (int s = lane; s < n; s += 64) {
    f[s] = __builtin_amdgcn_exp2f((ml[2 * s] - mu) * c);
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

// -------------------------------------------------------------------------------------------------------- host side

// Workgroups per key/value head of a sequence. From 512 heads on one each: they fill the GPU, and the second launch and the
// parts cost more than even rounds gain (96 sequences of 8 heads of 64, window 1024: 38.7 us against 43.8 with two each). Long
// caches are the other way round (64 of 8 heads of 128, up to 8192 keys: 285 us against 265): the line lies where windows
// want it. With fewer heads, TARGET in all (256 heads of 128, up to 8192 keys: 148, 143 and 144 us with 2, 4 and 8 each; 32
// heads, up to 131072 keys: 293, 277 and 272 us with 16, 32 and 64), at most one per MIN_TILES tiles of the longest sequence
// that the table can hold (twice as many: the calls above as they are, one head with 131072 keys 31 us instead of 47).
int64_t splits(int64_t B, int64_t Hq, int64_t Hkv, int64_t page, int64_t max_pages, int64_t window, int64_t sinks) {
  int64_t n = page * max_pages;
  if (window > 0 && window + sinks < n) n = window + sinks;
  const int64_t tiles = (n + BK - 1) / BK + 2, units = B * Hkv * ((Hq / Hkv + HC - 1) / HC);
  if (units >= TARGET / 2) return 1;
  int64_t s = (TARGET + units - 1) / units;
  const int64_t most = (tiles + MIN_TILES - 1) / MIN_TILES;
  s = s < most ? s : most;
  return s < 1 ? 1 : s;
}

int check_paged(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages, int64_t window,
                int64_t sinks) {
  if (B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 8 || D > 128 || D % 8 || page < 8 || page % 8 || page > 65536 ||
      max_pages < 0 || window < 0 || sinks < 0 || Hq > 65536 || B > (int64_t(1) << 24) || B * Hq > (int64_t(1) << 24))
    return MCE_ATTN_EINVAL;
  if (B * Hkv * ((Hq / Hkv + HC - 1) / HC) > MAX_GROUPS) return MCE_ATTN_EINVAL;
  // key numbers in 30 bits, and exact division of an 8-row group's number by page / 8 through a 32-bit product
  if (max_pages > (int64_t(1) << 30) / page || max_pages * page > (int64_t(1) << 38) / page) return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

size_t ws_bytes_of(int64_t B, int64_t Hq, int64_t D, int64_t S) {
  return S == 1 ? 0 : (size_t)(align256(B * Hq * S * D * 4) + align256(B * Hq * S * 8));
}

template <typename T, int DP>
int launch(const Args& a, int64_t B, hipStream_t st) {
  const unsigned n = (unsigned)(B * a.Hkv * a.ng * a.S);
  hipLaunchKernelGGL((k_paged<T, DP>), dim3(n), dim3(THREADS), 0, st, a);
  if (a.S > 1) hipLaunchKernelGGL((k_paged_join<T>), dim3((unsigned)(B * a.Hq)), dim3(64), 0, st, a);
  return finish();
}

}  // namespace

extern "C" {

size_t mce_paged_ws_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages,
                          int64_t window, int64_t sinks) {
  if (check_paged(B, Hq, Hkv, D, page, max_pages, window, sinks) || B == 0) return 0;
  return ws_bytes_of(B, Hq, D, splits(B, Hq, Hkv, page, max_pages, window, sinks));
}

int mce_paged(const void* q, int64_t q_sb, int64_t q_sh, const void* k, int64_t k_sp, int64_t k_st, int64_t k_sh,
              const void* v, int64_t v_sp, int64_t v_st, int64_t v_sh, const int32_t* block_table, int64_t bt_sb,
              const int32_t* lengths, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t pages, int64_t page,
              int64_t max_pages, int64_t window, int64_t sinks, float scale, int dtype, void* out, void* ws,
              size_t ws_bytes, void* stream) {
  int rc = check_paged(B, Hq, Hkv, D, page, max_pages, window, sinks);
  if (rc) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16) || pages < 0 || pages > INT32_MAX ||
      bt_sb < 0)
    return MCE_ATTN_EINVAL;
  if (B == 0) return MCE_ATTN_OK;
  if (out == nullptr || lengths == nullptr || (block_table == nullptr && max_pages > 0)) return MCE_ATTN_EINVAL;
  if ((rc = check_strided(q, q_sb, q_sh, 0, D))) return rc;
  if (pages > 0 && ((rc = check_strided(k, k_sp, k_st, k_sh, D)) || (rc = check_strided(v, v_sp, v_st, v_sh, D))))
    return rc;
  if (reinterpret_cast<uintptr_t>(out) & 15) return MCE_ATTN_EALIGN;
  const int64_t S = splits(B, Hq, Hkv, page, max_pages, window, sinks), need = (int64_t)ws_bytes_of(B, Hq, D, S);
  if (need > 0 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < (size_t)need))
    return MCE_ATTN_EWORKSPACE;
  Args a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.k_sp = k_sp;
  a.k_st = k_st;
  a.k_sh = k_sh;
  a.v_sp = v_sp;
  a.v_st = v_st;
  a.v_sh = v_sh;
  a.table = block_table;
  a.bt_sb = bt_sb;
  a.lengths = lengths;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(static_cast<char*>(ws) + align256(B * Hq * S * D * 4));
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.ng = (a.grp + HC - 1) / HC;
  a.D = (int)D;
  a.pages = (int)pages;
  a.page = (int)page;
  a.max_pages = (int)max_pages;
  a.window = window == 0 || window > INT32_MAX ? INT32_MAX : (int)window;
  a.sinks = a.window == INT32_MAX ? 0 : (int)(sinks < (1 << 30) ? sinks : 1 << 30);
  a.S = (int)S;
  a.magic = page == 8 ? 0 : (uint32_t)((uint64_t(1) << 32) / (uint64_t)(page / 8) + 1);
  a.scale = scale;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch<__bf16, 64>(a, B, st) : launch<__bf16, 128>(a, B, st);
  return D <= 64 ? launch<_Float16, 64>(a, B, st) : launch<_Float16, 128>(a, B, st);
}

}  // extern "C"
