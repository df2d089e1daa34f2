// attn.hip — causal attention over a sliding window with first tokens that stay visible, forward and backward, for
// MI355X (gfx950). The C ABI is in include/mce_attn.h; tiles and fragments are in attn_tile.h.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_attn.h"
#include "attn_host.h"
#include "attn_tile.h"

namespace {

using namespace attn;

constexpr int NW = 4;               // waves per workgroup
constexpr int THREADS = 64 * NW;
constexpr int BQ = 32 * NW;         // query rows per workgroup of k_attn_fwd and k_attn_dq (32 per wave)
constexpr int BK = 64;              // keys per tile there
constexpr int BKV = 32 * NW;        // keys per workgroup of k_attn_dkv (32 per wave)
constexpr int BR = 32;              // query rows per tile there
constexpr int NS = 4;               // tiles of k_attn_dkv's ring

constexpr float LAZY = 8.f;         // k_attn_fwd: growth of a maximum (log2) up to which its old value is kept

struct Strided {
  const uint16_t* p;
  int64_t sb, st, sh;  // elements between batches, tokens, heads
};

struct Args {
  Strided q, k, v, go;
  const uint16_t *out, *res; // contiguous [B, T, Hq, D], backward
  uint16_t *o, *r, *dq, *dk, *dv;
  float* lse;                // [B, Hq, T]
  float* stat;               // [B, Hq, 2, T]: -lse and -delta, what the backward's scores and products start from
  const int32_t* lengths;
  int B, T, Hq, Hkv, grp, D;
  int window, sinks;         // window = INT32_MAX: none
  float scale;
  // k_attn_dkv: the first n_sb key blocks (those with first tokens) are shared by S_s workgroups each, the others by S_r
  int n_sb, S_s, S_r;
  float *part_s, *part_r;    // their fp32 parts [B Hkv, block, S, 2, BKV, D] where S > 1
};

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  if (a.lengths == nullptr) return a.T;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// The key tiles that rows q0 .. q1 (inclusive) see: those of the first `sinks` positions (n_sink tiles from 0) and then
// those from tile `lo` to tile `hi`.
struct KeyTiles {
  int n_sink, lo, n;
  __device__ __forceinline__ KeyTiles(const Args& a, int q0, int q1) {
    const int first = q0 - a.window + 1;   // first key of the window of row q0
    lo = first <= 0 ? 0 : first / BK;
    n_sink = (a.sinks + BK - 1) / BK;
    n_sink = n_sink < lo ? n_sink : lo;
    n = n_sink + q1 / BK - lo + 1;
  }
  __device__ __forceinline__ int key0(int it) const { return (it < n_sink ? it : lo + it - n_sink) * BK; }
  // keys that are read of the tile's: of those before the window the first tokens only, so that what lies behind them (a
  // NaN, say) meets no row that is far from it
  __device__ __forceinline__ int end(int it, const Args& a, int len) const {
    return it < n_sink && a.sinks < len ? a.sinks : len;
  }
};

// Which sequence, heads and block of rows (or keys) a workgroup takes. Workgroups go to the 8 XCDs in turn, each with an
// L2 of its own: where the key/value heads (or the query heads) of the batch are a multiple of 8, each XCD takes whole
// ones. Blocks of one length (a window) run head by head, the query heads of a group side by side on the same keys;
// without a window the longest blocks of all the XCD's heads run first, so that none is left over at the end.
struct Place {
  int b, hk, g, blk;   // sequence, key/value head, query head of its group, block (0: the longest without a window)
  // n: blocks per head; sub: query heads of a group that are workgroups of their own (grp, or 1)
  __device__ __forceinline__ Place(const Args& a, uint32_t bid, uint32_t n, uint32_t sub) {
    const uint32_t kv = (uint32_t)a.B * a.Hkv;
    const bool whole = kv % 8 == 0, heads = !whole && kv * sub % 8 == 0;
    const uint32_t units = heads ? kv * sub : kv, in = heads ? 1 : sub;   // units per XCD set, workgroups inside a unit
    const uint32_t x = whole || heads ? 8 : 1, xcd = bid % x, slot = bid / x, ux = units / x;
    uint32_t u, i;
    if (a.window == INT32_MAX) {
      blk = slot / (ux * in);
      const uint32_t r = slot - blk * (ux * in);
      u = r / in;
      i = r - u * in;
    } else {
      u = slot / (n * in);
      const uint32_t r = slot - u * (n * in);
      blk = r / in;
      i = r - blk * in;
    }
    u = u * x + xcd;
    const uint32_t k = heads ? u / sub : u;
    g = heads ? u - k * sub : i;
    b = k / a.Hkv;
    hk = k - b * a.Hkv;
  }
};

// Whether rows r0 .. r0 + 31 see one of the 32 keys from k0 on.
__device__ __forceinline__ bool some_keys(const Args& a, int r0, int k0) {
  return k0 <= r0 + 31 && (r0 - (k0 + 31) < a.window || k0 < a.sinks);
}

// Masks a 32 x 32 block of scores held as [keys][rows]: accumulator element e of lane l is key
// k0h + 8*(e/4) + e%4 (k0h = first key + 4*(l/32)) and row `row` (of lane l%32). Both forms are free of branches; the
// one without first tokens in the block is a compare and a select per element.
__device__ __forceinline__ void mask_keys(f32x16& s, int row, int k0h, int window, int sinks, bool with_sinks) {
  const int rel = row - k0h;
  if (with_sinks) {
    const int left = sinks - k0h;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int c = 8 * (e / 4) + e % 4;
      const bool see = ((uint32_t)(rel - c) < (uint32_t)window) | ((c < left) & (rel >= c));
      s[e] = see ? s[e] : -INFINITY;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int c = 8 * (e / 4) + e % 4;
      s[e] = (uint32_t)(rel - c) < (uint32_t)window ? s[e] : -INFINITY;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- forward
// out_i = sum_j exp(c s_ij - c m_i) v_j / sum_j exp(c s_ij - c m_i) in one pass over the keys, m_i a maximum of the scores so far.
// 32 rows per wave hold their scores as [keys][rows], so that a row's statistics lie in two lanes and the scores become an
// operand of the second product where they are; 64 KiB of LDS let two workgroups share a CU, whose products and
// exponentials fill each other's gaps. p is rounded to the element type: the matrix core takes no other.
// Measured (bf16, D = 128, 16 heads): 32768 tokens, every earlier one seen, 4.1 ms, 1.06 PFLOP/s; 4 x 16384 tokens, window
// 1024, 0.75 ms, 0.72 PFLOP/s of visible pairs with the matrix core busy 40% of the time; 32 x 1024, window 512, 0.27 ms,
// 23% busy: its workgroups are 2 to 11 tiles long and 1.4 of 2 waves per SIMD are there at a time.
// With D <= 64 vector work is busy half the time and the matrix core a quarter, so waves are what fills the gaps: four per
// SIMD, in 128 registers with the tile's offsets made again for each tile, take 96 us where three take 102 (8 texts of up to
// 2999 tokens, 12 heads, fp16). At D = 128 the registers leave room for two.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, DP == 64 ? 4 : 2) void k_attn_fwd(Args a) {
  constexpr int IMG = BK * DP * 2;                     // bytes of a tile
  __shared__ __attribute__((aligned(1024))) char lds[4 * IMG];   // K and V, two tiles each
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int nq = (a.T + BQ - 1) / BQ;
  const Place pl(a, blockIdx.x, nq, a.grp);
  const int qb = nq - 1 - pl.blk, b = pl.b, hk = pl.hk, hq = hk * a.grp + pl.g, bh = b * a.Hq + hq;
  const int len = seq_len(a, b);
  const int q0 = qb * BQ, r0 = q0 + wave * 32, row = r0 + (lane & 31);
  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;
  bool large = false;   // some row's m is beyond LARGE
  const float c = a.scale * LOG2E;
  if (q0 < len) {
    const int q1 = (q0 + BQ < len ? q0 + BQ : len) - 1;
    const KeyTiles kt(a, q0, q1);
    FragAddr<DP> ad;
    ad.init(lane);
    TileLoad<DP, BK, NW> tk, tv;
    tk.init((int)a.k.st * 2, a.D, wave, lane);
    tv.init((int)a.v.st * 2, a.D, wave, lane);
    const uint16_t* const kp = a.k.p + b * a.k.sb + hk * a.k.sh;
    const uint16_t* const vp = a.v.p + b * a.v.sb + hk * a.v.sh;
    auto issue = [&](int it, int buf) {
      const int k0 = kt.key0(it), end = kt.end(it, a, len);
      tk.issue(tile_rsrc<BK>(kp, a.k.st, k0, end, a.D), lds, buf * 2 * IMG, wave);
      tv.issue(tile_rsrc<BK>(vp, a.v.st, k0, end, a.D), lds, buf * 2 * IMG + IMG, wave);
    };
    issue(0, 0);
    // the wave's query rows as fragments: row l%32, columns 16 ks + 8 h + 0..7
    u32x4 qf[DP / 16];
    const i32x4 qr = tile_rsrc<32>(a.q.p + b * a.q.sb + hq * a.q.sh, a.q.st, r0, len, a.D);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int col = 16 * ks + 8 * h;
      qf[ks] = load16(qr, col < a.D ? (lane & 31) * (int)a.q.st * 2 + col * 2 : OOB);
    }
    wait_vmcnt<0>();
    __syncthreads();
    for (int it = 0; it < kt.n; ++it) {
      const int img = (it & 1) * 2 * IMG;
      if (it + 1 < kt.n) issue(it + 1, (it + 1) & 1);
      const int k0 = kt.key0(it);
      if constexpr (DP == 64) ad.refresh();            // 128 registers: four waves per SIMD
      // whether the wave's rows see a key of the tile
      if (k0 <= r0 + 31 && (r0 - (k0 + BK - 1) < a.window || k0 < a.sinks)) {
        f32x16 s[2] = {};
        // the key fragments are read three column slices (6 products) ahead
        u32x4 kf[4][2];
#pragma unroll
        for (int ks = 0; ks < 3; ++ks)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) kf[ks][kb] = frag_rows<DP>(lds, ad, img, kb, ks);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            if (ks + 3 < DP / 16) kf[(ks + 3) & 3][kb] = frag_rows<DP>(lds, ad, img, kb, ks + 3);
            s[kb] = mfma<T>(kf[ks & 3][kb], qf[ks], s[kb]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        const bool all = k0 + BK - 1 <= r0 && r0 + 31 - k0 < a.window;
        if (!all) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            mask_keys(s[kb], row, k0 + 32 * kb + 4 * h, a.window, a.sinks, k0 < a.sinks);
        }
        float mx = m;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
        mx = max_halves(mx);
        // The sums are rescaled only when some row's maximum has grown by more than LAZY since the last time: until
        // then its exponentials stay below 2^LAZY.
        if (__builtin_amdgcn_ballot_w64((mx - m) * c > LAZY) != 0) {
          const float al = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mx) * c);
          m = mx;
          large = __builtin_amdgcn_ballot_w64(fabsf(m * c) > LARGE && m != -INFINITY) != 0;
          l *= al;
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= al;
        }
        const float mu = m == -INFINITY ? 0.f : m;   // (a row that has seen nothing yet)
        float mc = mu * c;
        if (large) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] -= mu;
          mc = 0.f;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[kb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], c, -mc));
            l += s[kb][e];
          }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const u32x4 pf = frag_acc<T>(s[kk >> 1], kk & 1);
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = mfma<T>(frag_tr<DP>(lds, ad, img + IMG, dt, kk), pf, acc[dt]);
        }
      }
      wait_vmcnt<0>();
      __syncthreads();
    }
  }
  l = sum_halves(l);
  const int64_t ofs = ((int64_t)b * a.T + row) * a.Hq * a.D + (int64_t)hq * a.D;
  const bool in = row < a.T, see = row < len;
  const float inv = 1.f / l;
  store_acc<T, DP>(acc, inv, a.o + ofs, a.D, in, see, h);
  if (a.r != nullptr) store_acc<T, DP, true>(acc, inv, a.r + ofs, a.D, in, see, h);
  if (a.lse != nullptr && in && h == 0) a.lse[(int64_t)bh * a.T + row] = see ? m + __builtin_amdgcn_logf(l) / c : INFINITY;
}

// --------------------------------------------------------------------------------------------------------------- dq
// Keeps the compiler from moving anything past it.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
// The lane's number, worked out anew wherever it is asked for (registers are scarce in the loops).
__device__ __forceinline__ int lane_now() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
}
// x, copied at this place (of 16 copies of one value the compiler would keep a set for the whole loop)
__device__ __forceinline__ float now(float x) {
  asm volatile("" : "+v"(x));
  return x;
}
// the s-th four of eight packed pairs, as a fragment
__device__ __forceinline__ u32x4 four(const uint32_t (&w)[8], int s) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = w[4 * s + e];
  return r;
}

// dq_i = scale sum_j ds_ij k_j, ds_ij = p_ij (go_i . v_j - d_i), p from the forward's lse: rows stay in registers and keys
// pass, as in the forward, so that dq is summed by one wave in one order. It also forms d and leaves -lse and -d for
// k_attn_dkv. Measured (bf16, D = 128): 4 x 16384 tokens of 16 heads, window 1024: 1.10 ms, 0.73 PFLOP/s of visible pairs
// (6 D each), matrix core busy 46% of the time.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, 2) void k_attn_dq(Args a) {
  constexpr int IMG = BK * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[4 * IMG];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nq = (a.T + BQ - 1) / BQ;
  const Place pl(a, blockIdx.x, nq, a.grp);
  const int qb = nq - 1 - pl.blk, b = pl.b, hk = pl.hk, hq = hk * a.grp + pl.g, bh = b * a.Hq + hq;
  const int len = seq_len(a, b);
  const int q0 = qb * BQ, r0 = q0 + wave * 32;
  f32x16 acc[DP / 32] = {};
  float delta = 0.f, nl = -INFINITY, sum = 0.f;
  const float c = a.scale * LOG2E;
  if (q0 < len) {
    const int q1 = (q0 + BQ < len ? q0 + BQ : len) - 1;
    const KeyTiles kt(a, q0, q1);
    const int lane = lane_now();
    FragAddr<DP> ad;
    ad.init(lane);
    TileLoad<DP, BK, NW> tk, tv;
    tk.init((int)a.k.st * 2, a.D, wave, lane);
    tv.init((int)a.v.st * 2, a.D, wave, lane);
    const uint16_t* const kp = a.k.p + b * a.k.sb + hk * a.k.sh;
    const uint16_t* const vp = a.v.p + b * a.v.sb + hk * a.v.sh;
    auto issue = [&](int it, int buf) {
      const int k0 = kt.key0(it), end = kt.end(it, a, len);
      tk.issue(tile_rsrc<BK>(kp, a.k.st, k0, end, a.D), lds, buf * 2 * IMG, wave);
      tv.issue(tile_rsrc<BK>(vp, a.v.st, k0, end, a.D), lds, buf * 2 * IMG + IMG, wave);
    };
    issue(0, 0);
    u32x4 qf[DP / 16], gf[DP / 16];
    const i32x4 qr = tile_rsrc<32>(a.q.p + b * a.q.sb + hq * a.q.sh, a.q.st, r0, len, a.D);
    const i32x4 gr = tile_rsrc<32>(a.go.p + b * a.go.sb + hq * a.go.sh, a.go.st, r0, len, a.D);
    const int64_t head = (int64_t)b * a.T * a.Hq * a.D + (int64_t)hq * a.D, ldo = (int64_t)a.Hq * a.D;
    const i32x4 orr = tile_rsrc<32>(a.out + head, ldo, r0, len, a.D), rr = tile_rsrc<32>(a.res + head, ldo, r0, len, a.D);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int col = 16 * ks + 8 * (lane >> 5), r = lane & 31;
      qf[ks] = load16(qr, col < a.D ? r * (int)a.q.st * 2 + col * 2 : OOB);
      gf[ks] = load16(gr, col < a.D ? r * (int)a.go.st * 2 + col * 2 : OOB);
      const int oo = col < a.D ? r * (int)ldo * 2 + col * 2 : OOB;
      const u32x4 of = load16(orr, oo), rf = load16(rr, oo);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        delta = __builtin_fmaf(lo_f32<T>(gf[ks][e]), lo_f32<T>(of[e]) + lo_f32<T>(rf[e]), delta);
        delta = __builtin_fmaf(hi_f32<T>(gf[ks][e]), hi_f32<T>(of[e]) + hi_f32<T>(rf[e]), delta);
      }
    }
    delta = sum_halves(delta);
    const int row = r0 + (lane & 31);
    if (row < len) nl = -a.lse[(int64_t)bh * a.T + row];
    wait_vmcnt<0>();
    __syncthreads();
    for (int it = 0; it < kt.n; ++it) {
      const int img = (it & 1) * 2 * IMG;
      if (it + 1 < kt.n) issue(it + 1, (it + 1) & 1);
      const int k0 = kt.key0(it);
      ad.refresh();
      // the halves of the tile (32 keys) that the wave's rows see a key of: first .. last - 1
      const bool see0 = some_keys(a, r0, k0), see1 = some_keys(a, r0, k0 + 32);
      const int first = see0 ? 0 : 1, last = see1 ? 2 : 1;
      if (see0 || see1) {
        // The products of a tile in one sequence, half (32 keys) after half: scores (KS), go v (KS), dq (2 DT). The fragment
        // of each is read PD - 1 steps ahead, and the exponentials stand between the products of go v. Rounding ds is what
        // dq loses most by; of every second slice of 16 keys what the rounding leaves over goes into dq as well. In units
        // of dq's own rounding it is off by 1.3 to 1.4 then, for 3% of a training step; by 1.5 without any of the rest, by
        // 1.1 to 1.2 with all of it, for 7%.
        constexpr int KS = DP / 16, DT = DP / 32, H = 2 * KS + 2 * DT, PD = 3;
        static_assert(H % PD == 0, "each half starts at the ring's first place");
        auto read = [&](int kb, int i) {
          const int rows = img + kb * 32 * DP * 2;
          if (i < 2 * KS) return frag_rows<DP>(lds, ad, rows + i / KS * IMG, 0, i % KS);
          i -= 2 * KS;
          return frag_tr<DP>(lds, ad, rows, i % DT, i / DT);
        };
        u32x4 f[PD];
#pragma unroll
        for (int i = 0; i < PD - 1; ++i) f[i] = read(first, i);
        fence();
        for (int kb = first; kb < last; ++kb) {
          // the half's i-th fragment; reads the one PD - 1 further (behind the last half: the last's again)
          auto step = [&](int i) {
            const u32x4 x = f[i % PD];
            const int at = i + PD - 1;
            f[at % PD] = at < H ? read(kb, at) : read(last - 1, at - H);
            return x;
          };
          const int kh = k0 + 32 * kb;
          f32x16 s, ds;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = now(nl);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            s = mfma<T>(step(i), qf[i], s);
            fence();
          }
          if (!(kh + 31 <= r0 && r0 + 31 - kh < a.window)) {
            const int ln = lane_now();
            mask_keys(s, r0 + (ln & 31), kh + 4 * (ln >> 5), a.window, a.sinks, kh < a.sinks);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) ds[e] = now(-delta);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            ds = mfma<T>(step(KS + i), gf[i], ds);
#pragma unroll
            for (int e = i * (16 / KS); e < (i + 1) * (16 / KS); ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * c);
            fence();
          }
          // ds of 16 keys as fragments
          u32x4 hi[2], lo;
          auto split = [&](int sl, int i) {
            const int e = 8 * sl + 2 * i;
            const float x = s[e] * ds[e], y = s[e + 1] * ds[e + 1];
            sum += x + y;
            const uint32_t w = pack2<T>(x, y);
            hi[sl][i] = w;
            if (sl == 0) lo[i] = pack2<T>(x - lo_f32<T>(w), y - hi_f32<T>(w));
          };
#pragma unroll
          for (int i = 0; i < 4; ++i) split(0, i);
#pragma unroll
          for (int i = 0; i < 2 * DT; ++i) {
            const int sl = i / DT, dt = i % DT;
            const u32x4 x = step(2 * KS + i);
            acc[dt] = mfma<T>(x, hi[sl], acc[dt]);
            if (sl == 0) acc[dt] = mfma<T>(x, lo, acc[dt]);
            if (sl == 0) {
#pragma unroll
              for (int e = dt * 4 / DT; e < (dt + 1) * 4 / DT; ++e) split(1, e);
            }
            fence();
          }
        }
      }
      wait_vmcnt<0>();
      __syncthreads();
    }
  }
  sum = sum_halves(sum);
  const int ln = lane_now(), h = ln >> 5, row = r0 + (ln & 31);
  const int64_t ofs = ((int64_t)b * a.T + row) * a.Hq * a.D + (int64_t)hq * a.D;
  const bool in = row < a.T;
  store_acc<T, DP>(acc, a.scale, a.dq + ofs, a.D, in, row < len, h);
  if (in && h == 0) {
    // The output's probabilities were rounded, so delta is off by some of its rounding, and the sum of the row's ds, which
    // should be 0, by as much: what k_attn_dkv gets is put right by it (dk of 8 heads of 96, T = 1000: off by 1.42 times
    // its own rounding instead of 1.51).
    float* const p = a.stat + (int64_t)bh * 2 * a.T + row;
    p[0] = nl;
    p[a.T] = row < len ? -(delta + sum) : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------------------- dk, dv
// dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij go_i over the rows of all query heads that share the head: keys stay in
// registers, 32 per wave, and row tiles pass through a ring of NS. Scores and go v are formed a second time (seven
// products in the backward for the formula's five), which needs neither atomics nor ds in memory.
// Measured (bf16, D = 128): 4 x 16384 tokens of 16 heads over 4, window 1024: 1.24 ms, 0.86 PFLOP/s of visible pairs (8 D
// each), matrix core busy 45% of the time; the join of the first tokens' blocks 7 us.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, 2) void k_attn_dkv(Args a) {
  constexpr int IMG = BR * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[NS * 2 * IMG];   // Q and go of the ring's tiles
  __shared__ __attribute__((aligned(256))) float stats[NS][2][BR];    // -lse and -delta of their rows
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nk = (a.T + BKV - 1) / BKV, nr = nk - a.n_sb;
  // workgroups of the blocks with first tokens (the longest) first, then the others, those with the most rows first
  const uint32_t heads = (uint32_t)a.B * a.Hkv, sink_wgs = heads * a.n_sb * a.S_s;
  const bool sink = blockIdx.x < sink_wgs;
  const uint32_t w = sink ? blockIdx.x : blockIdx.x - sink_wgs;
  const int S = sink ? a.S_s : a.S_r, nb = sink ? a.n_sb : nr;
  const Place pl(a, w, nb * S, 1);
  const int sp = pl.blk % S, blk = pl.blk / S, b = pl.b, hk = pl.hk, bh = b * a.Hkv + hk;
  const int kblk = sink ? blk : a.n_sb + blk;
  const int len = seq_len(a, b);
  const int kb0 = kblk * BKV, j0 = kb0 + wave * 32;
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const float c = a.scale * LOG2E;
  int it0 = 0, it1 = 0;
  if (kb0 < len) {
    // rows kb0 .. q_end - 1 may see a key of the block
    int64_t q_end64 = kb0 < a.sinks ? len : (int64_t)kb0 + BKV - 1 + a.window;
    const int q_end = q_end64 < len ? (int)q_end64 : len;
    const int t0 = kb0 / BR, nt = (q_end + BR - 1) / BR - t0, total = nt * a.grp;
    it0 = (int)((int64_t)total * sp / S);
    it1 = (int)((int64_t)total * (sp + 1) / S);
    const int lane = lane_now();
    FragAddr<DP> ad;
    ad.init(lane);
    TileLoad<DP, BR, NW> tq, tg;
    tq.init((int)a.q.st * 2, a.D, wave, lane);
    tg.init((int)a.go.st * 2, a.D, wave, lane);
    // -lse and -delta: lanes 0..31 and 32..63 of one 4-byte load (every wave issues it, with the same values, so that all
    // have the same number of loads under way). Rows past the text read zeros: their Q and go are zeros too.
    constexpr int LOADS = decltype(tq)::N + decltype(tg)::N + 1;
    auto issue = [&](int it) {
      const int g = it / nt, i0 = (t0 + it - g * nt) * BR, hq = hk * a.grp + g, buf = (it - it0) & (NS - 1);
      tq.issue(tile_rsrc<BR>(a.q.p + b * a.q.sb + hq * a.q.sh, a.q.st, i0, len, a.D), lds, buf * 2 * IMG, wave);
      tg.issue(tile_rsrc<BR>(a.go.p + b * a.go.sb + hq * a.go.sh, a.go.st, i0, len, a.D), lds, buf * 2 * IMG + IMG, wave);
      const int rows = a.T - i0 < BR ? a.T - i0 : BR;
      const int ln = lane_now();
      dma4(make_rsrc(a.stat + ((int64_t)b * a.Hq + hq) * 2 * a.T + i0, (a.T + rows) * 4),
           reinterpret_cast<const char*>(&stats[0][0][0]), buf * 2 * BR * 4,
           (ln & 31) < rows ? ((ln & 31) + (ln >> 5) * a.T) * 4 : OOB);
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
      if (it0 + i < it1) issue(it0 + i);
    u32x4 kf[DP / 16], vf[DP / 16];
    const i32x4 kr = tile_rsrc<32>(a.k.p + b * a.k.sb + hk * a.k.sh, a.k.st, j0, len, a.D);
    const i32x4 vr = tile_rsrc<32>(a.v.p + b * a.v.sb + hk * a.v.sh, a.v.st, j0, len, a.D);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int col = 16 * ks + 8 * (lane >> 5), r = lane & 31;
      kf[ks] = load16(kr, col < a.D ? r * (int)a.k.st * 2 + col * 2 : OOB);
      vf[ks] = load16(vr, col < a.D ? r * (int)a.v.st * 2 + col * 2 : OOB);
    }
    // The key and value fragments are here before the loop: a wait for them that the compiler put among its products would
    // be a wait for the tile just asked for too, as loads return in order.
    wait_vmcnt<0>();
    for (int it = it0; it < it1; ++it) {
      const int buf = (it - it0) & (NS - 1), img = buf * 2 * IMG;
      // this wave's loads of tile `it` have arrived when only those of the later ones are under way; behind the barrier
      // all waves' have, and all are done with the tile whose place the next load takes
      if (it + 2 < it1) wait_vmcnt<2 * LOADS>();
      else if (it + 1 < it1) wait_vmcnt<LOADS>();
      else wait_vmcnt<0>();
      __syncthreads();
      if (it + NS - 1 < it1) issue(it + NS - 1);
      const int i0 = (t0 + it % nt) * BR;
      ad.refresh();
      const bool some = i0 + BR - 1 >= j0 && (i0 - (j0 + 31) < a.window || j0 < a.sinks);
      if (some) {
        // The products of a tile in one sequence: the scores (KS), go v (KS), dv (2 DT), dk (2 DT). The fragment of each
        // is read PD - 1 products ahead, and the vector work stands between the products that do not wait for it:
        // exponentials among go v, ds among dv. fence() keeps both where they are.
        constexpr int KS = DP / 16, DT = DP / 32, N = 2 * KS + 4 * DT, PD = 3;
        auto read = [&](int i) {
          if (i < KS) return frag_rows<DP>(lds, ad, img, 0, i);
          if (i < 2 * KS) return frag_rows<DP>(lds, ad, img + IMG, 0, i - KS);
          i -= 2 * KS;
          if (i < 2 * DT) return frag_tr<DP>(lds, ad, img + IMG, i % DT, i / DT);
          i -= 2 * DT;
          return frag_tr<DP>(lds, ad, img, i % DT, i / DT);
        };
        u32x4 f[PD];
#pragma unroll
        for (int i = 0; i < PD - 1; ++i) f[i] = read(i);
        const int h = lane_now() >> 5;
        f32x16 s, ds;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&stats[buf][0][8 * e4 + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * e4 + e] = x[e];
        }
        fence();
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          f[(i + PD - 1) % PD] = read(i + PD - 1);
          s = mfma<T>(f[i % PD], kf[i], s);
          fence();
        }
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(&stats[buf][1][8 * e4 + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) ds[4 * e4 + e] = y[e];
        }
        if (!(j0 + 31 <= i0 && i0 + BR - 1 - j0 < a.window)) {
          const int key = j0 + (lane_now() & 31), rel = i0 + 4 * h - key;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int d = rel + 8 * (e / 4) + e % 4;
            const bool see = ((uint32_t)d < (uint32_t)a.window) | ((key < a.sinks) & (d >= 0));
            s[e] = see ? s[e] : -INFINITY;
          }
        }
        uint32_t dw[8];
        fence();
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          f[(KS + i + PD - 1) % PD] = read(KS + i + PD - 1);
          ds = mfma<T>(f[(KS + i) % PD], vf[i], ds);
#pragma unroll
          for (int e = i * (8 / KS); e < (i + 1) * (8 / KS); ++e) {
            s[2 * e] = __builtin_amdgcn_exp2f(s[2 * e] * c);
            s[2 * e + 1] = __builtin_amdgcn_exp2f(s[2 * e + 1] * c);
          }
          fence();
        }
        u32x4 pf;
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
          f[(2 * KS + i + PD - 1) % PD] = read(2 * KS + i + PD - 1);
          if (i % DT == 0) pf = frag_acc<T>(s, i / DT);
          dv[i % DT] = mfma<T>(f[(2 * KS + i) % PD], pf, dv[i % DT]);
#pragma unroll
          for (int e = (i - 1) * 8 / (2 * DT - 1); e < i * 8 / (2 * DT - 1); ++e)
            dw[e] = pack2<T>(s[2 * e] * ds[2 * e], s[2 * e + 1] * ds[2 * e + 1]);
          fence();
        }
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
          constexpr int AT = 2 * KS + 2 * DT;
          if (AT + i + PD - 1 < N) f[(AT + i + PD - 1) % PD] = read(AT + i + PD - 1);
          dk[i % DT] = mfma<T>(f[(AT + i) % PD], four(dw, i / DT), dk[i % DT]);
          fence();
        }
      }
    }
  }
  const int ln = lane_now(), h = ln >> 5, key = j0 + (ln & 31);
  const bool in = key < a.T, live = key < len;
  if (S == 1) {
    const int64_t ofs = (((int64_t)b * a.T + key) * a.Hkv + hk) * a.D;
    store_acc<T, DP>(dk, a.scale, a.dk + ofs, a.D, in, live, h);
    store_acc<T, DP>(dv, 1.f, a.dv + ofs, a.D, in, live, h);
  } else {
    float* const p = (sink ? a.part_s : a.part_r) + ((((int64_t)bh * nb + blk) * S + sp) * 2 * BKV + key - kb0) * a.D;
    store_f32<DP>(dk, p, a.D, in, live, h);
    store_f32<DP>(dv, p + BKV * a.D, a.D, in, live, h);
  }
}

// dk and dv of the blocks whose rows are shared by several workgroups: the sum of their parts in order, 4 columns of a
// key per thread, `pieces` workgroups per block (few blocks with many parts each: the loads have to come from many
// threads).
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(Args a, int pieces) {
  const int nk = (a.T + BKV - 1) / BKV, nr = nk - a.n_sb;
  const uint32_t heads = (uint32_t)a.B * a.Hkv, sink_blocks = a.S_s > 1 ? heads * a.n_sb : 0;
  const int i = blockIdx.x % pieces * 256 + threadIdx.x;
  uint32_t w = blockIdx.x / pieces;
  const bool sink = w < sink_blocks;
  if (!sink) w -= sink_blocks;
  const int S = sink ? a.S_s : a.S_r, nb = sink ? a.n_sb : nr;
  const int blk = w % nb, bh = w / nb, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int kb0 = (sink ? blk : a.n_sb + blk) * BKV, cols = a.D / 4;
  const int which = i / (BKV * cols), r = i / cols % BKV, d = i % cols * 4, key = kb0 + r;
  if (which > 1 || key >= a.T) return;
  const float* const p = (sink ? a.part_s : a.part_r) + ((((int64_t)bh * nb + blk) * S * 2 + which) * BKV + r) * a.D + d;
  f32x4 x = {};
#pragma unroll 4
  for (int sp = 0; sp < S; ++sp) x += *reinterpret_cast<const f32x4*>(p + (int64_t)sp * 2 * BKV * a.D);
  if (which == 0) x *= a.scale;
  u32x2 v;
  v[0] = pack2<T>(x[0], x[1]);
  v[1] = pack2<T>(x[2], x[3]);
  *reinterpret_cast<u32x2*>((which ? a.dv : a.dk) + (((int64_t)b * a.T + key) * a.Hkv + hk) * a.D + d) = v;
}

// -------------------------------------------------------------------------------------------------------- host side
int check_sizes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks) {
  if (B < 0 || T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 8 || D > 128 || D % 8 || window < 0 || sinks < 0)
    return MCE_ATTN_EINVAL;
  if (T > (int64_t(1) << 27) || Hq * D > MAX_ST) return MCE_ATTN_EINVAL;
  // one workgroup per 128 rows of every head (the backward's own are counted by its plan)
  if (T > 0 && B > MAX_GROUPS / Hq / ((T + BQ - 1) / BQ)) return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

Args make_args(Strided q, Strided k, Strided v, const int32_t* lengths, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
               int64_t D, int64_t window, int64_t sinks, float scale) {
  Args a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.lengths = lengths;
  a.B = (int)B;
  a.T = (int)T;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.D = (int)D;
  a.window = window == 0 || window >= T ? INT32_MAX : (int)window;
  a.sinks = a.window == INT32_MAX ? 0 : (int)(sinks > T ? T : sinks);
  a.scale = scale;
  return a;
}

template <typename T, int DP>
int launch_fwd(const Args& a, hipStream_t st) {
  const unsigned n = (unsigned)((int64_t)a.B * a.Hq * ((a.T + BQ - 1) / BQ));
  hipLaunchKernelGGL((k_attn_fwd<T, DP>), dim3(n), dim3(THREADS), 0, st, a);
  return finish();
}

// How many workgroups share a key block's rows in k_attn_dkv. Lengths are not known to the host: T stands for all.
struct Plan {
  int n_sb, S_s, S_r;
  int64_t part_s, part_r;   // floats of the parts
};
constexpr int64_t SLOTS = 512;    // workgroups of k_attn_dkv that run at once
constexpr int64_t MIN_ITERS = 64; // row tiles below which a workgroup is not divided
Plan make_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks) {
  Plan p = {0, 1, 1, 0, 0};
  const int64_t grp = Hq / Hkv, nk = (T + BKV - 1) / BKV, nt = (T + BR - 1) / BR, heads = B * Hkv;
  const bool causal = window == 0 || window >= T;
  if (!causal && sinks > 0) {
    p.n_sb = (int)((sinks + BKV - 1) / BKV);
    if (p.n_sb > nk) p.n_sb = (int)nk;
  }
  const int64_t units = heads * (nk - p.n_sb);
  // row tiles of the longest of the other blocks, and of all of them
  int64_t longest = causal ? nt * grp : ((BKV - 1 + window + BR - 1) / BR + 1) * grp;
  if (longest > nt * grp) longest = nt * grp;
  const double work = (double)units * longest * (causal ? 0.5 : 1.0);
  // S that ends first: rounds of equal workgroups, or (rows of different length, the longest first) the mean load and
  // half of the last ones; a tenth of a round for the parts' traffic
  double best = 1e300;
  for (int S = 1; S <= 16 && (S == 1 || longest / S >= MIN_ITERS); ++S) {
    const double each = (double)longest / S;
    const double mean = work / SLOTS;
    double cost = causal ? (mean > each ? mean : each) + 0.5 * each
                         : (double)((units * S + SLOTS - 1) / SLOTS) * each;
    if (S > 1) cost += 0.1 * mean + 8;
    if (cost < best) {
      best = cost;
      p.S_r = S;
    }
  }
  if (p.n_sb > 0) {
    // a block with first tokens is seen by every later row: no workgroup longer than the others', or than a quarter of
    // the whole
    const double each = (double)longest / p.S_r, quarter = (work + (double)heads * p.n_sb * nt * grp) / SLOTS / 4;
    const double most = each > quarter ? each : quarter;
    const double s = (double)(nt * grp) / (most < MIN_ITERS ? MIN_ITERS : most);
    p.S_s = s <= 1 ? 1 : (s > 256 ? 256 : (int)(s + 0.999));
  }
  p.part_s = p.S_s > 1 ? heads * p.n_sb * p.S_s * 2 * BKV * D : 0;
  p.part_r = p.S_r > 1 ? heads * (nk - p.n_sb) * p.S_r * 2 * BKV * D : 0;
  return p;
}

template <typename T, int DP>
int launch_bwd(const Args& a, hipStream_t st) {
  const unsigned n = (unsigned)((int64_t)a.B * a.Hq * ((a.T + BQ - 1) / BQ));
  hipLaunchKernelGGL((k_attn_dq<T, DP>), dim3(n), dim3(THREADS), 0, st, a);
  const int64_t heads = (int64_t)a.B * a.Hkv, nr = (a.T + BKV - 1) / BKV - a.n_sb;
  hipLaunchKernelGGL((k_attn_dkv<T, DP>), dim3((unsigned)(heads * (a.n_sb * a.S_s + nr * a.S_r))), dim3(THREADS), 0, st,
                     a);
  const int64_t join = heads * ((a.S_s > 1 ? a.n_sb : 0) + (a.S_r > 1 ? nr : 0));
  const int pieces = (2 * BKV * (a.D / 4) + 255) / 256;
  if (join > 0) hipLaunchKernelGGL((k_attn_dkv_join<T>), dim3((unsigned)(join * pieces)), dim3(256), 0, st, a, pieces);
  return finish();
}

}  // namespace

thread_local int mce_attn_hip_error = 0;

extern "C" {

const char* mce_attn_error_string(int code) {
  switch (code) {
    case MCE_ATTN_OK: return "ok";
    case MCE_ATTN_EINVAL: return "invalid argument (size, stride, head count, scale, element type or null pointer)";
    case MCE_ATTN_EALIGN: return "misaligned (pointers must be 16-byte aligned, strides multiples of 8 elements)";
    case MCE_ATTN_EWORKSPACE: return "workspace missing, too small or not 256-byte aligned";
    case MCE_ATTN_ELAUNCH: return "a HIP launch failed";
    default: return "unknown error";
  }
}

int mce_attn_last_hip_error(void) { return mce_attn_hip_error; }

int mce_attn_fwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                 int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const int32_t* lengths,
                 int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks, float scale,
                 int dtype, void* out, void* res, float* lse, void* stream) {
  int rc = check_sizes(B, T, Hq, Hkv, D, window, sinks);
  if (rc) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16)) return MCE_ATTN_EINVAL;
  if (B == 0 || T == 0) return MCE_ATTN_OK;
  if ((rc = check_strided(q, q_sb, q_st, q_sh, D)) || (rc = check_strided(k, k_sb, k_st, k_sh, D)) ||
      (rc = check_strided(v, v_sb, v_st, v_sh, D)))
    return rc;
  if (out == nullptr) return MCE_ATTN_EINVAL;
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(res)) & 15) return MCE_ATTN_EALIGN;
  Args a = make_args({static_cast<const uint16_t*>(q), q_sb, q_st, q_sh},
                     {static_cast<const uint16_t*>(k), k_sb, k_st, k_sh},
                     {static_cast<const uint16_t*>(v), v_sb, v_st, v_sh}, lengths, B, T, Hq, Hkv, D, window, sinks,
                     scale);
  a.o = static_cast<uint16_t*>(out);
  a.r = static_cast<uint16_t*>(res);
  a.lse = lse;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_fwd<__bf16, 64>(a, st) : launch_fwd<__bf16, 128>(a, st);
  return D <= 64 ? launch_fwd<_Float16, 64>(a, st) : launch_fwd<_Float16, 128>(a, st);
}

size_t mce_attn_bwd_ws_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                             int64_t sinks) {
  if (check_sizes(B, T, Hq, Hkv, D, window, sinks)) return 0;
  const Plan p = make_plan(B, T, Hq, Hkv, D, window, sinks);
  return (size_t)(align256(B * Hq * T * 8) + align256(p.part_s * 4) + align256(p.part_r * 4));
}

int mce_attn_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                 int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* go, int64_t go_sb,
                 int64_t go_st, int64_t go_sh, const int32_t* lengths, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                 int64_t D, int64_t window, int64_t sinks, float scale, int dtype, const void* out, const void* res,
                 const float* lse, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_sizes(B, T, Hq, Hkv, D, window, sinks);
  if (rc) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16)) return MCE_ATTN_EINVAL;
  if (B == 0 || T == 0) return MCE_ATTN_OK;
  if ((rc = check_strided(q, q_sb, q_st, q_sh, D)) || (rc = check_strided(k, k_sb, k_st, k_sh, D)) ||
      (rc = check_strided(v, v_sb, v_st, v_sh, D)) || (rc = check_strided(go, go_sb, go_st, go_sh, D)))
    return rc;
  if (out == nullptr || res == nullptr || lse == nullptr || dq == nullptr || dk == nullptr || dv == nullptr) return MCE_ATTN_EINVAL;
  for (const void* p : {out, res, (const void*)dq, (const void*)dk, (const void*)dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return MCE_ATTN_EALIGN;
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) ||
      ws_bytes < mce_attn_bwd_ws_bytes(B, T, Hq, Hkv, D, window, sinks))
    return MCE_ATTN_EWORKSPACE;
  Args a = make_args({static_cast<const uint16_t*>(q), q_sb, q_st, q_sh},
                     {static_cast<const uint16_t*>(k), k_sb, k_st, k_sh},
                     {static_cast<const uint16_t*>(v), v_sb, v_st, v_sh}, lengths, B, T, Hq, Hkv, D, window, sinks,
                     scale);
  a.go = {static_cast<const uint16_t*>(go), go_sb, go_st, go_sh};
  a.out = static_cast<const uint16_t*>(out);
  a.res = static_cast<const uint16_t*>(res);
  a.lse = const_cast<float*>(lse);
  const Plan p = make_plan(B, T, Hq, Hkv, D, window, sinks);
  const int64_t nr = (T + BKV - 1) / BKV - p.n_sb;
  if (B * Hkv * ((int64_t)p.n_sb * p.S_s + nr * p.S_r) > MAX_GROUPS) return MCE_ATTN_EINVAL;
  a.n_sb = p.n_sb;
  a.S_s = p.S_s;
  a.S_r = p.S_r;
  a.stat = static_cast<float*>(ws);
  a.part_s = a.stat + align256(B * Hq * T * 8) / 4;
  a.part_r = a.part_s + align256(p.part_s * 4) / 4;
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_bwd<__bf16, 64>(a, st) : launch_bwd<__bf16, 128>(a, st);
  return D <= 64 ? launch_bwd<_Float16, 64>(a, st) : launch_bwd<_Float16, 128>(a, st);
}

}  // extern "C"
