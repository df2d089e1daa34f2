// cache_attn.hip — attention of one new token per sequence over a paged cache of e4m3 codes, for MI355X (gfx950). The C ABI
// is in include/mce_cache.h.
//
// Every code that a sequence sees is read once and used for the query heads that share it: the pass is bound by HBM, by the
// bytes in flight, and by the instructions of a tile (32 keys of one wave), which stand in one row: half of them convert
// codes (exactly) to the element type. Products are v_mfma_f32_16x16x32 with 16 query heads as columns:
//   scores  rows are keys: lane l has 16 bytes at 16 (l/16) of every 64 of the key 8 ((l%16)/4) + 4 k + (l%16)%4 of the
//           k-th product. The summed index is the same permutation of the head's columns for the query fragments. Lane
//           l's results are then the keys 8 (l/16) + 0..7 under the query head l%16: 8 neighbouring tokens, which lie in
//           one page and share one scale.
//   values  rows are columns of the head: lane l has DP/16 neighbouring columns of the same 8 keys, so that exp(score) is
//           the other operand where it is; bytes of two keys are put side by side (one permutation per 4 bytes) and
//           converted in pairs. Product i gives the columns (DP/16) row + i.
// No value crosses lanes. A value's scale goes into its probability's exponent: w_j = exp(s_j) scale_j is what multiplies
// the codes. The denominator has an exponential and a maximum of its own: where scales lie far apart (a block of zeros has 2^-100)
// the w_j next to the largest are lost in fp32, while their exp(s_j) count (8 sequences of 131072 tokens: 203.4 us with the
// denominator from w_j / scale_j, 204.1 so; 1 of 1000 16.1 and 16.6).
// Codes come through LDS, whole memory lines by neighbouring lanes: loads straight into the registers that the products
// want them in took one request per 16 bytes, and 240 us where this took 215 (8 sequences, 131072 tokens each, 4 heads of
// 128; 200 us now, 5.4 TB/s). Each wave has its own two tiles in LDS and walks its own keys without barriers. Where the
// codes lie is worked out for 16 tiles at once, a group of 8 tokens per lane (as scalar loads of page numbers and scales,
// whose counter the reads of LDS share, a tile took 1.44 us alone on its CU; 1.03 so).
// Workgroups share the batch's tiles evenly (struct Cut): 64 sequences of 5000 tokens, 4 heads of 128, with the write of
// the new token and the join 84 us (81 now); one part size for all, 91; a fixed number of parts for each sequence 96.
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
constexpr int MIN_TILES = 2 * NW;  // tiles below which a sequence is not split further
constexpr float LAZY = 8.f;        // growth of a maximum (log2) up to which its old value is kept

struct Args {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  Codes k, v;
  Paged g;
  const int32_t* lengths;
  uint16_t* out;
  float *part, *ml;        // parts of the outputs [2 W, Hq, D]; their maxima and denominators [2 W, Hq, 2]
  int Hq, Hkv, grp, ng, D; // ng: workgroups that share a key/value head's query heads
  int page, max_pages, window, sinks;
  int B, W, G, total;      // W: workgroups per head that share the batch's tiles (0: one per sequence); G: those in a row on
                           // one XCD
  float scale;
};

// Which tiles a workgroup takes. The batch's tiles stand in a row for each head, sequence after sequence, and the W
// workgroups of the head take `run` of them each, so that all end together however far the lengths are apart; a sequence
// that goes on past a workgroup's end leaves parts, which a second launch joins: in place 2 w where it begins workgroup
// w's run, else in 2 w + 1. Every wave finds its place from the lengths, 64 sequences at a time. A sequence without a tile
// counts as one, for somebody has to write its zeros.
struct Cut {
  int run;
  static __device__ __forceinline__ int tiles_of(const Args& a, int b) {
    const int t = Seen<BK>(a, b).tiles;
    return t < 1 ? 1 : t;
  }
  static __device__ __forceinline__ int64_t sum_of(const Args& a, int n) {
    int64_t sum = 0;
    for (int i = threadIdx.x & 63; i < n; i += 64) sum += tiles_of(a, i);
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    return sum;
  }
  __device__ __forceinline__ explicit Cut(const Args& a) {
    const float r = (float)sum_of(a, a.B) / (float)a.W * 1.0001f + 1.f;   // W run is the sum at least, roundings and all
    run = __builtin_amdgcn_readfirstlane((int)r < MIN_TILES ? MIN_TILES : (int)r);
  }
  // the sequence (B: none) that holds place `at` of the row, and the place of its first tile
  static __device__ __forceinline__ int seq_of(const Args& a, int64_t at, int64_t* first) {
    int64_t before = 0;
    for (int i0 = 0; i0 < a.B; i0 += 64) {
      const int i = i0 + (threadIdx.x & 63), own = i < a.B ? tiles_of(a, i) : 0;
      int64_t n = own;
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(n, o);
        n += (int)(threadIdx.x & 63) >= o ? up : 0;
      }
      const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before + n <= at));
      if (c < 64) {
        *first = __shfl(before + n - own, c);
        return i0 + c;
      }
      before += __shfl(n, 63);
    }
    return a.B;
  }
};

// Waves per SIMD, and workgroups per CU: what 160 KiB of LDS (DP = 128) and 512 registers (DP = 64, CB = 2) leave.
constexpr int waves_per_simd(int dp, int cb) { return dp == 128 ? 2 : (cb == 1 ? 4 : 3); }

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

// Keeps the compiler from moving anything past it: it would convert a whole tile ahead of its products, in registers that
// another wave could have.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// The wave's loads into LDS but the N youngest have arrived; every read of LDS has returned. (The compiler knows nothing of
// the loads.)
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Where a tile's tokens lie: PG parts of 32 / PG tokens, each in one page, in scalar registers, and the scales of the
// lane's 8 tokens.
template <int PG>
struct Place {
  const uint8_t *k[PG], *v[PG];
  int rows[PG];          // tokens of the part in the cache and in the sequence: 0 where it is in no page, or not seen
  float ks, vs;
};

// The same of a wave's next 16 tiles: lane l has the part of group l % 4 (of 8 tokens) of the (l / 4)-th, and its scales.
struct Ahead {
  uint64_t k, v;
  int rows;
  float ks, vs;
};

// CB: column blocks of 16 query heads per workgroup. PG: pages that a tile's tokens can lie in (1 where pages are multiples
// of 32 tokens, 2 of 16, 4 of 8): what is worked out for each of them by scalar instructions is most of a tile's work.
template <typename T, int DP, int CB, int PG>
__global__ __launch_bounds__(THREADS, waves_per_simd(DP, CB)) void k_cache_attn(Args a) {
  constexpr int VB = DP / 16, VW = DP / 64;             // value columns per lane, their dwords
  constexpr int IMG = BK * DP;                          // bytes of a tile's keys or values
  __shared__ __attribute__((aligned(1024))) char lds[NW * 4 * IMG];   // two tiles per wave
  __shared__ float stat[NW][3][CB * HC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, quad = lane >> 4;
  // Workgroups go to the 8 XCDs in turn: those of G neighbouring heads, whose rows share memory lines, follow each other on
  // one of them.
  const uint32_t in = blockIdx.x / 8 % a.G, at = (blockIdx.x / 8 / a.G * 8 + blockIdx.x % 8) * a.G + in;
  if (at >= (uint32_t)a.total) return;
  const int gi = at % a.ng, hk = at / a.ng % a.Hkv, w = at / (a.ng * a.Hkv);
  const int h0 = hk * a.grp + gi * CB * HC;             // first query head
  int heads = a.grp - gi * CB * HC;
  heads = heads < CB * HC ? heads : CB * HC;
  const Paged& g = a.g;
  int b = w;
  int64_t pos0 = 0, end = INT64_MAX, first = 0;         // the workgroup's next place in the row, its end, and b's first
  if (a.W > 0) {
    const Cut cut(a);
    pos0 = (int64_t)w * cut.run;
    end = pos0 + cut.run;
    b = __builtin_amdgcn_readfirstlane(Cut::seq_of(a, pos0, &first));
    if (b >= a.B) return;
  }
  for (int place0 = 2 * w;; place0 = 2 * w + 1) {       // sequence after sequence
    const Seen<BK> sn(a, b);
    const int own = sn.tiles < 1 ? 1 : sn.tiles, t0 = __builtin_amdgcn_readfirstlane((int)(pos0 - first));
    const int stop = __builtin_amdgcn_readfirstlane((int)(end - first < own ? end - first : own));
    const int t1 = stop < sn.tiles ? stop : sn.tiles;
    const bool alone = t0 == 0 && stop == own;            // the whole sequence: no join
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
    // l = sum_j 2^((s_j - m) c), acc = sum_j 2^((s_j - m) c - u) scale_j code_j: m a maximum of the scores s_j before they are
    // scaled, u one of (s_j - m) c + log2 scale_j
    f32x4 acc[CB][VB] = {};
    float m[CB], l[CB], u[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      m[cb] = u[cb] = -INFINITY;
      l[cb] = 0.f;
    }
    const float c = a.scale * LOG2E;
    // Places in a tile. Token t has DP bytes from t DP on, in chunks of 16 bytes, chunk c at c ^ swz(t): then 8 neighbouring
    // lanes of a key fragment's read (tokens 8 ((l%16)/4) + (l%16)%4 + ...) fall on 8 different places of 128 bytes.
    auto swz = [](int t) { return DP == 128 ? (t & 3) | (t >> 3 & 1) << 2 : (t >> 1 & 1) | (t >> 3 & 1) << 1; };
    const int img = wave * 4 * IMG;
    uint32_t fk[2][DP / 64];                              // the keys' chunks of a fragment
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < DP / 64; ++e) {
        const int t = 8 * (r16 >> 2) + 4 * y + (r16 & 3);
        fk[y][e] = t * DP + (((4 * e + quad) ^ swz(t)) << 4);
      }
    // A load instruction moves 1 KiB, 16 bytes per lane: 8 tokens of 128 bytes, or 16 of 64, each half of the lanes its own 8.
    // What a lane loads lies at lds + 16 lane of the instruction's place.
    constexpr int PER = DP / 16;                          // lanes per token
    constexpr int GP = 4 / PG;                            // groups of 8 tokens per part
    constexpr bool HALVES = DP == 64 && PG == 4;          // the two halves of an instruction in different pages
    constexpr int LOADS = DP == 128 || HALVES ? 4 : 2;    // instructions for a tile's keys, and for its values
    constexpr int TPI = DP == 128 ? 8 : 16;               // tokens per instruction
    int ko[LOADS], vo[LOADS];                             // from the part's first token on
#pragma unroll
    for (int y = 0; y < LOADS; ++y) {
      const int t = (HALVES ? y / 2 : y) * TPI + lane / PER, col = ((lane % PER) ^ swz(t)) * 16, in = t % (8 * GP);
      ko[y] = col < a.D ? in * (int)a.k.st + col : OOB;
      vo[y] = col < a.D ? in * (int)a.v.st + col : OOB;
    }
    const uint8_t* const kp = a.k.p + hk * a.k.sh;
    const uint8_t* const vp = a.v.p + hk * a.v.sh;
    const int32_t* const table = g.table + b * g.bt_sb;
    // No load hangs on a condition: what is not wanted takes the table's first entry and then the cache's first page.
    auto look_up = [&](int it) {
      const int my = it + (lane >> 2) * NW, pos8 = sn.key0(my) + 8 * (lane & 3), pos = pos8 & -(8 * GP);
      const bool want = (my < t1) & (pos < sn.n) & ((pos + 8 * GP - 1 >= sn.lo) | (pos < a.sinks));
      const uint32_t g8 = ((uint32_t)pos >> 3) & -(uint32_t)want, pi = g.page8(g8);
      const int pg = table[pi];
      const bool ok = want & ((uint32_t)pg < (uint32_t)g.pages);
      const uint32_t mask = -(uint32_t)ok, at = pg & mask, slot = (g8 * 8 - pi * a.page) & mask;
      const int64_t e = g.scale_at((int)at, (slot >> 3) + ((lane & 3) % GP & mask), hk);
      Ahead h;
      h.ks = a.k.scale[e];
      h.vs = a.v.scale[e];
      h.k = (uint64_t)at * a.k.sp + (uint64_t)slot * a.k.st;
      h.v = (uint64_t)at * a.v.sp + (uint64_t)slot * a.v.st;
      const int left = sn.n - pos;
      h.rows = (left < 8 * GP ? left : 8 * GP) & (int)mask;
      return h;
    };
    auto lane64 = [](uint64_t x, int at) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), at) << 32 |
             (uint32_t)__builtin_amdgcn_readlane((int)x, at);
    };
    // i: the tile's number among the 16
    auto place = [&](const Ahead& h, int i) {
      Place<PG> t;
#pragma unroll
      for (int y = 0; y < PG; ++y) {
        t.k[y] = kp + lane64(h.k, 4 * i + GP * y);
        t.v[y] = vp + lane64(h.v, 4 * i + GP * y);
        t.rows[y] = __builtin_amdgcn_readlane(h.rows, 4 * i + GP * y);
      }
      t.ks = __shfl(h.ks, 4 * i + quad);
      t.vs = __shfl(h.vs, 4 * i + quad);
      return t;
    };
    // parts without rows, and rows behind the sequence's end, come as zeros and touch no memory
    auto load = [&](const uint8_t* const (&p)[PG], const int (&rows)[PG], int st, const int (&o)[LOADS], int to) {
#pragma unroll
      for (int y = 0; y < PG; ++y) {
        const i32x4 rs = make_rsrc(p[y], rows[y] > 0 ? (rows[y] - 1) * st + a.D : 0);
        if constexpr (HALVES) {
          if (lane >> 5 == (y & 1)) dma16(rs, lds, to + (y >> 1) * 1024, o[y]);
        } else {
#pragma unroll
          for (int z = y * LOADS / PG; z < (y + 1) * LOADS / PG; ++z) dma16(rs, lds, to + z * 1024, o[z]);
        }
      }
    };
    const int kst_b = (int)a.k.st, vst_b = (int)a.v.st;
    // Tile it, which lies at buf, and the loads of tile it + 2 NW (`then`) into its place: the keys' when the scores are
    // there, the values' when they are in registers. Three quarters of two tiles are under way at every wait.
    auto use = [&](int it, int buf, const Place<PG>& t, const Place<PG>& then) {
      float ks = t.ks, vs = t.vs;
      const int k0 = sn.key0(it);
      const int pos = k0 + 8 * quad;                      // the lane's first token
      int all = 8 * GP;
#pragma unroll
      for (int y = 0; y < PG; ++y) all &= t.rows[y];      // (a part has 8 GP rows, a power of two, or fewer)
      const bool edge = (all != 8 * GP) | (k0 < sn.lo);
      uint32_t see = 0xFF;
      if (edge) {
        int n = t.rows[0];
#pragma unroll
        for (int y = 1; y < PG; ++y) n = quad / GP == y ? t.rows[y] : n;
        n -= quad % GP * 8;
        see = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) see |= (uint32_t)((j < n) & ((pos + j >= sn.lo) | (pos + j < a.sinks))) << j;
        ks = see ? ks : 1.f;
        vs = see ? vs : 1.f;
      }
      wait_loads<3 * LOADS>();
      f32x4 sc[CB][2] = {};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < DP / 64; ++e) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(lds + buf + fk[kb][e]);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            u32x4 f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              f[2 * w] = from_codes<T, false>(x[2 * hf + w]);
              f[2 * w + 1] = from_codes<T, true>(x[2 * hf + w]);
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) sc[cb][kb] = mfma16<T>(f, qf[cb][2 * e + hf], sc[cb][kb]);
          }
        }
      wait_reads();
      load(then.k, then.rows, kst_b, ko, buf);
      const float lv = __builtin_amdgcn_logf(vs);
      u32x4 pf[CB];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        auto over_heads = [](float y) { return max_halves(fmaxf(y, __shfl_xor(y, 16))); };   // a head's maximum
        float x[8], mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = sc[cb][e / 4][e % 4] * ks;
          if (edge) x[e] = (see >> e & 1) ? x[e] : -INFINITY;
          mx = fmaxf(mx, x[e]);
        }
        const float mu0 = m[cb] == -INFINITY ? 0.f : m[cb];
        // the sums are rescaled only when some head's maximum has grown by more than LAZY since the last time
        if (__builtin_amdgcn_ballot_w64(((mx - m[cb]) * c > LAZY) | ((mx - mu0) * c + lv - u[cb] > LAZY)) != 0) {
          const float top = fmaxf(m[cb], over_heads(mx)), by = top == -INFINITY ? 0.f : (m[cb] - top) * c;
          l[cb] *= __builtin_amdgcn_exp2f(by);
          m[cb] = top;
          const float y = over_heads((mx - (top == -INFINITY ? 0.f : top)) * c + lv);
          const float un = fmaxf(u[cb] + by, y);
          const float al = un == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(u[cb] + by - un);
          u[cb] = un;
#pragma unroll
          for (int i = 0; i < VB; ++i) acc[cb][i] *= al;
        }
        const float mu = m[cb] == -INFINITY ? 0.f : m[cb], d = lv - (u[cb] == -INFINITY ? 0.f : u[cb]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = (x[e] - mu) * c;
          sum += __builtin_amdgcn_exp2f(x[e]);
          x[e] = __builtin_amdgcn_exp2f(x[e] + d);
        }
        l[cb] += sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[cb][e] = pack2<T>(x[2 * e], x[2 * e + 1]);
      }
      wait_loads<3 * LOADS>();
      uint32_t v[8][VW];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 8 * quad + j, col = r16 * VB;
        const char* const p = lds + buf + IMG + t * DP + (((col >> 4) ^ swz(t)) << 4) + (col & 15);
        if constexpr (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p);
          v[j][0] = x[0];
          v[j][1] = x[1];
        } else {
          v[j][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
      wait_reads();
      load(then.v, then.rows, vst_b, vo, buf + IMG);
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int w = 0; w < VW; ++w) v[j][w] &= -(see >> j & 1);   // (0 times a NaN is one)
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {                  // bytes 2 hf and 2 hf + 1 of each dword
          u32x4 f[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t p = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], hf ? 0x07030602u : 0x05010400u);
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
          fence();
        }
    };
    // the query fragments are here before the first tile's loads go out: a wait for them would be a wait for those
    wait_vmcnt<0>();
    int it = t0 + wave, buf = img;
    if (it < t1) {
      Ahead next = look_up(it);
      Place<PG> one = place(next, 0), two = place(next, 1);
      load(one.k, one.rows, kst_b, ko, buf);
      load(one.v, one.rows, vst_b, vo, buf + IMG);
      load(two.k, two.rows, kst_b, ko, buf ^ (2 * IMG));
      load(two.v, two.rows, vst_b, vo, (buf ^ (2 * IMG)) + IMG);
      for (int i = 2; it < t1; it += NW, ++i) {           // tile it, and the loads of the i-th
        if ((i & 15) == 0) next = look_up(it + 2 * NW);
        const Place<PG> then = place(next, i & 15);       // (behind the last tile: zeros)
        use(it, buf, one, then);
        one = two;
        two = then;
        buf ^= 2 * IMG;
      }
      wait_loads<0>();                                    // (the zeros: the sums below go where they go)
    }
    // join the waves: each leaves its sums [head][D] and its state
    static_assert(CB * HC * DP * 4 <= 4 * IMG, "a wave's sums fit into its tiles");
    float* const mine = reinterpret_cast<float*>(lds + img);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      l[cb] += __shfl_xor(l[cb], 16);
      l[cb] = sum_halves(l[cb]);
      if (quad == 0) {
        stat[wave][0][cb * HC + r16] = m[cb];
        stat[wave][1][cb * HC + r16] = l[cb];
        stat[wave][2][cb * HC + r16] = u[cb];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i4 = 0; i4 < VB; i4 += 4) {
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = acc[cb][i4 + i][e];
          *reinterpret_cast<f32x4*>(mine + (cb * HC + r16) * DP + (4 * quad + e) * VB + i4) = x;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (DP / 4); i += THREADS) {
      const int hd = i / (DP / 4), d = i % (DP / 4) * 4;
      if (d >= a.D) continue;
      float mm = -INFINITY, ll = 0.f, t[NW], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) mm = fmaxf(mm, stat[w][0][hd]);
      const float mu = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        t[w] = (stat[w][0][hd] - mu) * c;
        ll = __builtin_fmaf(stat[w][1][hd], __builtin_amdgcn_exp2f(t[w]), ll);
        t[w] += stat[w][2][hd];
        top = fmaxf(top, t[w]);
      }
      top = top == -INFINITY ? 0.f : top;
      f32x4 o = {};
#pragma unroll
      for (int w = 0; w < NW; ++w)
        o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * 4 * IMG) + hd * DP + d) *
             __builtin_amdgcn_exp2f(t[w] - top);
      // nothing seen: 0; NaN stays
      o *= (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll)) * __builtin_amdgcn_exp2f(top);
      const int64_t row = (int64_t)b * a.Hq + h0 + hd;
      if (alone) {
        u32x2 w;
        w[0] = pack2<T>(o[0], o[1]);
        w[1] = pack2<T>(o[2], o[3]);
        *reinterpret_cast<u32x2*>(a.out + row * a.D + d) = w;
      } else {
        const int64_t to = (int64_t)place0 * a.Hq + h0 + hd;
        *reinterpret_cast<f32x4*>(a.part + to * a.D + d) = o;
        if (d == 0) {
          a.ml[to * 2] = mm;
          a.ml[to * 2 + 1] = ll;
        }
      }
    }
    first += own;
    if (a.W == 0 || first >= end || ++b >= a.B) return;
    pos0 = first;
    __syncthreads();                                      // the sums were read: tiles go in their place
  }
}

// out = the parts of one query head joined, each by its share of the denominator: one wave per head, 2 columns per lane, 64
// parts at a time. Their states are read by all lanes at once and their factors shared through LDS, so that the sums' loads
// depend on nothing. A wave looks at
// a sequence, or, where workgroups are fewer, at the place where one of them ends, and takes the sequence that goes on there
// for the first time (4096 sequences, 32 heads: 433 us by sequences, 57 by ends).
template <typename T>
__global__ __launch_bounds__(64) void k_cache_join(Args a) {
  __shared__ float f[64];
  const int h = blockIdx.x % a.Hq, at = blockIdx.x / a.Hq, lane = threadIdx.x, d = lane * 2;
  const int64_t run = Cut(a).run;
  int b = at;
  int64_t first;
  if (a.B <= a.W) {
    first = Cut::sum_of(a, b);
  } else {
    b = Cut::seq_of(a, (at + 1) * run, &first);
    if (b >= a.B || first / run != at) return;
  }
  const int64_t w0 = first / run;
  const int n = (int)((first + Cut::tiles_of(a, b) - 1) / run - w0) + 1;
  if (n == 1) return;
  // part s: place 2 (w0 + s), the first one behind if it does not begin its workgroup's run
  const int64_t late = first % run != 0 ? 1 : 0;
  auto row = [&](int s) { return (2 * (w0 + s) + (s == 0 ? late : 0)) * a.Hq + h; };
  float mm = -INFINITY;
  for (int s = lane; s < n; s += 64) mm = fmaxf(mm, a.ml[row(s) * 2]);
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
  const float mu = mm == -INFINITY ? 0.f : mm, c = a.scale * LOG2E;
  auto own = [&](int s) { return a.ml[row(s) * 2 + 1] * __builtin_amdgcn_exp2f((a.ml[row(s) * 2] - mu) * c); };
  float ll = 0.f, x = 0.f, y = 0.f;
  for (int s = lane; s < n; s += 64) ll += own(s);
  for (int o = 32; o > 0; o >>= 1) ll += __shfl_xor(ll, o);
  const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);   // nothing seen: 0; NaN stays
  for (int s0 = 0; s0 < n; s0 += 64) {
    const int s = s0 + lane, c = n - s0 < 64 ? n - s0 : 64;
    __syncthreads();
    if (s < n) f[lane] = own(s) * inv;
    __syncthreads();
    if (d < a.D) {
#pragma unroll 8
      for (int i = 0; i < c; ++i) {
        const float2 v = *reinterpret_cast<const float2*>(a.part + row(s0 + i) * a.D + d);
        x = __builtin_fmaf(v.x, f[i], x);
        y = __builtin_fmaf(v.y, f[i], y);
      }
    }
  }
  if (d < a.D) *reinterpret_cast<uint32_t*>(a.out + ((int64_t)b * a.Hq + h) * a.D + d) = pack2<T>(x, y);
}

// --------------------------------------------------------------------------------------------------------- host side

int64_t heads_of(int64_t grp) { return grp <= HC ? HC : 2 * HC; }

// Workgroups that share a head's tiles, 0 where each sequence has one of its own. Lengths are not known here.
int64_t shared_by(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages, int64_t window,
                  int64_t sinks) {
  int64_t n = page * max_pages;
  if (window > 0 && window + sinks < n) n = window + sinks;
  const int64_t grp = Hq / Hkv, tiles = (n + BK - 1) / BK + 2, heads = Hkv * ((grp + heads_of(grp) - 1) / heads_of(grp));
  const int64_t slots = 256 * waves_per_simd(D > 64 ? 128 : 64, grp > HC ? 2 : 1);   // workgroups that run at once
  if (tiles <= MIN_TILES || (B * heads >= slots / 2 && B * heads * tiles < 65536)) return 0;
  const int64_t w = slots / heads, most = B * ((tiles + MIN_TILES - 1) / MIN_TILES);
  return w < 1 ? 1 : (w < most ? w : most);
}

int64_t gcd(int64_t x, int64_t y) { return y == 0 ? x : gcd(y, x % y); }

int check_attn(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages, int64_t window,
               int64_t sinks) {
  const int rc = check_paged_sizes(B, Hkv, D, 0, page, 8, max_pages, 0);
  if (rc) return rc;
  if (Hq < 1 || Hq > 65536 || Hq % Hkv || window < 0 || sinks < 0 || B * Hq > MAX_GROUPS) return MCE_ATTN_EINVAL;
  const int64_t grp = Hq / Hkv, heads = Hkv * ((grp + heads_of(grp) - 1) / heads_of(grp));
  if (B > (MAX_GROUPS - (1 << 20)) / heads) return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

size_t ws_bytes_of(int64_t Hq, int64_t D, int64_t W) {
  return (size_t)(align256(2 * W * Hq * D * 4) + align256(2 * W * Hq * 8));
}

template <typename T, int DP>
int launch(const Args& a, int64_t B, hipStream_t st) {
  const int set = 8 * a.G;   // workgroups of G heads on each XCD
  const dim3 grid((unsigned)((a.total + set - 1) / set * set)), threads(THREADS);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, threads, 0, st, a); };
  const int pg = a.page % 32 == 0 ? 1 : (a.page % 16 == 0 ? 2 : 4);
  if (a.grp <= HC) run(pg == 1 ? k_cache_attn<T, DP, 1, 1> : (pg == 2 ? k_cache_attn<T, DP, 1, 2> : k_cache_attn<T, DP, 1, 4>));
  else run(pg == 1 ? k_cache_attn<T, DP, 2, 1> : (pg == 2 ? k_cache_attn<T, DP, 2, 2> : k_cache_attn<T, DP, 2, 4>));
  const int64_t joins = B <= a.W ? B : (a.W > 0 ? a.W - 1 : 0);
  if (joins > 0) hipLaunchKernelGGL((k_cache_join<T>), dim3((unsigned)(joins * a.Hq)), dim3(64), 0, st, a);
  return finish();
}

}  // namespace

extern "C" {

size_t mce_cache_attn_ws_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t max_pages,
                               int64_t window, int64_t sinks) {
  if (check_attn(B, Hq, Hkv, D, page, max_pages, window, sinks) || B == 0) return 0;
  return ws_bytes_of(Hq, D, shared_by(B, Hq, Hkv, D, page, max_pages, window, sinks));
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
  const int64_t W = shared_by(B, Hq, Hkv, D, page, max_pages, window, sinks), need = (int64_t)ws_bytes_of(Hq, D, W);
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
  a.ml = reinterpret_cast<float*>(static_cast<char*>(ws) + align256(2 * W * Hq * D * 4));
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.ng = (int)((a.grp + heads_of(a.grp) - 1) / heads_of(a.grp));
  a.D = (int)D;
  a.page = (int)page;
  a.max_pages = a.g.max_pages;
  a.window = window == 0 || window > INT32_MAX ? INT32_MAX : (int)window;
  a.sinks = a.window == INT32_MAX ? 0 : (int)(sinks < (1 << 30) ? sinks : 1 << 30);
  a.B = (int)B;
  a.W = (int)W;
  a.total = (int)((W > 0 ? W : B) * Hkv * a.ng);
  a.G = a.ng * (int)gcd(Hkv, 128 / gcd(D, 128));   // heads whose rows of D bytes fill whole memory lines of 128
  a.scale = scale;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch<__bf16, 64>(a, B, st) : launch<__bf16, 128>(a, B, st);
  return D <= 64 ? launch<_Float16, 64>(a, B, st) : launch<_Float16, 128>(a, B, st);
}

}  // extern "C"
