// attn_kernels.h — causal attention over a sliding window with first tokens that stay visible, forward and backward, for
// MI355X (gfx950): the kernels of window_attention (attn.hip: a padded batch) and packed_attention (packed.hip: PK, sequences
// that lie behind each other). Tiles and fragments are in attn_tile.h.
#ifndef MEMARCH_ATTN_KERNELS_H
#define MEMARCH_ATTN_KERNELS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_host.h"
#include "attn_tile.h"
#include "seq_find.h"

namespace {

using namespace attn;

constexpr int NW = 4;               // waves per workgroup
constexpr int THREADS = 64 * NW;
constexpr int BQ = 32 * NW;         // query rows per workgroup of k_attn_fwd and k_attn_dq (32 per wave)
constexpr int BK = 64;              // keys per tile there
constexpr int BKV = 32 * NW;        // keys per workgroup of k_attn_dkv (32 per wave)
constexpr int BR = 32;              // query rows per tile there
constexpr int NS = 4;               // tiles of k_attn_dkv's ring

constexpr int64_t MIN_ITERS = 64;   // row tiles below which a workgroup of k_attn_dkv is not divided
constexpr int64_t MIN_PACK = 32;    // the same of packed sequences (4 of 4096 tokens, 4 heads on one, window 512: 60 us; 78
                                    // with 64)

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
  // Packed sequences (below): B = 1, T = rows of q. [B, T, ...] above are [N, ...] or [head, ..., N], and the parts are
  // [unit Hkv, S, 2, BKV, D].
  const int32_t *cu, *cu_k;  // starts of the nseq sequences in the rows of q and of k, and their ends
  int nseq, M;               // M: rows of k
  int uq, uk;                // units of BQ rows of q and of BKV rows of k
  int us, by_key;            // units of key blocks with first tokens: n_sb of every sequence, or (by_key) those of k
  struct Unit* plan;         // those of q and then those of k, the longest first; null: in their own order
  // workgroups that share the key tiles of a unit of q (1: SPLIT is false); query heads of each (1, 2 or 4) then, and
  // whether sequences have no more rows on average than one workgroup takes of a head
  int S_q, fold, thin;
  float *part_q, *ml;        // their sums [S_q, N, Hq, D], and maxima and denominators (sums of ds and d) [S_q, N, Hq, 2]
};

// Packed sequences: rows of different sequences lie behind each other, sequence s in rows cu[s] .. cu[s + 1] - 1 of q and
// cu_k[s] .. cu_k[s + 1] - 1 of k, and its rows of q are the last of its rows of k. The rows before the first sequence and
// behind the last are sequences of their own (numbers 0 and nseq + 1, the others one further) without keys or without
// rows, so that every row of the results is written. Sequence s's blocks of BLK rows are the units from
// floor(start(s) / BLK) + s on: those are at least as many as it has blocks, as floor((c + n) / BLK) + 1 - floor(c / BLK)
// >= ceil(n / BLK), so that a unit finds its sequence from the starts alone, whatever the lengths, which the host need
// not know; at most one unit per sequence is left over. Starts outside 0 .. rows count as the nearest of the two.
__device__ __forceinline__ int start_of(const int32_t* cu, int nseq, int rows, int s) {
  return s == 0 ? 0 : (s > nseq + 1 ? rows : start_in(cu, s - 1, rows));
}
// A block of BQ rows of q or BKV rows of k: what its workgroup has to know of its sequence.
struct Unit {
  int q0, k0;      // first rows
  int lq, lk;      // rows of q and of k (outside every sequence they have nothing in common: the other's are 0)
  int blk;         // which of the sequence's blocks (below 0, where starts fall: none)
  int outside;
  int pad[2];
};
template <bool KEYS>
__device__ __forceinline__ Unit unit_of(const Args& a, int s, int u) {
  Unit x;
  x.q0 = start_of(a.cu, a.nseq, a.T, s);
  x.lq = start_of(a.cu, a.nseq, a.T, s + 1) - x.q0;
  x.k0 = start_of(a.cu_k, a.nseq, a.M, s);
  x.lk = start_of(a.cu_k, a.nseq, a.M, s + 1) - x.k0;
  x.outside = s == 0 || s == a.nseq + 1;
  x.blk = u - (KEYS ? x.k0 / BKV : x.q0 / BQ) - s;
  x.lq = x.lq < 0 || (KEYS && x.outside) ? 0 : x.lq;
  x.lk = x.lk < 0 || (!KEYS && x.outside) ? 0 : x.lk;
  return x;
}
// The u-th unit of the launch's order.
template <bool KEYS>
__device__ __forceinline__ Unit unit_at(const Args& a, int u) {
  if (a.plan != nullptr) {
    typedef const int __attribute__((address_space(4))) * Ints;
    const Ints p = (Ints)(a.plan + (KEYS ? a.uq : 0) + u);
    Unit x;
    x.q0 = p[0];
    x.k0 = p[1];
    x.lq = p[2];
    x.lk = p[3];
    x.blk = p[4];
    x.outside = p[5];
    return x;
  }
  constexpr int BLK = KEYS ? BKV : BQ;
  const int32_t* const cu = KEYS ? a.cu_k : a.cu;
  const int rows = KEYS ? a.M : a.T;
  return unit_of<KEYS>(a, last_from(a.nseq + 2, u, [&](int s) { return start_of(cu, a.nseq, rows, s) / BLK + s; }), u);
}

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  if (a.lengths == nullptr) return a.T;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// The block of BQ rows of q that a workgroup takes. Rows are named by their positions: q0 of the first, `off` less is its
// place in the sequence's rows of q, of which `own` are written; there are `len` keys. In the packed form positions below
// 0 see nothing.
template <bool PK>
struct Rows {
  int q0, len, off, own;
  int64_t qrow, krow;   // first row of q and of k (packed)
  __device__ __forceinline__ explicit Rows(const Unit& x) {
    own = x.blk < 0 ? 0 : x.lq;
    len = x.blk < 0 ? 0 : x.lk;
    off = len - own;
    qrow = x.q0;
    krow = x.k0;
    q0 = (x.blk < 0 ? 0 : x.blk) * BQ + off;
  }
  __device__ __forceinline__ Rows(const Args& a, int b, int blk) {
    if constexpr (PK) {
      *this = Rows(unit_at<false>(a, blk));
    } else {
      q0 = blk * BQ;
      len = seq_len(a, b);
      off = 0;
      own = a.T;
      qrow = krow = 0;
    }
  }
  // rows that are read of q's; the first and the last position that sees a key, and whether one does
  __device__ __forceinline__ int read() const { return PK ? own : len; }
  __device__ __forceinline__ int first() const { return PK && q0 < 0 ? 0 : q0; }
  __device__ __forceinline__ int last() const { return (q0 + BQ < len ? q0 + BQ : len) - 1; }
  __device__ __forceinline__ bool any() const { return q0 < len && (!PK || last() >= 0); }
  // whether a row is the sequence's (and written), and whether it sees a key
  __device__ __forceinline__ bool in(int row) const { return row - off < own; }
  __device__ __forceinline__ bool live(int row) const { return PK ? row >= 0 && in(row) : row < len; }
};

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
  // n: blocks per head; sub: query heads of a group that are workgroups of their own (grp, or 1); sorted: block 0 is the
  // longest all the same
  __device__ __forceinline__ Place(const Args& a, uint32_t bid, uint32_t n, uint32_t sub, bool sorted) {
    const uint32_t kv = (uint32_t)a.B * a.Hkv;
    const bool whole = kv % 8 == 0, heads = !whole && kv * sub % 8 == 0;
    const uint32_t units = heads ? kv * sub : kv, in = heads ? 1 : sub;   // units per XCD set, workgroups inside a unit
    const uint32_t x = whole || heads ? 8 : 1, xcd = bid % x, slot = bid / x, ux = units / x;
    uint32_t u, i;
    if (sorted || a.window == INT32_MAX) {
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

// Few rows behind many keys: the key tiles of a block of rows are shared by up to S_q workgroups (SPLIT), none of which
// gets fewer than MIN_KEYS tiles, and a launch of its own joins their fp32 sums. A workgroup's waves take up to 4 (`fold`)
// query heads of a group with fewer rows each, so that the group's keys are loaded once, and its other heads follow on the
// same XCD (1 row behind 131072 keys, 16 heads over 4, in us: 2282 by one workgroup per head; in parts 227, with a group on one
// XCD 149, folded and in better order 66, which is 4.0 TB/s; 16 heads over 16 are as fast as HBM). The host does not know how many
// rows and parts a block has: those that are left over come behind the others, as between them they left those on few CUs
// (64 rows: 88 us, 46 so).
constexpr int MIN_KEYS = 8;
struct SplitPlace {
  int hk, g, r, blk, sp;   // g: the wave's query head of its group; r: its first row in the block
  bool none;
  __device__ __forceinline__ SplitPlace(const Args& a, uint32_t bid, int wave) {
    const uint32_t slot = bid / 8, rows = BQ / a.fold, in = rows / 32;   // rows of each head, waves for them
    // i: which `fold` heads of the group; q: which quarter (half) of the block's rows
    uint32_t i = slot % a.grp, q = i % a.fold, at = slot / a.grp;
    i /= a.fold;
    if (a.thin) {                                       // few sequences have rows for more than the first
      const uint32_t heads = a.grp / a.fold, all = ((uint32_t)a.Hkv * a.uq * a.S_q + 7) / 8 * heads;
      q = slot / all;
      i = slot % all % heads;
      at = slot % all / heads;
    }
    const uint32_t set = at * 8 + bid % 8, w = set / a.Hkv;
    g = i * a.fold + wave / in;
    r = q * rows + wave % in * 32;
    hk = set % a.Hkv;
    blk = w / a.S_q;
    sp = w % a.S_q;
    none = blk >= a.uq;
  }
};
__device__ __forceinline__ int key_parts(const Args& a, int tiles) {
  const int n = tiles / MIN_KEYS;
  return n < 1 ? 1 : (n < a.S_q ? n : a.S_q);
}
// The sums of a block's rows that a joining workgroup puts together: 4 columns of a row at a time.
struct Joint {
  Rows<true> at;
  int hq, parts;
  __device__ __forceinline__ Joint(const Args& a, uint32_t w) : at(a, 0, (int)(w / a.Hq)), hq(w % a.Hq), parts(1) {
    if (at.any()) parts = key_parts(a, KeyTiles(a, at.first(), at.last()).n);
  }
  // f(row, its number among all rows, column); pieces workgroups share the block
  template <typename F>
  __device__ __forceinline__ void each(const Args& a, int pieces, F f) const {
    const int cols = a.D / 4;
    for (int i = blockIdx.x % pieces * 256 + threadIdx.x; i < BQ * cols; i += pieces * 256) {
      const int row = at.q0 + i / cols;
      if (!at.in(row)) return;
      f(row, at.qrow + row - at.off, i % cols * 4);
    }
  }
};
__device__ __forceinline__ int64_t part_at(const Args& a, int sp, int64_t line, int hq) {
  return (((int64_t)sp * a.T + line) * a.Hq + hq);
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
template <typename T, int DP, bool PK, bool SPLIT>
__global__ __launch_bounds__(THREADS, DP == 64 ? 4 : 2) void k_attn_fwd(Args a) {
  constexpr int IMG = BK * DP * 2;                     // bytes of a tile
  __shared__ __attribute__((aligned(1024))) char lds[4 * IMG];   // K and V, two tiles each
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int nq = PK ? a.uq : (a.T + BQ - 1) / BQ;
  int b = 0, hk, g, blk, sp = 0, parts = 1, r = wave * 32;
  if constexpr (SPLIT) {
    const SplitPlace pl(a, blockIdx.x, wave);
    if (pl.none) return;
    hk = pl.hk;
    g = pl.g;
    blk = pl.blk;
    sp = pl.sp;
    r = pl.r;
  } else {
    const Place pl(a, blockIdx.x, nq, a.grp, PK && a.plan != nullptr);
    b = pl.b;
    hk = pl.hk;
    g = pl.g;
    blk = PK && a.plan ? pl.blk : nq - 1 - pl.blk;
  }
  const int hq = hk * a.grp + g, bh = b * a.Hq + hq;
  const Rows<PK> at(a, b, blk);
  const int len = at.len, q0 = at.q0, r0 = q0 + r, row = r0 + (lane & 31);
  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;
  bool large = false;   // some row's m is beyond LARGE
  const float c = a.scale * LOG2E;
  if (at.any()) {
    const KeyTiles kt(a, at.first(), at.last());
    if constexpr (SPLIT) parts = key_parts(a, kt.n);
    if (SPLIT && (sp >= parts || !at.in(q0 + r / (BQ / a.fold) * (BQ / a.fold)))) return;
    const int t0 = SPLIT ? kt.n * sp / parts : 0, t1 = SPLIT ? kt.n * (sp + 1) / parts : kt.n;
    FragAddr<DP> ad;
    ad.init(lane);
    TileLoad<DP, BK, NW> tk, tv;
    tk.init((int)a.k.st * 2, a.D, wave, lane);
    tv.init((int)a.v.st * 2, a.D, wave, lane);
    const uint16_t* const kp = a.k.p + (PK ? at.krow * a.k.st : b * a.k.sb) + hk * a.k.sh;
    const uint16_t* const vp = a.v.p + (PK ? at.krow * a.v.st : b * a.v.sb) + hk * a.v.sh;
    auto issue = [&](int it, int buf) {
      const int k0 = kt.key0(it), end = kt.end(it, a, len);
      tk.issue(tile_rsrc<BK>(kp, a.k.st, k0, end, a.D), lds, buf * 2 * IMG, wave);
      tv.issue(tile_rsrc<BK>(vp, a.v.st, k0, end, a.D), lds, buf * 2 * IMG + IMG, wave);
    };
    issue(t0, 0);
    // the wave's query rows as fragments: row l%32, columns 16 ks + 8 h + 0..7
    u32x4 qf[DP / 16];
    const i32x4 qr = tile_rsrc<32>(a.q.p + (PK ? at.qrow * a.q.st : b * a.q.sb) + hq * a.q.sh, a.q.st, r0 - at.off, at.read(), a.D);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int col = 16 * ks + 8 * h;
      qf[ks] = load16(qr, col < a.D ? (lane & 31) * (int)a.q.st * 2 + col * 2 : OOB);
    }
    wait_vmcnt<0>();
    __syncthreads();
    for (int it = t0; it < t1; ++it) {
      const int img = (it - t0 & 1) * 2 * IMG;
      if (it + 1 < t1) issue(it + 1, it + 1 - t0 & 1);
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
  if (SPLIT && sp >= parts) return;                       // (a block that sees nothing)
  l = sum_halves(l);
  const int64_t line = at.qrow + row - at.off;
  const int64_t ofs = ((int64_t)b * a.T + line) * a.Hq * a.D + (int64_t)hq * a.D;
  const bool in = at.in(row), see = at.live(row);
  if (SPLIT && parts > 1) {
    const int64_t to = part_at(a, sp, line, hq);
    store_f32<DP>(acc, a.part_q + to * a.D, a.D, in, see, h);
    if (in && h == 0) {
      a.ml[to * 2] = m;
      a.ml[to * 2 + 1] = l;
    }
    return;
  }
  const float inv = 1.f / l;
  store_acc<T, DP>(acc, inv, a.o + ofs, a.D, in, see, h);
  if (a.r != nullptr) store_acc<T, DP, true>(acc, inv, a.r + ofs, a.D, in, see, h);
  if (a.lse != nullptr && in && h == 0) a.lse[(int64_t)bh * a.T + line] = see ? m + __builtin_amdgcn_logf(l) / c : INFINITY;
}

// out, res and lse of the rows whose keys were shared.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_fwd_join(Args a, int pieces) {
  const Joint jt(a, blockIdx.x / pieces);
  if (jt.parts == 1) return;
  const float c = a.scale * LOG2E;
  jt.each(a, pieces, [&](int row, int64_t line, int d) {
    const bool live = jt.at.live(row);
    float mm = -INFINITY, l = 0.f;
#pragma unroll 16
    for (int sp = 0; sp < jt.parts; ++sp) mm = fmaxf(mm, a.ml[part_at(a, sp, line, jt.hq) * 2]);
    f32x4 x = {};
#pragma unroll 16
    for (int sp = 0; sp < jt.parts; ++sp) {
      const int64_t p = part_at(a, sp, line, jt.hq);
      const float f = __builtin_amdgcn_exp2f((a.ml[p * 2] - mm) * c);
      l = __builtin_fmaf(a.ml[p * 2 + 1], f, l);
      x += *reinterpret_cast<const f32x4*>(a.part_q + p * a.D + d) * f;
    }
    x *= 1.f / l;
    const int64_t to = (line * a.Hq + jt.hq) * a.D + d;
    u32x2 o, e;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      o[i] = live ? pack2<T>(x[2 * i], x[2 * i + 1]) : 0;
      e[i] = live ? pack2<T>(x[2 * i] - lo_f32<T>(o[i]), x[2 * i + 1] - hi_f32<T>(o[i])) : 0;
    }
    *reinterpret_cast<u32x2*>(a.o + to) = o;
    if (a.r != nullptr) *reinterpret_cast<u32x2*>(a.r + to) = e;
    if (a.lse != nullptr && d == 0)
      a.lse[(int64_t)jt.hq * a.T + line] = live ? mm + __builtin_amdgcn_logf(l) / c : INFINITY;
  });
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
template <typename T, int DP, bool PK, bool SPLIT>
__global__ __launch_bounds__(THREADS, 2) void k_attn_dq(Args a) {
  constexpr int IMG = BK * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[4 * IMG];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nq = PK ? a.uq : (a.T + BQ - 1) / BQ;
  int b = 0, hk, g, blk, sp = 0, parts = 1, r = wave * 32;
  if constexpr (SPLIT) {
    const SplitPlace pl(a, blockIdx.x, wave);
    if (pl.none) return;
    hk = pl.hk;
    g = pl.g;
    blk = pl.blk;
    sp = pl.sp;
    r = pl.r;
  } else {
    const Place pl(a, blockIdx.x, nq, a.grp, PK && a.plan != nullptr);
    b = pl.b;
    hk = pl.hk;
    g = pl.g;
    blk = PK && a.plan ? pl.blk : nq - 1 - pl.blk;
  }
  const int hq = hk * a.grp + g, bh = b * a.Hq + hq;
  const Rows<PK> at(a, b, blk);
  const int len = at.len, q0 = at.q0, r0 = q0 + r;
  f32x16 acc[DP / 32] = {};
  float delta = 0.f, nl = -INFINITY, sum = 0.f;
  const float c = a.scale * LOG2E;
  if (at.any()) {
    const KeyTiles kt(a, at.first(), at.last());
    if constexpr (SPLIT) parts = key_parts(a, kt.n);
    if (SPLIT && (sp >= parts || !at.in(q0 + r / (BQ / a.fold) * (BQ / a.fold)))) return;
    const int t0 = SPLIT ? kt.n * sp / parts : 0, t1 = SPLIT ? kt.n * (sp + 1) / parts : kt.n;
    const int lane = lane_now();
    FragAddr<DP> ad;
    ad.init(lane);
    TileLoad<DP, BK, NW> tk, tv;
    tk.init((int)a.k.st * 2, a.D, wave, lane);
    tv.init((int)a.v.st * 2, a.D, wave, lane);
    const uint16_t* const kp = a.k.p + (PK ? at.krow * a.k.st : b * a.k.sb) + hk * a.k.sh;
    const uint16_t* const vp = a.v.p + (PK ? at.krow * a.v.st : b * a.v.sb) + hk * a.v.sh;
    auto issue = [&](int it, int buf) {
      const int k0 = kt.key0(it), end = kt.end(it, a, len);
      tk.issue(tile_rsrc<BK>(kp, a.k.st, k0, end, a.D), lds, buf * 2 * IMG, wave);
      tv.issue(tile_rsrc<BK>(vp, a.v.st, k0, end, a.D), lds, buf * 2 * IMG + IMG, wave);
    };
    issue(t0, 0);
    u32x4 qf[DP / 16], gf[DP / 16];
    const i32x4 qr = tile_rsrc<32>(a.q.p + (PK ? at.qrow * a.q.st : b * a.q.sb) + hq * a.q.sh, a.q.st, r0 - at.off, at.read(), a.D);
    const i32x4 gr = tile_rsrc<32>(a.go.p + (PK ? at.qrow * a.go.st : b * a.go.sb) + hq * a.go.sh, a.go.st, r0 - at.off, at.read(), a.D);
    const int64_t ldo = (int64_t)a.Hq * a.D, head = ((int64_t)b * a.T + at.qrow) * ldo + (int64_t)hq * a.D;
    const i32x4 orr = tile_rsrc<32>(a.out + head, ldo, r0 - at.off, at.read(), a.D);
    const i32x4 rr = tile_rsrc<32>(a.res + head, ldo, r0 - at.off, at.read(), a.D);
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
    if (PK ? at.in(row) : row < len) nl = -a.lse[(int64_t)bh * a.T + at.qrow + row - at.off];
    wait_vmcnt<0>();
    __syncthreads();
    for (int it = t0; it < t1; ++it) {
      const int img = (it - t0 & 1) * 2 * IMG;
      if (it + 1 < t1) issue(it + 1, it + 1 - t0 & 1);
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
  if (SPLIT && sp >= parts) return;
  sum = sum_halves(sum);
  const int ln = lane_now(), h = ln >> 5, row = r0 + (ln & 31);
  const int64_t line = at.qrow + row - at.off;
  const int64_t ofs = ((int64_t)b * a.T + line) * a.Hq * a.D + (int64_t)hq * a.D;
  const bool in = at.in(row), live = at.live(row);
  if (SPLIT && parts > 1) {
    const int64_t to = part_at(a, sp, line, hq);
    store_f32<DP>(acc, a.part_q + to * a.D, a.D, in, live, h);
    if (in && h == 0) {
      a.ml[to * 2] = sum;
      a.ml[to * 2 + 1] = delta;
    }
    return;
  }
  store_acc<T, DP>(acc, a.scale, a.dq + ofs, a.D, in, live, h);
  if (in && h == 0) {
    // The output's probabilities were rounded, so delta is off by some of its rounding, and the sum of the row's ds, which
    // should be 0, by as much: what k_attn_dkv gets is put right by it (dk of 8 heads of 96, T = 1000: off by 1.42 times
    // its own rounding instead of 1.51).
    float* const p = a.stat + (int64_t)bh * 2 * a.T + line;
    p[0] = PK && !live ? -INFINITY : nl;
    p[a.T] = live ? -(delta + sum) : 0.f;
  }
}

// dq of the rows whose keys were shared, and what k_attn_dkv gets of them.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dq_join(Args a, int pieces) {
  const Joint jt(a, blockIdx.x / pieces);
  if (jt.parts == 1) return;
  jt.each(a, pieces, [&](int row, int64_t line, int d) {
    const bool live = jt.at.live(row);
    f32x4 x = {};
#pragma unroll 16
    for (int sp = 0; sp < jt.parts; ++sp) x += *reinterpret_cast<const f32x4*>(a.part_q + part_at(a, sp, line, jt.hq) * a.D + d);
    u32x2 v;
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = live ? pack2<T>(x[2 * i] * a.scale, x[2 * i + 1] * a.scale) : 0;
    *reinterpret_cast<u32x2*>(a.dq + (line * a.Hq + jt.hq) * a.D + d) = v;
    if (d > 0) return;
    float sum = a.ml[part_at(a, 0, line, jt.hq) * 2 + 1];
    for (int sp = 0; sp < jt.parts; ++sp) sum += a.ml[part_at(a, sp, line, jt.hq) * 2];
    float* const p = a.stat + (int64_t)jt.hq * 2 * a.T + line;
    p[0] = live ? -a.lse[(int64_t)jt.hq * a.T + line] : -INFINITY;
    p[a.T] = live ? -sum : 0.f;
  });
}

// ---------------------------------------------------------------------------------------------------------- dk, dv
// The block of BKV keys that a workgroup takes, and the row tiles of the sequence whose rows may see one of its keys: nt
// from t0 on (by place among the sequence's rows of q, `off` less than their positions).
template <bool PK>
struct Keys {
  int kb0, len, off, own, t0, nt;
  bool skip;            // packed: no block of this unit, or one of those with first tokens among the others (or the reverse)
  int64_t qrow, krow;
  // blk: the block among those with first tokens, or among the others
  __device__ __forceinline__ Keys(const Args& a, int b, bool sink, int blk) {
    if constexpr (PK) {
      if (sink && a.by_key) {
        const Unit x = unit_at<true>(a, blk);
        set(a, x, true);
        skip |= x.blk >= a.n_sb || x.outside;
      } else if (sink) {
        Unit x = unit_of<true>(a, 1 + blk / a.n_sb, 0);
        x.blk = blk % a.n_sb;
        set(a, x, true);
      } else {
        set(a, unit_at<true>(a, blk), false);
      }
    } else {
      skip = false;
      kb0 = (sink ? blk : a.n_sb + blk) * BKV;
      len = seq_len(a, b);
      off = 0;
      own = a.T;
      qrow = krow = 0;
      t0 = kb0 / BR;
      nt = (end_row(a) + BR - 1) / BR - t0;
    }
  }
  __device__ __forceinline__ Keys(const Args& a, const Unit& x) { set(a, x, false); }
  __device__ __forceinline__ void set(const Args& a, const Unit& x, bool sink) {
    own = x.lq;
    len = x.lk;
    off = len - own;
    qrow = x.q0;
    krow = x.k0;
    kb0 = x.blk * BKV;
    skip = x.blk < 0 || kb0 >= len || (!sink && x.blk < a.n_sb && !x.outside);
    const int first = kb0 - off, end = end_row(a) - off;
    t0 = (first < 0 ? 0 : first) / BR;
    nt = (end + BR - 1) / BR - t0;
    nt = end <= 0 || nt < 0 ? 0 : nt;
  }
  // rows kb0 .. end_row - 1 may see a key of the block
  __device__ __forceinline__ int end_row(const Args& a) const {
    const int64_t end = kb0 < a.sinks ? len : (int64_t)kb0 + BKV - 1 + a.window;
    return end < len ? (int)end : len;
  }
  __device__ __forceinline__ int read() const { return PK ? own : len; }
  // workgroups that share the block
  __device__ __forceinline__ int parts(const Args& a, int S) const {
    if constexpr (!PK) return S;
    const int n = (int)(((int64_t)nt * a.grp + MIN_PACK - 1) / MIN_PACK);
    return n < 1 ? 1 : (n < S ? n : S);
  }
};

// dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij go_i over the rows of all query heads that share the head: keys stay in
// registers, 32 per wave, and row tiles pass through a ring of NS. Scores and go v are formed a second time (seven
// products in the backward for the formula's five), which needs neither atomics nor ds in memory.
// Packed sequences: the host does not know how long the blocks are, so S is what the workspace has room for, and a block
// is shared by no more workgroups than get MIN_PACK row tiles each; one that is not shared is written at once.
// Measured (bf16, D = 128): 4 x 16384 tokens of 16 heads over 4, window 1024: 1.24 ms, 0.86 PFLOP/s of visible pairs (8 D
// each), matrix core busy 45% of the time; the join of the first tokens' blocks 7 us.
template <typename T, int DP, bool PK>
__global__ __launch_bounds__(THREADS, 2) void k_attn_dkv(Args a) {
  constexpr int IMG = BR * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[NS * 2 * IMG];   // Q and go of the ring's tiles
  __shared__ __attribute__((aligned(256))) float stats[NS][2][BR];    // -lse and -delta of their rows
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nsink = PK ? a.us : a.n_sb, nr = PK ? a.uk : (a.T + BKV - 1) / BKV - a.n_sb;
  // workgroups of the blocks with first tokens (the longest) first, then the others, those with the most rows first
  const uint32_t heads = (uint32_t)a.B * a.Hkv, sink_wgs = heads * nsink * a.S_s;
  const bool sink = blockIdx.x < sink_wgs;
  const uint32_t w = sink ? blockIdx.x : blockIdx.x - sink_wgs;
  const int S = sink ? a.S_s : a.S_r, nb = sink ? nsink : nr;
  const Place pl(a, w, nb * S, 1, PK && a.plan != nullptr && !sink);
  // Packed: the parts that are not used come last. Between the others they left those on few CUs (52 sequences of 339
  // tokens, 12 heads, window 44 and a first token: 223 us, 127 so).
  const int sp = PK ? pl.blk / nb : pl.blk % S, blk = PK ? pl.blk % nb : pl.blk / S, b = pl.b, hk = pl.hk, bh = b * a.Hkv + hk;
  const Keys<PK> at(a, b, sink, blk);
  const int len = at.len, kb0 = at.kb0, j0 = kb0 + wave * 32;
  const int parts = at.parts(a, S);
  if (PK && (at.skip || sp >= parts)) return;
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const float c = a.scale * LOG2E;
  int it0 = 0, it1 = 0;
  if (kb0 < len) {
    const int t0 = at.t0, nt = at.nt, total = nt * a.grp;
    it0 = (int)((int64_t)total * sp / parts);
    it1 = (int)((int64_t)total * (sp + 1) / parts);
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
      const int64_t qo = PK ? at.qrow * a.q.st : b * a.q.sb, go = PK ? at.qrow * a.go.st : b * a.go.sb;
      tq.issue(tile_rsrc<BR>(a.q.p + qo + hq * a.q.sh, a.q.st, i0, at.read(), a.D), lds, buf * 2 * IMG, wave);
      tg.issue(tile_rsrc<BR>(a.go.p + go + hq * a.go.sh, a.go.st, i0, at.read(), a.D), lds, buf * 2 * IMG + IMG, wave);
      const int own = PK ? at.own : a.T, rows = own - i0 < BR ? own - i0 : BR;
      const int ln = lane_now();
      dma4(make_rsrc(a.stat + ((int64_t)b * a.Hq + hq) * 2 * a.T + at.qrow + i0, (a.T + rows) * 4),
           reinterpret_cast<const char*>(&stats[0][0][0]), buf * 2 * BR * 4,
           (ln & 31) < rows ? ((ln & 31) + (ln >> 5) * a.T) * 4 : OOB);
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
      if (it0 + i < it1) issue(it0 + i);
    u32x4 kf[DP / 16], vf[DP / 16];
    const i32x4 kr = tile_rsrc<32>(a.k.p + (PK ? at.krow * a.k.st : b * a.k.sb) + hk * a.k.sh, a.k.st, j0, len, a.D);
    const i32x4 vr = tile_rsrc<32>(a.v.p + (PK ? at.krow * a.v.st : b * a.v.sb) + hk * a.v.sh, a.v.st, j0, len, a.D);
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
      const int i0 = (t0 + it % nt) * BR + at.off;   // position of the tile's first row
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
  const bool in = key < (PK ? len : a.T), live = key < len;
  if (PK ? parts == 1 : S == 1) {
    const int64_t ofs = (((int64_t)b * a.T + at.krow + key) * a.Hkv + hk) * a.D;
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
template <typename T, bool PK>
__global__ __launch_bounds__(256) void k_attn_dkv_join(Args a, int pieces) {
  const int nsink = PK ? a.us : a.n_sb, nr = PK ? a.uk : (a.T + BKV - 1) / BKV - a.n_sb;
  const uint32_t heads = (uint32_t)a.B * a.Hkv, sink_blocks = a.S_s > 1 ? heads * nsink : 0;
  uint32_t w = blockIdx.x / pieces;
  const bool sink = w < sink_blocks;
  if (!sink) w -= sink_blocks;
  const int S = sink ? a.S_s : a.S_r, nb = sink ? nsink : nr;
  const int blk = w % nb, bh = w / nb, b = bh / a.Hkv, hk = bh % a.Hkv;
  int kb0 = 0, rows = a.T, parts = S;
  int64_t krow = 0;
  if constexpr (PK) {
    const Keys<true> at(a, 0, sink, blk);
    parts = at.parts(a, S);
    if (at.skip || parts == 1) return;
    kb0 = at.kb0;
    rows = at.len;
    krow = at.krow;
  } else {
    kb0 = (sink ? blk : a.n_sb + blk) * BKV;
  }
  const int cols = a.D / 4;
  for (int i = blockIdx.x % pieces * 256 + threadIdx.x;; i += pieces * 256) {
    const int which = i / (BKV * cols), r = i / cols % BKV, d = i % cols * 4, key = kb0 + r;
    if (which > 1) return;
    if (key >= rows) {
      if (PK) continue;
      return;                                             // (pieces for all)
    }
    const float* const p = (sink ? a.part_s : a.part_r) + ((((int64_t)bh * nb + blk) * S * 2 + which) * BKV + r) * a.D + d;
    f32x4 x = {};
#pragma unroll 4
    for (int sp = 0; sp < parts; ++sp) x += *reinterpret_cast<const f32x4*>(p + (int64_t)sp * 2 * BKV * a.D);
    if (which == 0) x *= a.scale;
    u32x2 v;
    v[0] = pack2<T>(x[0], x[1]);
    v[1] = pack2<T>(x[2], x[3]);
    *reinterpret_cast<u32x2*>((which ? a.dv : a.dk) + (((int64_t)b * a.T + krow + key) * a.Hkv + hk) * a.D + d) = v;
    if (!PK) return;
  }
}

}  // namespace

#endif  // MEMARCH_ATTN_KERNELS_H
