// seq_find.h — which sequence a unit of work belongs to, and which keys the last token of a sequence sees: shared by the
// kernels over packed sequences and over paged caches (gfx950).
#ifndef MEMARCH_SEQ_FIND_H
#define MEMARCH_SEQ_FIND_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace attn {

// The last i of 0 .. n - 1 with first(i) <= u, where first(0) <= u and first does not fall: all 64 lanes look at once.
// (Where it falls all the same, some i.)
template <typename F>
__device__ __forceinline__ int last_from(int n, int u, F first) {
  const int lane = threadIdx.x & 63;
  int at = 0, step = 1;
  while (step * 64 < n) step *= 64;
  for (;; step /= 64) {
    const int i = at + lane * step;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && first(i) <= u));
    at += (c > 0 ? c - 1 : 0) * step;
    if (step == 1) return __builtin_amdgcn_readfirstlane(at);
  }
}

// Entry i of the starts of packed sequences, in 0 .. rows.
__device__ __forceinline__ int start_in(const int32_t* cu, int i, int rows) {
  const int x = cu[i];
  return x < 0 ? 0 : (x > rows ? rows : x);
}

// The tiles of BK keys that the last of a sequence's n tokens sees: those of the first `sinks` positions, then those of
// the window. A: kernel arguments with lengths, max_pages, page, window and sinks.
template <int BK>
struct Seen {
  int n, lo, n_sink, lo_tile, tiles;
  template <typename A>
  __device__ __forceinline__ Seen(const A& a, int b) {
    n = a.lengths[b];
    const int64_t cap = (int64_t)a.max_pages * a.page;
    n = n < 0 ? 0 : (n > cap ? (int)cap : n);
    lo = n - a.window;
    lo = lo < 0 ? 0 : lo;
    lo_tile = lo / BK;
    n_sink = (a.sinks + BK - 1) / BK;
    n_sink = n_sink < lo_tile ? n_sink : lo_tile;
    tiles = n_sink + (n + BK - 1) / BK - lo_tile;
  }
  __device__ __forceinline__ int key0(int it) const { return (it < n_sink ? it : lo_tile + it - n_sink) * BK; }
  // tiles per workgroup when they are shared among S, a multiple of its NW waves and at least `least`
  template <int NW>
  __device__ __forceinline__ int run(int S, int least) const {
    const int r = ((tiles + S - 1) / S + NW - 1) / NW * NW;
    return r < least ? least : r;
  }
};

}  // namespace attn

#endif  // MEMARCH_SEQ_FIND_H
