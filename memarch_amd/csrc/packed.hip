// packed.hip — causal attention over packed sequences, forward and backward, for MI355X (gfx950): the order of the work and
// the host side. The C ABI is in include/mce_pack.h, the attention's kernels in attn_kernels.h (PK).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mce_pack.h"
#include "attn_host.h"
#include "attn_kernels.h"

namespace {

using namespace attn;

// The units of packed sequences in the order in which they are taken, so that no long one is left over at the end (few queries
// behind many keys, 8 pieces of 8192 rows over 139264 keys, 16 heads: 1206 us in their own order, half of the workgroups gone
// from 60% of the time on; 1147 in this). Without a window: the sequences with the most keys first, each one's
// blocks together, from the longest on, as they share keys (taken by their own lengths from everywhere, 16 prompts of up to
// 7491 tokens read all keys from HBM: 1531 us, 1466 so). With a window: the longest blocks first,
// few of which are shorter than the others and fill the end. Counting sorts by length in steps of 1/16, one workgroup for
// the units of q and one for those of k; which of two alike comes first is open, and no result hangs on it.
constexpr int PLAN_THREADS = 1024;
template <bool KEYS>
__device__ __forceinline__ void plan_units(const Args& a) {
  constexpr int BLK = KEYS ? BKV : BQ, BUCKETS = 512;
  __shared__ int count[BUCKETS], wsum[PLAN_THREADS / 64];
  const int t = threadIdx.x, n = KEYS ? a.uk : a.uq, rows = KEYS ? a.M : a.T, seqs = a.nseq + 2;
  const int32_t* const cu = KEYS ? a.cu_k : a.cu;
  Unit* const out = a.plan + (KEYS ? a.uq : 0);
  int* const place = reinterpret_cast<int*>(a.plan + a.uq + a.uk) + (KEYS ? seqs : 0);   // a sequence's first unit
  const bool whole = a.window == INT32_MAX;
  auto find = [&](int u, int* s) {
    int lo = 0, hi = seqs;                             // the last s with its first unit not behind u
    while (hi - lo > 1) {
      const int m = (lo + hi) / 2;
      if (start_of(cu, a.nseq, rows, m) / BLK + m <= u) lo = m;
      else hi = m;
    }
    *s = lo;
    return unit_of<KEYS>(a, lo, u);
  };
  auto blocks = [&](const Unit& x) { return ((KEYS ? x.lk : x.lq) + BLK - 1) / BLK; };
  // 0: the longest; exponent and four bits behind it (lengths are below 2^28)
  auto bucket = [&](int len) {
    const int b = (int)(__builtin_bit_cast(uint32_t, (float)len) >> 19) - (127 << 4);
    return BUCKETS - 1 - (b < 0 ? 0 : b);
  };
  auto tiles = [&](const Unit& x) {
    if constexpr (KEYS) {
      const Keys<true> at(a, x);
      return at.skip ? 0 : at.nt + 1;
    } else {
      const Rows<true> at(x);
      return at.any() ? KeyTiles(a, at.first(), at.last()).n + 1 : 1;
    }
  };
  for (int i = t; i < BUCKETS; i += PLAN_THREADS) count[i] = 0;
  // units that are left over have no block (nor those that nobody writes where starts fall)
  for (int u = t; u < n; u += PLAN_THREADS) {
    Unit x = {};
    x.blk = -1;
    out[u] = x;
  }
  __syncthreads();
  if (whole) {
    for (int s = t; s < seqs; s += PLAN_THREADS) {
      const Unit x = unit_of<KEYS>(a, s, 0);
      atomicAdd(&count[bucket(KEYS ? x.lq : x.lk)], blocks(x));
    }
  } else {
    for (int u = t, s; u < n; u += PLAN_THREADS) {
      const Unit x = find(u, &s);
      if (x.blk < blocks(x)) atomicAdd(&count[bucket(tiles(x))], 1);
    }
  }
  __syncthreads();
  const int own = t < BUCKETS ? count[t] : 0;
  int sum = own;
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(sum, o);
    sum += (t & 63) >= o ? up : 0;
  }
  if ((t & 63) == 63) wsum[t >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < t >> 6; ++w) sum += wsum[w];
  if (t < BUCKETS) count[t] = sum - own;
  __syncthreads();
  if (whole) {
    for (int s = t; s < seqs; s += PLAN_THREADS) {
      const Unit x = unit_of<KEYS>(a, s, 0);
      place[s] = atomicAdd(&count[bucket(KEYS ? x.lq : x.lk)], blocks(x));
    }
    __syncthreads();
  }
  for (int u = t, s; u < n; u += PLAN_THREADS) {
    const Unit x = find(u, &s);
    const int nb = blocks(x);
    if (x.blk < 0 || x.blk >= nb) continue;
    const int to = whole ? place[s] + (KEYS ? x.blk : nb - 1 - x.blk) : atomicAdd(&count[bucket(tiles(x))], 1);
    if ((unsigned)to < (unsigned)n) out[to] = x;       // (more than n blocks: where starts fall)
  }
}
__global__ __launch_bounds__(PLAN_THREADS) void k_attn_plan(Args a) {
  if (blockIdx.x == 0) plan_units<false>(a);
  else plan_units<true>(a);
}

// -------------------------------------------------------------------------------------------------------- host side
constexpr int64_t MAX_ROWS = int64_t(1) << 27;

struct Plan {
  int64_t uq, uk;           // units of rows of q and of keys
  int64_t us;               // units of key blocks with first tokens
  int n_sb, S_s, S_r;
  int64_t part_s, part_r;   // floats of the parts
  int fold, S_q;
  int64_t part_q;           // rows of the parts of the rows' sums
};

// How many workgroups may share a key block's rows (the kernels use fewer where its rows are few). Lengths are not known
// here: key blocks are shared where there are too few of them to fill the GPU, blocks with first tokens of windowed
// sequences, which every later row sees, until there are 2048 workgroups for them. Those are taken as the first n_sb of each
// sequence, or, where that is more than all units of keys (many sequences that cannot all be so long), found among the units.
Plan make_plan(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks) {
  Plan p = {N / BQ + nseq + 2, M / BKV + nseq + 2, 0, 0, 1, 1, 0, 0, 1, 1, 0};
  // parts that a block can have when it sees n rows
  auto most_parts = [&](int64_t n) { return ((n + BR - 1) / BR * (Hq / Hkv) + MIN_PACK - 1) / MIN_PACK; };
  const bool windowed = window > 0 && window < M;
  if (windowed && sinks > 0) {
    const int64_t most = M / BKV + 1, n = (sinks + BKV - 1) / BKV;
    p.n_sb = (int)(n < most ? n : most);
    p.us = std::min(nseq * p.n_sb, p.uk);
    const int64_t units = p.us * Hkv;
    const int64_t s = units > 0 ? (2048 + units - 1) / units : 1;
    p.S_s = (int)std::clamp(std::min(s, most_parts(N)), int64_t(1), int64_t(64));
  }
  const int64_t s = (768 + p.uk * Hkv - 1) / (p.uk * Hkv);
  const int64_t rows = windowed && window + BKV + BR < N ? window + BKV + BR : N;
  p.S_r = (int)std::clamp(std::min(s, most_parts(rows)), int64_t(1), int64_t(16));
  p.part_s = p.S_s > 1 ? p.us * Hkv * p.S_s * 2 * BKV * D : 0;
  p.part_r = p.S_r > 1 ? p.uk * Hkv * p.S_r * 2 * BKV * D : 0;
  // Few rows: the keys of a block are shared where the workgroups are not half of the 512 that run at once, and a block of
  // the mean saves 16 tiles, as the parts and their launch take the time of about 8 (one sequence of 2048 tokens, 8 heads:
  // 43 us alone and 45 shared; 4096 tokens, 4 heads: 61 and 42; 4 x 16 rows behind 16384 keys: 293 and 46). Long blocks are cut
  // finer, into parts of 32 tiles (1500 rows behind 131072 keys: 1920 us in two parts, 1710 so); more than 64 take longer to
  // join than they save (1 row behind 131072 keys, 16 heads over 4: 95 us with 32, 66 with 64, 97 with 128).
  p.fold = Hq / Hkv % 4 == 0 ? 4 : (Hq / Hkv % 2 == 0 ? 2 : 1);
  const int64_t keys = windowed && window + sinks + BQ < M ? window + sinks + BQ : M, tiles = keys / BK;
  const int64_t blocks = (N * p.fold / BQ + nseq) * (Hq / p.fold);
  if (N > 0 && nseq > 0 && blocks <= 256) {
    const int64_t mean = std::min(keys, M / nseq - N / nseq / 2);
    const int64_t fill = std::min(512 / blocks, tiles / MIN_KEYS), fine = std::min(1024 / blocks, mean / (32 * BK));
    const int64_t S = std::min(std::max(fill, fine), int64_t(64));
    if (mean * (S - 1) >= 16 * BK * S) p.S_q = (int)S;
  }
  p.part_q = p.S_q > 1 ? p.S_q * N * Hq : 0;
  return p;
}

int check_sizes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks) {
  if (nseq < 0 || N < 0 || M < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 8 || D > 128 || D % 8 || window < 0 || sinks < 0)
    return MCE_ATTN_EINVAL;
  if (N > MAX_ROWS || M > MAX_ROWS || nseq > MAX_GROUPS || Hq * D > MAX_ST) return MCE_ATTN_EINVAL;
  const Plan p = make_plan(nseq, N, M, Hq, Hkv, D, window, sinks);
  // the products are below 2^63: sinks' blocks are at most M / BKV + 1 per sequence
  if (p.uq > MAX_GROUPS / Hq || p.uk * p.S_r > MAX_GROUPS / Hkv || nseq * p.n_sb > INT32_MAX ||
      p.us * p.S_s > MAX_GROUPS / Hkv - p.uk * p.S_r)
    return MCE_ATTN_EINVAL;
  return MCE_ATTN_OK;
}

Args make_args(Strided q, Strided k, Strided v, const int32_t* cu, const int32_t* cu_k, int64_t nseq, int64_t N, int64_t M,
               int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks, float scale, const Plan& p) {
  Args a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.cu = cu;
  a.cu_k = cu_k == nullptr ? cu : cu_k;
  a.nseq = (int)nseq;
  a.B = 1;
  a.T = (int)N;
  a.M = (int)M;
  a.uq = (int)p.uq;
  a.uk = (int)p.uk;
  a.us = (int)p.us;
  a.by_key = p.us < nseq * p.n_sb;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.D = (int)D;
  a.window = window == 0 || window >= M ? INT32_MAX : (int)window;
  a.sinks = a.window == INT32_MAX ? 0 : (int)(sinks > M ? M : sinks);
  a.n_sb = p.n_sb;
  a.S_s = p.S_s;
  a.S_r = p.S_r;
  a.S_q = p.S_q;
  a.fold = p.fold;
  a.thin = N <= nseq * (BQ / p.fold);
  a.scale = scale;
  return a;
}

// Bytes of the plan: none where all workgroups of the forward run at once, and with sequences below 1024 tokens on average.
// Steps in their own order and with the plan, whose kernel takes 7 us of it, in us: 49999 tokens, 16 heads over 4, D = 64, window
// 1024, mean 4096: 1289 and 1214, 1365: 1071 and 974; 32768 tokens, 16 heads, D = 128, no window, mean 1365: 1406 and 1412. Below
// the line it pays too where workgroups are many (65536 tokens, 16 heads over 4, D = 128, no window, mean 256: 1201 and 1143; 64:
// 1184 and 1078), and not where they are few or short (the forward alone of 65536 tokens, 8 heads over 2, D = 64, window 128, mean
// 512: 61 and 66; of 8192, 16 over 4, window 64, mean 256: 22 and 26).
int64_t plan_bytes_of(const Plan& p, int64_t nseq, int64_t M, int64_t Hq) {
  const int64_t seqs = nseq + 2;
  return p.uq * Hq <= 512 || p.S_q > 1 || M < 1024 * nseq ? 0 : (p.uq + p.uk) * (int64_t)sizeof(Unit) + 8 * seqs;
}

// Bytes of the parts of the rows' sums, and of the two numbers of each.
int64_t sums_bytes(const Plan& p, int64_t D) { return align256(p.part_q * D * 4); }
int64_t split_bytes(const Plan& p, int64_t D) { return sums_bytes(p, D) + align256(p.part_q * 8); }
unsigned split_grid(const Args& a) { return ((unsigned)(a.Hkv * a.uq * a.S_q) + 7) / 8 * 8 * a.grp; }
constexpr int JOIN_PIECES = 4;   // workgroups per block of rows that join parts

template <typename T, int DP>
int launch_fwd(const Args& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.Hq * a.uq)), joins((unsigned)(a.Hq * a.uq * JOIN_PIECES));
  if (a.S_q > 1) {
    hipLaunchKernelGGL((k_attn_fwd<T, DP, true, true>), dim3(split_grid(a)), dim3(THREADS), 0, st, a);
    hipLaunchKernelGGL((k_attn_fwd_join<T>), joins, dim3(256), 0, st, a, JOIN_PIECES);
    return finish();
  }
  if (a.plan != nullptr) {
    hipLaunchKernelGGL(k_attn_plan, dim3(a.r != nullptr ? 2 : 1), dim3(PLAN_THREADS), 0, st, a);
    const int rc = finish();
    if (rc) return rc;
  }
  hipLaunchKernelGGL((k_attn_fwd<T, DP, true, false>), grid, dim3(THREADS), 0, st, a);
  return finish();
}

template <typename T, int DP>
int launch_bwd(const Args& a, hipStream_t st) {
  if (a.T > 0) {
    const dim3 grid((unsigned)(a.Hq * a.uq)), joins((unsigned)(a.Hq * a.uq * JOIN_PIECES));
    if (a.S_q > 1) {
      hipLaunchKernelGGL((k_attn_dq<T, DP, true, true>), dim3(split_grid(a)), dim3(THREADS), 0, st, a);
      hipLaunchKernelGGL((k_attn_dq_join<T>), joins, dim3(256), 0, st, a, JOIN_PIECES);
    } else {
      hipLaunchKernelGGL((k_attn_dq<T, DP, true, false>), grid, dim3(THREADS), 0, st, a);
    }
    const int rc = finish();
    if (rc) return rc;
  }
  if (a.M == 0) return MCE_ATTN_OK;
  hipLaunchKernelGGL((k_attn_dkv<T, DP, true>), dim3((unsigned)(a.Hkv * ((int64_t)a.us * a.S_s + (int64_t)a.uk * a.S_r))),
                     dim3(THREADS), 0, st, a);
  const int64_t join = a.Hkv * ((a.S_s > 1 ? (int64_t)a.us : 0) + (a.S_r > 1 ? (int64_t)a.uk : 0));
  // few blocks need many threads each; of many most are not shared, and a workgroup that only finds that out costs 1 ns
  const int64_t all = (2 * BKV * (a.D / 4) + 255) / 256;
  const int pieces = (int)std::clamp(4096 / std::max(join, int64_t(1)), int64_t(1), all);
  if (join > 0)
    hipLaunchKernelGGL((k_attn_dkv_join<T, true>), dim3((unsigned)(join * pieces)), dim3(256), 0, st, a, pieces);
  return finish();
}

}  // namespace

thread_local int mce_attn_hip_error = 0;

extern "C" {

const char* mce_serve_error_string(int code) {
  switch (code) {
    case MCE_ATTN_OK: return "ok";
    case MCE_ATTN_EINVAL: return "invalid argument (size, stride, head count, scale, element type or null pointer)";
    case MCE_ATTN_EALIGN: return "misaligned (a pointer or a stride)";
    case MCE_ATTN_EWORKSPACE: return "workspace missing, too small or not 256-byte aligned";
    case MCE_ATTN_ELAUNCH: return "a HIP launch failed";
    default: return "unknown error";
  }
}

int mce_serve_last_hip_error(void) { return mce_attn_hip_error; }

int mce_pack_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                 int64_t v_st, int64_t v_sh, const int32_t* cu, const int32_t* cu_k, int64_t nseq, int64_t N, int64_t M,
                 int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t sinks, float scale, int dtype, void* out,
                 void* res, float* lse, void* plan, size_t plan_bytes, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_sizes(nseq, N, M, Hq, Hkv, D, window, sinks);
  if (rc) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16) || (cu_k == nullptr && N != M))
    return MCE_ATTN_EINVAL;
  if (N == 0) return MCE_ATTN_OK;
  if (cu == nullptr || out == nullptr || (rc = check_strided(q, 0, q_st, q_sh, D))) return rc ? rc : MCE_ATTN_EINVAL;
  if (M > 0 && ((rc = check_strided(k, 0, k_st, k_sh, D)) || (rc = check_strided(v, 0, v_st, v_sh, D)))) return rc;
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(res)) & 15) return MCE_ATTN_EALIGN;
  const Plan p = make_plan(nseq, N, M, Hq, Hkv, D, window, sinks);
  const int64_t need = plan_bytes_of(p, nseq, M, Hq);
  if (need > 0 && (plan == nullptr || (reinterpret_cast<uintptr_t>(plan) & 255) || plan_bytes < (size_t)need))
    return MCE_ATTN_EWORKSPACE;
  const int64_t split = split_bytes(p, D);
  if (split > 0 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < (size_t)split))
    return MCE_ATTN_EWORKSPACE;
  Args a = make_args({static_cast<const uint16_t*>(q), 0, q_st, q_sh}, {static_cast<const uint16_t*>(k), 0, k_st, k_sh},
                     {static_cast<const uint16_t*>(v), 0, v_st, v_sh}, cu, cu_k, nseq, N, M, Hq, Hkv, D, window, sinks,
                     scale, p);
  a.plan = need > 0 ? static_cast<Unit*>(plan) : nullptr;
  a.o = static_cast<uint16_t*>(out);
  a.r = static_cast<uint16_t*>(res);
  a.lse = lse;
  a.part_q = static_cast<float*>(ws);
  a.ml = split > 0 ? a.part_q + sums_bytes(p, D) / 4 : nullptr;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_fwd<__bf16, 64>(a, st) : launch_fwd<__bf16, 128>(a, st);
  return D <= 64 ? launch_fwd<_Float16, 64>(a, st) : launch_fwd<_Float16, 128>(a, st);
}

size_t mce_pack_plan_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                           int64_t sinks) {
  if (check_sizes(nseq, N, M, Hq, Hkv, D, window, sinks) || N == 0) return 0;
  return (size_t)plan_bytes_of(make_plan(nseq, N, M, Hq, Hkv, D, window, sinks), nseq, M, Hq);
}

size_t mce_pack_fwd_ws_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                             int64_t sinks) {
  if (check_sizes(nseq, N, M, Hq, Hkv, D, window, sinks)) return 0;
  return (size_t)split_bytes(make_plan(nseq, N, M, Hq, Hkv, D, window, sinks), D);
}

size_t mce_pack_bwd_ws_bytes(int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                             int64_t sinks) {
  if (check_sizes(nseq, N, M, Hq, Hkv, D, window, sinks)) return 0;
  const Plan p = make_plan(nseq, N, M, Hq, Hkv, D, window, sinks);
  return (size_t)(align256(N * Hq * 8) + align256(p.part_s * 4) + align256(p.part_r * 4) + split_bytes(p, D));
}

int mce_pack_bwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                 int64_t v_st, int64_t v_sh, const void* go, int64_t go_st, int64_t go_sh, const int32_t* cu,
                 const int32_t* cu_k, int64_t nseq, int64_t N, int64_t M, int64_t Hq, int64_t Hkv, int64_t D,
                 int64_t window, int64_t sinks, float scale, int dtype, const void* out, const void* res,
                 const float* lse, const void* plan, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes,
                 void* stream) {
  int rc = check_sizes(nseq, N, M, Hq, Hkv, D, window, sinks);
  if (rc) return rc;
  if (!good_scale(scale) || (dtype != MCE_ATTN_BF16 && dtype != MCE_ATTN_F16) || (cu_k == nullptr && N != M))
    return MCE_ATTN_EINVAL;
  if (N == 0 && M == 0) return MCE_ATTN_OK;
  if (cu == nullptr) return MCE_ATTN_EINVAL;
  if (N > 0) {
    if ((rc = check_strided(q, 0, q_st, q_sh, D)) || (rc = check_strided(go, 0, go_st, go_sh, D))) return rc;
    if (out == nullptr || res == nullptr || lse == nullptr || dq == nullptr) return MCE_ATTN_EINVAL;
  }
  if (M > 0) {
    if ((rc = check_strided(k, 0, k_st, k_sh, D)) || (rc = check_strided(v, 0, v_st, v_sh, D))) return rc;
    if (dk == nullptr || dv == nullptr) return MCE_ATTN_EINVAL;
  }
  for (const void* p : {out, res, (const void*)dq, (const void*)dk, (const void*)dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return MCE_ATTN_EALIGN;
  const Plan p = make_plan(nseq, N, M, Hq, Hkv, D, window, sinks);
  const bool planned = N > 0 && plan_bytes_of(p, nseq, M, Hq) > 0;
  if (planned && (plan == nullptr || (reinterpret_cast<uintptr_t>(plan) & 255))) return MCE_ATTN_EWORKSPACE;
  const int64_t stat = align256(N * Hq * 8), part_s = align256(p.part_s * 4), part_r = align256(p.part_r * 4);
  const int64_t all = stat + part_s + part_r + split_bytes(p, D);
  if (all > 0 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) ||
                  ws_bytes < (size_t)all))
    return MCE_ATTN_EWORKSPACE;
  Args a = make_args({static_cast<const uint16_t*>(q), 0, q_st, q_sh}, {static_cast<const uint16_t*>(k), 0, k_st, k_sh},
                     {static_cast<const uint16_t*>(v), 0, v_st, v_sh}, cu, cu_k, nseq, N, M, Hq, Hkv, D, window, sinks,
                     scale, p);
  a.plan = planned ? static_cast<Unit*>(const_cast<void*>(plan)) : nullptr;
  a.go = {static_cast<const uint16_t*>(go), 0, go_st, go_sh};
  a.out = static_cast<const uint16_t*>(out);
  a.res = static_cast<const uint16_t*>(res);
  a.lse = const_cast<float*>(lse);
  a.stat = static_cast<float*>(ws);
  a.part_s = a.stat + stat / 4;
  a.part_r = a.part_s + part_s / 4;
  a.part_q = a.part_r + part_r / 4;
  a.ml = a.part_q + sums_bytes(p, D) / 4;
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MCE_ATTN_BF16) return D <= 64 ? launch_bwd<__bf16, 64>(a, st) : launch_bwd<__bf16, 128>(a, st);
  return D <= 64 ? launch_bwd<_Float16, 64>(a, st) : launch_bwd<_Float16, 128>(a, st);
}

}  // extern "C"
