// attn.hip — causal attention over a sliding window with first tokens that stay visible, forward and backward, for
// MI355X (gfx950): the host side over a padded batch. The C ABI is in include/mce_attn.h, the kernels in attn_kernels.h.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mce_attn.h"
#include "attn_host.h"
#include "attn_kernels.h"

namespace {

using namespace attn;

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
  hipLaunchKernelGGL((k_attn_fwd<T, DP, false, false>), dim3(n), dim3(THREADS), 0, st, a);
  return finish();
}

// How many workgroups share a key block's rows in k_attn_dkv. Lengths are not known to the host: T stands for all.
struct Plan {
  int n_sb, S_s, S_r;
  int64_t part_s, part_r;   // floats of the parts
};
constexpr int64_t SLOTS = 512;    // workgroups of k_attn_dkv that run at once
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
  hipLaunchKernelGGL((k_attn_dq<T, DP, false, false>), dim3(n), dim3(THREADS), 0, st, a);
  const int64_t heads = (int64_t)a.B * a.Hkv, nr = (a.T + BKV - 1) / BKV - a.n_sb;
  hipLaunchKernelGGL((k_attn_dkv<T, DP, false>), dim3((unsigned)(heads * (a.n_sb * a.S_s + nr * a.S_r))), dim3(THREADS), 0, st,
                     a);
  const int64_t join = heads * ((a.S_s > 1 ? a.n_sb : 0) + (a.S_r > 1 ? nr : 0));
  const int pieces = (2 * BKV * (a.D / 4) + 255) / 256;
  if (join > 0) hipLaunchKernelGGL((k_attn_dkv_join<T, false>), dim3((unsigned)(join * pieces)), dim3(256), 0, st, a, pieces);
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
