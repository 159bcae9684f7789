// C ABI of the windowed attention over dense keys (declared in include/fas.h).
//
// Validates a request, packs the kernel parameter blocks and enqueues the
// launches on the caller's stream.  No device memory is allocated here and
// nothing is synchronised.
#include "fas.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "fas_check.hpp"
#include "fas_launch.hpp"
#include "fas_params.hpp"
#include "fas_rows_plan.hpp"

namespace {

using fas::align256;
using fas::check_tensor;
using fas::fail;
using fas::hip_status;
using fas::kCus;
using fas::Problem;
using fas::slice_bytes;

int check_window(const char* fn, const fas_attn_args* a, int64_t window, int64_t sinks, Problem* pr) {
  int rc;
  if ((rc = fas::check_shape(fn, a, pr))) return rc;
  if (!pr->causal) return fail(FAS_ERR_INVALID, fn, "causal must be 1: a window looks back");
  if (pr->dropout) return fail(FAS_ERR_UNSUPPORTED, fn, "no dropout");
  if (window < 1 || sinks < 0)
    return fail(FAS_ERR_INVALID, fn, "window must be at least 1 and sinks not negative");
  if ((int64_t)pr->G * pr->M > (1 << 28))
    return fail(FAS_ERR_UNSUPPORTED, fn, "sizes exceed the index range of the kernels");
  return FAS_OK;
}

fas::RowsSplit fwd_split(const Problem& pr, int64_t window, int64_t sinks) {
  const int64_t rows = (int64_t)pr.G * pr.M;
  return fas::rows_split(pr.B, (int64_t)pr.B * pr.Hk, rows, pr.M, pr.N, window, sinks, pr.D,
                         rows <= fas::kFewRows, false);
}

// How the dK/dV kernel's row tiles (64 rows, G heads) are dealt, and its
// workspace.  One workgroup a CU runs at D = 128, two below.  Whole key blocks
// end with the longest, or with whole rounds; equal runs of the list of units
// cost about four more a workgroup (K and V again, and parts written) and 8 us
// for the parts' sum.  The cheaper end is taken.
struct BwdPlan {
  int64_t mpad, nkb, wgs, chunk, head_units;
  size_t delta, part, total;
};
BwdPlan bwd_plan(const Problem& pr, int64_t window, int64_t sinks) {
  BwdPlan w{};
  const int64_t bk = fas::kBwdBlock, heads = (int64_t)pr.B * pr.Hk;
  w.mpad = (pr.M + bk - 1) / bk * bk;
  w.nkb = (pr.N + bk - 1) / bk;
  int64_t longest = 0;
  for (int64_t kb = 0; kb < w.nkb; ++kb) {
    const int64_t off = (int64_t)pr.N - pr.M, k0 = kb * bk;
    const int64_t lo = std::max<int64_t>(0, k0 - off) / 64;
    const int64_t hi = k0 < sinks ? pr.M : std::min<int64_t>(pr.M, k0 + bk - 1 - off + std::min<int64_t>(window, pr.N));
    const int64_t n = pr.G * std::max<int64_t>(0, (hi + 63) / 64 - lo);
    const int64_t units = n > 0 ? n + fas::kBlockUnits : 0;
    longest = std::max(longest, units);
    w.head_units += units;
  }
  const int64_t all = heads * w.head_units, slots = pr.D == 128 ? kCus : 2 * kCus;
  const int64_t blocks = heads * w.nkb;
  w.wgs = blocks;
  if (all > 0) {
    const double mean = (double)all / (double)blocks, us_per_tile = pr.D == 128 ? 2.0 : 1.6;
    const double whole = std::max({(double)longest, (double)all / (double)slots,
                                   blocks <= slots ? 0.0
                                                   : mean * (double)((blocks + slots - 1) / slots)});
    const int64_t chunk = std::max<int64_t>(4 + fas::kBlockUnits, (all + slots - 1) / slots);
    if ((double)chunk + 4.0 + 8.0 / us_per_tile < whole && chunk < INT_MAX) {
      w.chunk = chunk;
      w.wgs = (all + chunk - 1) / chunk;
      w.wgs = (w.wgs + 7) / 8 * 8;  // an equal number for each XCD; the last may find no tiles
    }
  }
  const size_t rows = (size_t)pr.B * pr.H * w.mpad * 4;
  w.delta = align256(rows);
  w.part = 2 * align256(rows);
  w.total = w.part + (w.chunk > 0 ? (size_t)w.wgs * 2 * bk * 2 * pr.D * 4 : 0);
  return w;
}

}  // namespace

extern "C" {

size_t fas_attention_window_workspace(const fas_attn_args* a, int64_t window, int64_t sinks,
                                      int backward) {
  Problem pr;
  if (check_window("fas_attention_window_workspace", a, window, sinks, &pr)) return (size_t)-1;
  return backward ? bwd_plan(pr, window, sinks).total : fwd_split(pr, window, sinks).total;
}

int fas_attention_window(const fas_attn_args* a, int64_t window, int64_t sinks, float* lse,
                         const int64_t lst[3], void* ws, size_t ws_bytes, void* stream) {
  static const char* fn = "fas_attention_window";
  Problem pr;
  int rc;
  if ((rc = check_window(fn, a, window, sinks, &pr))) return rc;
  if ((rc = fas::check_args(fn, a, &pr))) return rc;
  if ((int64_t)pr.B * pr.M == 0) return FAS_OK;
  if (lse != nullptr) {
    if (lst == nullptr) return fail(FAS_ERR_INVALID, fn, "lse strides are NULL");
    if (fas::strides_out_of_range(lst, 3))
      return fail(FAS_ERR_INVALID, fn, "lse strides must lie in [0, 2^46)");
  }
  const fas::RowsSplit w = fwd_split(pr, window, sinks);
  if ((rc = fas::check_rows_workspace(fn, w.total, ws, ws_bytes))) return rc;
  if (w.grid > INT_MAX)
    return fail(FAS_ERR_UNSUPPORTED, fn, "more row blocks than one launch takes");
  fas::RowsParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.o = static_cast<uint16_t*>(a->out);
  p.lse = lse;
  p.k = static_cast<const uint8_t*>(a->k);
  p.v = static_cast<const uint8_t*>(a->v);
  p.sq0 = a->q_stride[0]; p.sq1 = a->q_stride[1]; p.sq2 = a->q_stride[2];
  p.so0 = a->out_stride[0]; p.so1 = a->out_stride[1]; p.so2 = a->out_stride[2];
  if (lse != nullptr) {
    p.sl0 = lst[0]; p.sl1 = lst[1]; p.sl2 = lst[2];
  }
  p.sk0 = 2 * a->k_stride[0]; p.sk1 = 2 * a->k_stride[1]; p.sk2 = 2 * a->k_stride[2];
  p.sv0 = 2 * a->v_stride[0]; p.sv1 = 2 * a->v_stride[1]; p.sv2 = 2 * a->v_stride[2];
  p.k_bytes = slice_bytes(pr.N, a->k_stride[2], pr.D);
  p.v_bytes = slice_bytes(pr.N, a->v_stride[2], pr.D);
  p.lengths_all = p.capacity = pr.N;
  p.B = pr.B; p.H = pr.H; p.Hk = pr.Hk; p.G = pr.G; p.M = pr.M;
  p.window = (int)std::min<int64_t>(window, fas::kNoWindow);
  p.sinks = (int)std::min<int64_t>(sinks, fas::kNoWindow);
  fas::apply_rows_split(p, w, ws);
  p.qk_scale = fas::qk_scale_of(pr.sm_scale);
  p.qneg = pr.sm_scale < 0.f ? 0x80008000u : 0u;
  return hip_status(fn, fas::launch_window_fwd(p, pr.dtype, pr.D, static_cast<hipStream_t>(stream)));
}

int fas_attention_window_backward(const fas_attn_args* a, int64_t window, int64_t sinks,
                                  const void* dout, const int64_t gst[4], const float* lse,
                                  const int64_t lst[3], void* dq, const int64_t qst[4], void* dk,
                                  const int64_t kst[4], void* dv, const int64_t vst[4], void* ws,
                                  size_t ws_bytes, void* stream) {
  static const char* fn = "fas_attention_window_backward";
  Problem pr;
  int rc;
  if ((rc = check_window(fn, a, window, sinks, &pr))) return rc;
  if ((rc = fas::check_args(fn, a, &pr))) return rc;
  if (pr.B == 0) return FAS_OK;
  if (pr.M > 0) {
    if (gst == nullptr || qst == nullptr || lst == nullptr || lse == nullptr)
      return fail(FAS_ERR_INVALID, fn, "dout, dq or lse is NULL");
    if (fas::strides_out_of_range(lst, 3))
      return fail(FAS_ERR_INVALID, fn, "lse strides must lie in [0, 2^46)");
    if ((rc = check_tensor(fn, "dout", dout, gst, pr.M, pr.D))) return rc;
    if ((rc = check_tensor(fn, "dq", dq, qst, pr.M, pr.D))) return rc;
  }
  if (pr.N > 0) {
    if (kst == nullptr || vst == nullptr) return fail(FAS_ERR_INVALID, fn, "dk or dv is NULL");
    if ((rc = check_tensor(fn, "dk", dk, kst, pr.N, pr.D))) return rc;
    if ((rc = check_tensor(fn, "dv", dv, vst, pr.N, pr.D))) return rc;
  }
  if (pr.M > (1 << 26)) return fail(FAS_ERR_UNSUPPORTED, fn, "seqlen_q exceeds 2^26");
  const BwdPlan w = bwd_plan(pr, window, sinks);
  if ((rc = fas::check_rows_workspace(fn, w.total, ws, ws_bytes))) return rc;
  if (w.wgs > INT_MAX || (int64_t)pr.B * pr.Hk * w.nkb * 8 > INT_MAX ||
      (int64_t)pr.B * pr.H * (w.mpad / fas::kBwdBlock) > INT_MAX)
    return fail(FAS_ERR_UNSUPPORTED, fn, "more row blocks than one launch takes");

  fas::WindowBwdParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.o = static_cast<const uint16_t*>(a->out);
  p.dout = static_cast<const uint16_t*>(dout);
  p.lse = lse;
  char* base = static_cast<char*>(ws);
  p.nl = reinterpret_cast<float*>(base);
  p.delta = reinterpret_cast<float*>(base + w.delta);
  p.part = reinterpret_cast<float*>(base + w.part);
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.sq0 = a->q_stride[0]; p.sq1 = a->q_stride[1]; p.sq2 = a->q_stride[2];
  p.sk0 = a->k_stride[0]; p.sk1 = a->k_stride[1]; p.sk2 = a->k_stride[2];
  p.sv0 = a->v_stride[0]; p.sv1 = a->v_stride[1]; p.sv2 = a->v_stride[2];
  p.so0 = a->out_stride[0]; p.so1 = a->out_stride[1]; p.so2 = a->out_stride[2];
  if (pr.M > 0) {
    p.sg0 = gst[0]; p.sg1 = gst[1]; p.sg2 = gst[2];
    p.sdq0 = qst[0]; p.sdq1 = qst[1]; p.sdq2 = qst[2];
    p.sl0 = lst[0]; p.sl1 = lst[1]; p.sl2 = lst[2];
    p.q_bytes = slice_bytes(pr.M, p.sq2, pr.D);
    p.g_bytes = slice_bytes(pr.M, p.sg2, pr.D);
    p.o_bytes = slice_bytes(pr.M, p.so2, pr.D);
  }
  if (pr.N > 0) {
    p.sdk0 = kst[0]; p.sdk1 = kst[1]; p.sdk2 = kst[2];
    p.sdv0 = vst[0]; p.sdv1 = vst[1]; p.sdv2 = vst[2];
    p.k_bytes = slice_bytes(pr.N, p.sk2, pr.D);
    p.v_bytes = slice_bytes(pr.N, p.sv2, pr.D);
  }
  p.qneg = pr.sm_scale < 0.f ? 0x80008000u : 0u;
  p.B = pr.B; p.H = pr.H; p.G = pr.G; p.Hk = pr.Hk; p.M = pr.M; p.N = pr.N;
  p.Mpad = (int)w.mpad;
  p.causal = 1;
  p.causal_off = pr.N - pr.M;
  p.nkb = (int)w.nkb;
  p.nrb = (int)(w.mpad / fas::kBwdBlock);
  p.wgs = (int)w.wgs;
  p.chunk = (int)w.chunk;
  p.head_units = w.head_units;
  p.window = (int)std::min<int64_t>(window, fas::kNoWindow);
  p.sinks = (int)std::min<int64_t>(sinks, fas::kNoWindow);
  p.sm_scale = std::fabs(pr.sm_scale);
  p.scale_signed = pr.sm_scale;
  p.qk_scale = fas::qk_scale_of(pr.sm_scale);
  return hip_status(fn, fas::launch_window_bwd(p, pr.dtype, pr.D, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
