// C ABI of the quantised KV cache and the attention over it (declared in
// include/fas.h).
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

using fas::check_tensor;
using fas::fail;
using fas::hip_status;

// Sizes and form of the cache (no pointers).
int check_cache_shape(const char* fn, const fas_kv_cache* c) {
  if (c == nullptr) return fail(FAS_ERR_INVALID, fn, "cache is NULL");
  if (c->dtype != FAS_DTYPE_F16 && c->dtype != FAS_DTYPE_BF16)
    return fail(FAS_ERR_UNSUPPORTED, fn, "dtype %d is not fp16 (0) or bf16 (1)", (int)c->dtype);
  if (c->bits != 4 && c->bits != 8)
    return fail(FAS_ERR_UNSUPPORTED, fn, "bits %d is not 4 or 8", (int)c->bits);
  const int64_t D = c->head_dim;
  if (D != 16 && D != 32 && D != 64 && D != 128)
    return fail(FAS_ERR_UNSUPPORTED, fn, "head_dim %lld not in {16, 32, 64, 128}", (long long)D);
  if (c->batch < 0 || c->heads <= 0 || c->capacity < 0)
    return fail(FAS_ERR_INVALID, fn, "negative or zero size");
  if (c->capacity > (1 << 28) || c->heads > (1 << 24) || c->batch > (1 << 24) ||
      c->batch * c->heads > (1 << 24))
    return fail(FAS_ERR_UNSUPPORTED, fn, "sizes exceed the index range of the kernels");
  return FAS_OK;
}

// One array of the cache: rows of `bytes` contiguous bytes, aligned to their
// size up to 16.
int check_cache_array(const char* fn, const char* name, const void* ptr, const int64_t* st,
                      int64_t bytes) {
  if (ptr == nullptr) return fail(FAS_ERR_INVALID, fn, "%s is NULL", name);
  if (fas::strides_out_of_range(st, 3))
    return fail(FAS_ERR_INVALID, fn, "%s strides must lie in [0, 2^46)", name);
  const int64_t align = std::min<int64_t>(bytes, 16);
  if (reinterpret_cast<uintptr_t>(ptr) % align || st[0] % align || st[1] % align || st[2] % align)
    return fail(FAS_ERR_INVALID, fn, "%s rows must be aligned to %lld bytes", name,
                (long long)align);
  if (st[2] < bytes) return fail(FAS_ERR_INVALID, fn, "%s rows overlap", name);
  // Row index < 2^28: the offset product stays inside int64.
  if (st[2] > ((int64_t)1 << 31))
    return fail(FAS_ERR_UNSUPPORTED, fn, "%s row stride exceeds 2^31 bytes", name);
  return FAS_OK;
}

int check_cache(const char* fn, const fas_kv_cache* c) {
  int rc;
  if ((rc = check_cache_shape(fn, c))) return rc;
  if (c->batch == 0 || c->capacity == 0) return FAS_OK;  // no rows
  const int64_t codes = c->head_dim * c->bits / 8, scales = std::max<int64_t>(1, c->head_dim / 32);
  if ((rc = check_cache_array(fn, "k_codes", c->k_codes, c->k_codes_stride, codes))) return rc;
  if ((rc = check_cache_array(fn, "v_codes", c->v_codes, c->v_codes_stride, codes))) return rc;
  if ((rc = check_cache_array(fn, "k_scales", c->k_scales, c->k_scales_stride, scales))) return rc;
  return check_cache_array(fn, "v_scales", c->v_scales, c->v_scales_stride, scales);
}

// Rows that are written: no two sequences, heads or sides in one place.
int check_distinct(const char* fn, const fas_kv_cache* c) {
  for (const int64_t* st : {c->k_codes_stride, c->v_codes_stride, c->k_scales_stride, c->v_scales_stride})
    if ((c->batch > 1 && st[0] == 0) || (c->heads > 1 && st[1] == 0))
      return fail(FAS_ERR_INVALID, fn, "the cache's rows repeat (stride 0): it cannot be written");
  if (c->k_codes == c->v_codes || c->k_scales == c->v_scales)
    return fail(FAS_ERR_INVALID, fn, "keys and values share an array: it cannot be written");
  return FAS_OK;
}

int check_per_sequence(const char* fn, const char* name, const int32_t* ptr) {
  if (reinterpret_cast<uintptr_t>(ptr) % 4)
    return fail(FAS_ERR_INVALID, fn, "%s must be aligned to 4 bytes", name);
  return FAS_OK;
}

int move_rows(const char* fn, bool append, const fas_kv_cache* c, const void* k, const int64_t* kst,
              const void* v, const int64_t* vst, int64_t tokens, const int32_t* start,
              int64_t start_all, const int32_t* counts, void* stream) {
  int rc;
  if ((rc = check_cache(fn, c))) return rc;
  if (tokens < 0) return fail(FAS_ERR_INVALID, fn, "negative number of tokens");
  if (tokens > (1 << 28))
    return fail(FAS_ERR_UNSUPPORTED, fn, "sizes exceed the index range of the kernels");
  if ((rc = check_per_sequence(fn, "start", start))) return rc;
  if ((rc = check_per_sequence(fn, "counts", counts))) return rc;
  if (start == nullptr && (start_all < 0 || start_all > c->capacity - tokens))
    return fail(FAS_ERR_INVALID, fn, "%lld rows from %lld lie outside the cache of %lld",
                (long long)tokens, (long long)start_all, (long long)c->capacity);
  if (c->batch == 0 || tokens == 0) return FAS_OK;
  if (kst == nullptr || vst == nullptr) return fail(FAS_ERR_INVALID, fn, "k or v strides are NULL");
  if ((rc = check_tensor(fn, "k", k, kst, tokens, c->head_dim))) return rc;
  if ((rc = check_tensor(fn, "v", v, vst, tokens, c->head_dim))) return rc;
  if (append && c->capacity > 0 && (rc = check_distinct(fn, c))) return rc;
  // Four rows a thread where that still fills the chip four times over.
  const int64_t beside = 256 / (c->head_dim / 8), heads = 2 * c->batch * c->heads;
  const int64_t per = heads * ((tokens + 4 * beside - 1) / (4 * beside)) >= 4 * fas::kCus ? 4 : 1;
  const int64_t chunks = (tokens + per * beside - 1) / (per * beside);
  if (heads * chunks > INT_MAX)
    return fail(FAS_ERR_UNSUPPORTED, fn, "more rows than one launch takes");
  fas::CacheParams p{};
  auto side = [](fas::CacheSide& s, const void* rows, const int64_t* st, void* codes,
                 const int64_t* cst, void* scales, const int64_t* sst) {
    s.rows = static_cast<uint16_t*>(const_cast<void*>(rows));
    s.codes = static_cast<uint8_t*>(codes);
    s.scales = static_cast<uint8_t*>(scales);
    s.sr0 = st[0]; s.sr1 = st[1]; s.sr2 = st[2];
    s.sc0 = cst[0]; s.sc1 = cst[1]; s.sc2 = cst[2];
    s.ss0 = sst[0]; s.ss1 = sst[1]; s.ss2 = sst[2];
  };
  side(p.side[0], k, kst, c->k_codes, c->k_codes_stride, c->k_scales, c->k_scales_stride);
  side(p.side[1], v, vst, c->v_codes, c->v_codes_stride, c->v_scales, c->v_scales_stride);
  p.start = start;
  p.start_all = (int)start_all;
  p.counts = counts;
  p.B = (int)c->batch;
  p.H = (int)c->heads;
  p.M = (int)tokens;
  p.capacity = (int)c->capacity;
  p.rows = (int)per;
  p.chunks = (int)chunks;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int d = (int)c->head_dim;
  return hip_status(fn, append ? fas::launch_cache_append(p, c->dtype, d, c->bits, s)
                               : fas::launch_cache_read(p, c->dtype, d, c->bits, s));
}

int check_attn(const char* fn, const fas_kv_cache* c, const fas_kv_query* a) {
  int rc;
  if ((rc = check_cache_shape(fn, c))) return rc;
  if (a == nullptr) return fail(FAS_ERR_INVALID, fn, "query is NULL");
  if (a->tokens < 0 || a->heads_q <= 0)
    return fail(FAS_ERR_INVALID, fn, "negative or zero size");
  if (a->heads_q % c->heads != 0)
    return fail(FAS_ERR_INVALID, fn, "heads_q (%lld) is not a multiple of the cache's heads (%lld)",
                (long long)a->heads_q, (long long)c->heads);
  if (a->tokens > (1 << 28) || a->heads_q > (1 << 24) || c->batch * a->heads_q > (1 << 24) ||
      a->heads_q / c->heads * a->tokens > (1 << 28))
    return fail(FAS_ERR_UNSUPPORTED, fn, "sizes exceed the index range of the kernels");
  if (a->window < 0 || a->sinks < 0)
    return fail(FAS_ERR_INVALID, fn, "window and sinks must not be negative");
  if (!std::isfinite(a->sm_scale)) return fail(FAS_ERR_INVALID, fn, "sm_scale is not finite");
  if (a->lengths == nullptr && (a->lengths_all < 0 || a->lengths_all > c->capacity))
    return fail(FAS_ERR_INVALID, fn, "length %lld lies outside [0, %lld]",
                (long long)a->lengths_all, (long long)c->capacity);
  return FAS_OK;
}

fas::RowsSplit attn_split(const fas_kv_cache* c, const fas_kv_query* a) {
  const int64_t rows = a->heads_q / c->heads * a->tokens;
  return fas::rows_split(c->batch, c->batch * c->heads, rows, a->tokens,
                         a->lengths == nullptr ? a->lengths_all : c->capacity, a->window, a->sinks,
                         c->head_dim, rows <= fas::kFewRows, a->lengths != nullptr);
}

}  // namespace

extern "C" {

int fas_kv_cache_append(const fas_kv_cache* c, const void* k, const int64_t kst[4], const void* v,
                        const int64_t vst[4], int64_t tokens, const int32_t* start,
                        int64_t start_all, const int32_t* counts, void* stream) {
  return move_rows("fas_kv_cache_append", true, c, k, kst, v, vst, tokens, start, start_all, counts,
                   stream);
}

int fas_kv_cache_read(const fas_kv_cache* c, void* k, const int64_t kst[4], void* v,
                      const int64_t vst[4], int64_t tokens, const int32_t* start,
                      int64_t start_all, void* stream) {
  return move_rows("fas_kv_cache_read", false, c, k, kst, v, vst, tokens, start, start_all, nullptr,
                   stream);
}

size_t fas_attention_kv_cache_workspace(const fas_kv_cache* c, const fas_kv_query* a) {
  if (check_attn("fas_attention_kv_cache_workspace", c, a)) return (size_t)-1;
  return attn_split(c, a).total;
}

int fas_attention_kv_cache(const fas_kv_cache* c, const fas_kv_query* a, float* lse,
                           const int64_t lst[3], void* ws, size_t ws_bytes, void* stream) {
  static const char* fn = "fas_attention_kv_cache";
  int rc;
  if ((rc = check_attn(fn, c, a))) return rc;
  if ((rc = check_cache(fn, c))) return rc;
  if (c->batch * a->tokens == 0) return FAS_OK;
  if ((rc = check_tensor(fn, "q", a->q, a->q_stride, a->tokens, c->head_dim))) return rc;
  if ((rc = check_tensor(fn, "out", a->out, a->out_stride, a->tokens, c->head_dim))) return rc;
  if ((rc = check_per_sequence(fn, "lengths", a->lengths))) return rc;
  if ((rc = check_per_sequence(fn, "counts", a->counts))) return rc;
  if (lse != nullptr) {
    if (lst == nullptr) return fail(FAS_ERR_INVALID, fn, "lse strides are NULL");
    if (fas::strides_out_of_range(lst, 3))
      return fail(FAS_ERR_INVALID, fn, "lse strides must lie in [0, 2^46)");
  }
  const fas::RowsSplit w = attn_split(c, a);
  if ((rc = fas::check_rows_workspace(fn, w.total, ws, ws_bytes))) return rc;
  if (w.grid > INT_MAX)
    return fail(FAS_ERR_UNSUPPORTED, fn, "more row blocks than one launch takes");
  fas::RowsParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.o = static_cast<uint16_t*>(a->out);
  p.lse = lse;
  p.k = static_cast<const uint8_t*>(c->k_codes);
  p.ks = static_cast<const uint8_t*>(c->k_scales);
  p.v = static_cast<const uint8_t*>(c->v_codes);
  p.vs = static_cast<const uint8_t*>(c->v_scales);
  p.sq0 = a->q_stride[0]; p.sq1 = a->q_stride[1]; p.sq2 = a->q_stride[2];
  p.so0 = a->out_stride[0]; p.so1 = a->out_stride[1]; p.so2 = a->out_stride[2];
  if (lse != nullptr) {
    p.sl0 = lst[0]; p.sl1 = lst[1]; p.sl2 = lst[2];
  }
  p.sk0 = c->k_codes_stride[0]; p.sk1 = c->k_codes_stride[1]; p.sk2 = c->k_codes_stride[2];
  p.sks0 = c->k_scales_stride[0]; p.sks1 = c->k_scales_stride[1]; p.sks2 = c->k_scales_stride[2];
  p.sv0 = c->v_codes_stride[0]; p.sv1 = c->v_codes_stride[1]; p.sv2 = c->v_codes_stride[2];
  p.svs0 = c->v_scales_stride[0]; p.svs1 = c->v_scales_stride[1]; p.svs2 = c->v_scales_stride[2];
  p.lengths = a->lengths;
  p.lengths_all = a->lengths == nullptr ? (int)a->lengths_all : 0;
  p.counts = a->counts;
  p.B = (int)c->batch;
  p.H = (int)a->heads_q;
  p.Hk = (int)c->heads;
  p.G = p.H / p.Hk;
  p.M = (int)a->tokens;
  p.capacity = (int)c->capacity;
  p.window = a->window == 0 ? fas::kNoWindow
                            : (int)std::min<int64_t>(a->window, fas::kNoWindow);
  p.sinks = (int)std::min<int64_t>(a->sinks, fas::kNoWindow);
  fas::apply_rows_split(p, w, ws);
  p.qk_scale = fas::qk_scale_of(a->sm_scale);
  p.qneg = a->sm_scale < 0.f ? 0x80008000u : 0u;
  return hip_status(fn, fas::launch_cache_attn(p, c->dtype, (int)c->head_dim, c->bits,
                                               static_cast<hipStream_t>(stream)));
}

}  // extern "C"
