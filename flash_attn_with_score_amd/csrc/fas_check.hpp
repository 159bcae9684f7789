// Argument checks and error reporting shared by the C ABI's entry points
// (fas_api.cpp and the other *_api.cpp files).  Host code only.
#pragma once
#include "fas.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace fas {

// Sets fas_last_error() of this thread to "fn: message" and returns code
// (fas_api.cpp).
int fail(int code, const char* fn, const char* fmt, ...);

inline int hip_status(const char* fn, hipError_t e) {
  if (e == hipSuccess) return FAS_OK;
  return fail(FAS_ERR_HIP, fn, "HIP launch failed: %s", hipGetErrorString(e));
}

inline bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr int64_t kMaxSliceBytes = (int64_t)1 << 31;
// Largest batch or head stride (elements): 2^46 two-byte elements span 128
// TiB, beyond any device's address space, and keep every offset product of
// the kernels (index * stride, index < 2^24) inside int64.
constexpr int64_t kMaxOuterStride = (int64_t)1 << 46;

// Checks one (B, H, L, D)-shaped 16-bit tensor: innermost stride 1, 16-byte
// aligned rows, and a (batch, head) slice addressable with 32-bit offsets
// (including the tile overhang the kernels read past the last row).  Each
// bound is tested before the product that uses it, so no arithmetic here
// can overflow whatever strides the caller passes.
inline int check_tensor(const char* fn, const char* name, const void* ptr, const int64_t* st,
                        int64_t rows, int64_t D) {
  if (ptr == nullptr) return fail(FAS_ERR_INVALID, fn, "%s is NULL", name);
  if (st[3] != 1)
    return fail(FAS_ERR_INVALID, fn, "%s innermost stride must be 1 (got %lld)", name,
                (long long)st[3]);
  if (st[0] < 0 || st[1] < 0 || st[2] < 0)
    return fail(FAS_ERR_INVALID, fn, "%s has a negative stride", name);
  if (!aligned16(ptr) || st[0] % 8 || st[1] % 8 || st[2] % 8)
    return fail(FAS_ERR_INVALID, fn,
                "%s rows must be 16-byte aligned (pointer and outer strides multiples of 8)", name);
  if (st[2] < D) return fail(FAS_ERR_INVALID, fn, "%s rows overlap (row stride < head_dim)", name);
  if (st[0] >= kMaxOuterStride || st[1] >= kMaxOuterStride)
    return fail(FAS_ERR_UNSUPPORTED, fn, "%s batch or head stride exceeds 2^46 elements", name);
  // rows <= 2^28 (check_shape), so with st[2] < 2^31 the product fits.
  if (st[2] >= kMaxSliceBytes || (rows + 512) * st[2] * 2 >= kMaxSliceBytes)
    return fail(FAS_ERR_UNSUPPORTED, fn, "%s (batch, head) slice exceeds 2 GiB", name);
  return FAS_OK;
}

constexpr int64_t kCus = 256;  // MI355X compute units

// Compute units of the current device (fas_api.cpp).
int device_cu_count();

inline uint32_t slice_bytes(int64_t rows, int64_t row_stride, int64_t D) {
  return rows <= 0 ? 0u : (uint32_t)(((rows - 1) * row_stride + D) * 2);
}

struct Problem {
  int B, H, Hk, G, M, N, D, dtype, causal;
  bool dropout;  // dropout_p > 0
  bool keep;     // dropout with a caller keep-bit buffer (fas_attn_args.keep_bits)
  float sm_scale;
  int pack;  // query heads per forward workgroup (GQA packing): G, or 1
};

// Sizes, dtype and flags of a request (no pointers), and with its tensors
// (fas_api.cpp).
int check_shape(const char* fn, const fas_attn_args* a, Problem* pr);
int check_args(const char* fn, const fas_attn_args* a, Problem* pr);

// Exponent scale of the base-2 softmax, |sm_scale| * log2(e).  For
// sm_scale == 0 the weights are uniform over the admissible keys; a zero
// scale would turn the masked scores' -inf into NaN (-inf * 0) and the
// column pass's starting value -lse2 / qk_scale into a division by zero, so
// a tiny positive scale stands in: finite scores then contribute exp2(~0) = 1
// exactly in fp32, masked ones exp2(-inf) = 0.
inline float qk_scale_of(float sm_scale) {
  if (sm_scale == 0.f) return 1e-30f;
  return (float)((double)std::fabs(sm_scale) * 1.4426950408889634);
}

// Whether one of the first n strides is negative or past kMaxOuterStride.
inline bool strides_out_of_range(const int64_t* st, int n) {
  for (int i = 0; i < n; ++i)
    if (st[i] < 0 || st[i] >= kMaxOuterStride) return true;
  return false;
}

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace fas
