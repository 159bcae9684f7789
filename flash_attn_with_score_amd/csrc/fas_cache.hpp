// gfx950 kernels of the quantised KV cache: rows in (append), rows out (read).
// The attention over it is in fas_cache_attn.hpp.
//
// A row of D channels is stored as codes of 4 bits (e2m1: 0, 1/2, 1, 3/2, 2,
// 3, 4, 6 and their negatives; the lower channel in the low half of a byte)
// or 8 bits (e4m3, largest 448), with one scale 2^(byte - 127) per block of 32
// channels (16 where D = 16).  gfx950 converts a pair of such codes to fp16 or
// bf16 with the scale applied in one instruction, and back (round to nearest
// even; checked against the definition over every fp16 and bf16 value and
// every code), which is why the cache has this form: a key row costs D / 2
// conversions and nothing else, and a value is the same number in both types.
//
// The scale is the least power of two with amax <= C s, C the largest code, so
// no value is clipped, but for the largest of the type: the exponent stops
// where C s would pass the type's range, and values above C s become C s.  A
// block that holds an infinity or NaN gets byte 255, whose values all read as
// NaN.
#pragma once
#include "fas_device.hpp"
#include "fas_params.hpp"

namespace fas {

// Reads and writes of cache elements of type E as codes of BITS bits.
template <class E, int BITS>
struct CacheCode;

template <>
struct CacheCode<BF16, 4> {
  // Largest biased scale exponent: 6 * 2^125 < 2^128.
  static constexpr uint32_t kMaxScale = 125 + 127;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
  }
  template <int I>
  static __device__ __forceinline__ uint32_t put(uint32_t w, uint32_t x, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, x), s, I);
  }
};
template <>
struct CacheCode<F16, 4> {
  static constexpr uint32_t kMaxScale = 13 + 127;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, I));
  }
  template <int I>
  static __device__ __forceinline__ uint32_t put(uint32_t w, uint32_t x, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, x), s, I);
  }
};
typedef short s16x2 __attribute__((ext_vector_type(2)));
template <>
struct CacheCode<BF16, 8> {
  static constexpr uint32_t kMaxScale = 119 + 127;  // 448 * 2^119 < 2^128
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, I != 0));
  }
  template <int I>
  static __device__ __forceinline__ uint32_t put(uint32_t w, uint32_t x, float s) {
    return __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(s16x2, w),
                                                            __builtin_bit_cast(bf16x2, x), s, I != 0));
  }
};
template <>
struct CacheCode<F16, 8> {
  static constexpr uint32_t kMaxScale = 7 + 127;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, I != 0));
  }
  template <int I>
  static __device__ __forceinline__ uint32_t put(uint32_t w, uint32_t x, float s) {
    return __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(s16x2, w),
                                                           __builtin_bit_cast(f16x2, x), s, I != 0));
  }
};

// Scale byte to scale (byte 255: an fp32 infinity, which the conversions turn
// into NaN; byte 0 stands for 2^-127 in the conversions, which read the
// exponent field alone).
__device__ __forceinline__ float cache_scale(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

// Eight elements from their codes: one word of 4-bit codes, two of 8-bit.
template <class E, int BITS>
__device__ __forceinline__ u32x4 cache_unpack8(const uint32_t* w, float s) {
  using C = CacheCode<E, BITS>;
  if constexpr (BITS == 4)
    return u32x4{C::template pair<0>(w[0], s), C::template pair<1>(w[0], s),
                 C::template pair<2>(w[0], s), C::template pair<3>(w[0], s)};
  else
    return u32x4{C::template pair<0>(w[0], s), C::template pair<1>(w[0], s),
                 C::template pair<0>(w[1], s), C::template pair<1>(w[1], s)};
}

// Element type's bits of +inf: anything at or above it (sign off) is not
// finite.
template <class E>
constexpr uint32_t kInfBits = std::is_same_v<E, BF16> ? 0x7f80u : 0x7c00u;

// First row of sequence b: start[b], or start_all without a tensor.
__device__ __forceinline__ int cache_start(const CacheParams& p, int b) {
  return p.start != nullptr ? p.start[b] : p.start_all;
}

// Workgroup -> (tensor: 0 keys, 1 values; batch; head; first token); thread ->
// unit of 8 channels of R tokens, kRows apart.  With R = 4 a thread has four
// loads under way (B8 Hk8 N16384 D128, 4 bits: append 177 -> 117 us, read 161 ->
// 94); R = 1 spreads calls of few rows over more CUs (Hk8 N512: append 3.1 us,
// with four 4.5).
template <int D, int R>
struct CacheUnit {
  static constexpr int kUnits = D / 8;        // threads per row
  static constexpr int kRows = 256 / kUnits;  // rows side by side
  int which, b, h, token, unit;
  __device__ __forceinline__ CacheUnit(const CacheParams& p) {
    uint32_t id = blockIdx.x;
    which = (int)(id & 1u);
    id >>= 1;
    const uint32_t bh = id / (uint32_t)p.chunks;
    token = (int)(id - bh * (uint32_t)p.chunks) * (kRows * R) + (int)threadIdx.x / kUnits;
    b = (int)(bh / (uint32_t)p.H);
    h = (int)(bh - (uint32_t)b * (uint32_t)p.H);
    unit = (int)threadIdx.x % kUnits;
  }
};

// Quantises rows [0, counts[b]) of k and v into cache rows start[b] + row.
// Rows past the capacity (or before row 0) are not written.  The block's
// largest magnitude comes from the four threads (two where D = 16) that share
// it.  Bound by the bytes: 16 in, 4 or 8 out a thread and row.
template <class E, int D, int BITS, int R>
__global__ __launch_bounds__(256) void cache_append_kernel(const CacheParams p) {
  using C = CacheCode<E, BITS>;
  const CacheUnit<D, R> u(p);
  const int count = p.counts != nullptr ? min(p.counts[u.b], p.M) : p.M;
  const int64_t row0 = cache_start(p, u.b);
  const CacheSide& c = p.side[u.which];
  auto live = [&](int i) {
    const int token = u.token + i * CacheUnit<D, R>::kRows;
    return token < count && row0 + token >= 0 && row0 + token < p.capacity;
  };
  u32x4 rows[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    rows[i] = u32x4{};
    if (live(i))
      rows[i] = *reinterpret_cast<const u32x4*>(
          c.rows + u.b * c.sr0 + u.h * c.sr1 +
          (int64_t)(u.token + i * CacheUnit<D, R>::kRows) * c.sr2 + 8 * u.unit);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    u32x4 x = rows[i];
    // Magnitudes as 15-bit integers order like the values, infinities and NaN
    // last.
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      top = max(top, x[w] & 0x7fffu);
      top = max(top, (x[w] >> 16) & 0x7fffu);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    if constexpr (D >= 32) top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    // amax = f 2^e, 1 <= f < 2.  4 bits: C = 1.5 * 2^2, so s = 2^(e - 2), or
    // 2^(e - 1) for f > 1.5.  8 bits: C = 1.75 * 2^8.  The addition carries into
    // the exponent field where f passes C's fraction.
    const uint32_t bits = __builtin_bit_cast(uint32_t, E::to_f32((uint16_t)top));
    const int e =
        BITS == 4 ? (int)((bits + 0x3fffffu) >> 23) - 2 : (int)((bits + 0x1fffffu) >> 23) - 8;
    const uint32_t byte = top >= kInfBits<E> ? 255u : (uint32_t)min(max(e, 1), (int)C::kMaxScale);
    if (byte >= C::kMaxScale) {
      // The type's largest values pass C s (or the block is not finite: codes 0).
      const float lim = (BITS == 4 ? 6.f : 448.f) * cache_scale(C::kMaxScale);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float lo = E::to_f32((uint16_t)(x[w] & 0xffffu)), hi = E::to_f32((uint16_t)(x[w] >> 16));
        x[w] = byte == 255u ? 0u
                            : E::pack(fminf(fmaxf(lo, -lim), lim), fminf(fmaxf(hi, -lim), lim));
      }
    }
    const float s = byte == 255u ? 1.f : cache_scale(byte);
    if (!live(i)) continue;
    const int64_t row = row0 + u.token + i * CacheUnit<D, R>::kRows;
    uint8_t* code = c.codes + u.b * c.sc0 + u.h * c.sc1 + row * c.sc2;
    if constexpr (BITS == 4) {
      uint32_t w = 0;
      w = C::template put<0>(w, x[0], s);
      w = C::template put<1>(w, x[1], s);
      w = C::template put<2>(w, x[2], s);
      w = C::template put<3>(w, x[3], s);
      reinterpret_cast<uint32_t*>(code)[u.unit] = w;
    } else {
      u32x2 w{0u, 0u};
      w.x = C::template put<0>(w.x, x[0], s);
      w.x = C::template put<1>(w.x, x[1], s);
      w.y = C::template put<0>(w.y, x[2], s);
      w.y = C::template put<1>(w.y, x[3], s);
      reinterpret_cast<u32x2*>(code)[u.unit] = w;
    }
    if (D < 32 ? u.unit == 0 : u.unit % 4 == 0)
      c.scales[u.b * c.ss0 + u.h * c.ss1 + row * c.ss2 + u.unit / 4] = (uint8_t)byte;
  }
}

// Cache rows start[b] + row, row in [0, M), as values; rows outside the cache
// are zeros.  The values stream past the caches.
template <class E, int D, int BITS, int R>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheParams p) {
  const CacheUnit<D, R> u(p);
  const int64_t row0 = cache_start(p, u.b);
  const CacheSide& c = p.side[u.which];
  uint32_t w[R][2], byte[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int token = u.token + i * CacheUnit<D, R>::kRows;
    const int64_t row = row0 + token;
    w[i][0] = w[i][1] = byte[i] = 0u;
    if (token < p.M && row >= 0 && row < p.capacity) {
      const uint8_t* code = c.codes + u.b * c.sc0 + u.h * c.sc1 + row * c.sc2;
      byte[i] = c.scales[u.b * c.ss0 + u.h * c.ss1 + row * c.ss2 + u.unit / 4];
      if constexpr (BITS == 4) {
        w[i][0] = reinterpret_cast<const uint32_t*>(code)[u.unit];
      } else {
        const u32x2 t = reinterpret_cast<const u32x2*>(code)[u.unit];
        w[i][0] = t.x;
        w[i][1] = t.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int token = u.token + i * CacheUnit<D, R>::kRows;
    if (token < p.M)
      __builtin_nontemporal_store(
          cache_unpack8<E, BITS>(w[i], cache_scale(byte[i])),
          reinterpret_cast<u32x4*>(c.rows + u.b * c.sr0 + u.h * c.sr1 + (int64_t)token * c.sr2 +
                                   8 * u.unit));
  }
}

}  // namespace fas
