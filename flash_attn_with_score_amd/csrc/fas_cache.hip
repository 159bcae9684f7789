// Instances and launchers of the quantised KV cache's row kernels (fas_cache.hpp).
#include "fas_cache.hpp"
#include "fas_launch.hpp"

namespace fas {

template <class E, int D, int BITS, int R>
static hipError_t rows_r(const CacheParams& p, bool append, hipStream_t s) {
  const dim3 grid((unsigned)(2 * (int64_t)p.B * p.H * p.chunks)), block(256);
  if (append)
    hipLaunchKernelGGL((cache_append_kernel<E, D, BITS, R>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((cache_read_kernel<E, D, BITS, R>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <class E, int D, int BITS>
static hipError_t rows_t(const CacheParams& p, bool append, hipStream_t s) {
  return p.rows == 1 ? rows_r<E, D, BITS, 1>(p, append, s) : rows_r<E, D, BITS, 4>(p, append, s);
}

template <class E, int D>
static hipError_t rows_bits(const CacheParams& p, int bits, bool append, hipStream_t s) {
  return bits == 4 ? rows_t<E, D, 4>(p, append, s) : rows_t<E, D, 8>(p, append, s);
}

template <class E>
static hipError_t rows_d(const CacheParams& p, int d, int bits, bool append, hipStream_t s) {
  switch (d) {
    case 16: return rows_bits<E, 16>(p, bits, append, s);
    case 32: return rows_bits<E, 32>(p, bits, append, s);
    case 64: return rows_bits<E, 64>(p, bits, append, s);
    case 128: return rows_bits<E, 128>(p, bits, append, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_cache_append(const CacheParams& p, int dtype, int d, int bits, hipStream_t s) {
  return dtype == 0 ? rows_d<F16>(p, d, bits, true, s) : rows_d<BF16>(p, d, bits, true, s);
}
hipError_t launch_cache_read(const CacheParams& p, int dtype, int d, int bits, hipStream_t s) {
  return dtype == 0 ? rows_d<F16>(p, d, bits, false, s) : rows_d<BF16>(p, d, bits, false, s);
}

}  // namespace fas
