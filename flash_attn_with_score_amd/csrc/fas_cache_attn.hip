// Instances and launcher of the attention over the quantised KV cache
// (fas_cache_attn.hpp).
#include "fas_cache_attn.hpp"
#include "fas_launch.hpp"

namespace fas {

template <class E, int D, int BITS>
static hipError_t attn_t(const RowsParams& p, hipStream_t s) {
  const int rows = p.G * p.M;
  const dim3 grid((unsigned)((int64_t)p.B * p.Hk * p.nrb * p.nsplit)), block(256);
  const dim3 merge((unsigned)((int64_t)p.B * p.Hk * rows));
  if (rows <= kCacheFewRows) {
    hipLaunchKernelGGL((cache_few_kernel<E, D, BITS>), grid, block, 0, s, p);
    if (p.nsplit > 1)
      hipLaunchKernelGGL((merge_kernel<E, D, kCacheFewRows, kCacheFewKeys>), merge, block, 0,
                         s, p);
  } else {
    hipLaunchKernelGGL((rows_kernel<E, D, CacheSource<E, D, BITS>>), grid, block, 0, s, p);
    if (p.nsplit > 1)
      hipLaunchKernelGGL((merge_kernel<E, D, kRowsBlock, kRowsKeys>), merge, block,
                         0, s, p);
  }
  return hipGetLastError();
}

template <class E, int D>
static hipError_t attn_bits(const RowsParams& p, int bits, hipStream_t s) {
  return bits == 4 ? attn_t<E, D, 4>(p, s) : attn_t<E, D, 8>(p, s);
}

template <class E>
static hipError_t attn_d(const RowsParams& p, int d, int bits, hipStream_t s) {
  switch (d) {
    case 16: return attn_bits<E, 16>(p, bits, s);
    case 32: return attn_bits<E, 32>(p, bits, s);
    case 64: return attn_bits<E, 64>(p, bits, s);
    case 128: return attn_bits<E, 128>(p, bits, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_cache_attn(const RowsParams& p, int dtype, int d, int bits, hipStream_t s) {
  return dtype == 0 ? attn_d<F16>(p, d, bits, s) : attn_d<BF16>(p, d, bits, s);
}

}  // namespace fas
