// Instances and launcher of the attention over the quantised KV cache
// (fas_cache_attn.hpp).
#include "fas_cache_attn.hpp"
#include "fas_rows_launch.hpp"

namespace fas {

template <class E, int D, int BITS>
static hipError_t attn_t(const RowsParams& p, hipStream_t s) {
  return launch_rows<E, D, CacheFewSource<E, D, BITS>, CacheSource<E, D, BITS>>(p, s);
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
