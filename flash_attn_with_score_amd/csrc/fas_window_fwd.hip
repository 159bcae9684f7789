// Instances and launcher of the windowed attention's forward (fas_window.hpp).
#include "fas_rows_launch.hpp"
#include "fas_window.hpp"

namespace fas {

template <class E, int D>
static hipError_t fwd_t(const RowsParams& p, hipStream_t s) {
  return launch_rows<E, D, DenseFewSource<E, D>, DenseSource<E, D>>(p, s);
}

template <class E>
static hipError_t fwd_d(const RowsParams& p, int d, hipStream_t s) {
  switch (d) {
    case 16: return fwd_t<E, 16>(p, s);
    case 32: return fwd_t<E, 32>(p, s);
    case 64: return fwd_t<E, 64>(p, s);
    case 128: return fwd_t<E, 128>(p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_window_fwd(const RowsParams& p, int dtype, int d, hipStream_t s) {
  return dtype == 0 ? fwd_d<F16>(p, d, s) : fwd_d<BF16>(p, d, s);
}

}  // namespace fas
