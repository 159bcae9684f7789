// Instances and launcher of the windowed attention's backward (fas_window.hpp).
#include "fas_launch.hpp"
#include "fas_window.hpp"

#include <type_traits>

namespace fas {

template <class E, int D>
static hipError_t bwd_t(const WindowBwdParams& p, hipStream_t s) {
  const int64_t bh = (int64_t)p.B * p.H, bhk = (int64_t)p.B * p.Hk;
  if (p.M > 0)
    hipLaunchKernelGGL((window_dq_kernel<E, D>), dim3((unsigned)(bh * p.nrb)), dim3(256), 0, s, p);
  if (p.N > 0) {
    // Two waves for each 32 keys hand P over in fp16, which loses nothing beside
    // bf16's own rounding of dS, but would be a second rounding of the same size in
    // fp16 (dK's norm of error 1.74 times a mere rounding's, 1.43 without it).
    if constexpr (D == 128 && std::is_same_v<E, BF16>)
      hipLaunchKernelGGL((window_dkdv_kernel<E, D>), dim3((unsigned)p.wgs), dim3(512), 0, s, p);
    else
      hipLaunchKernelGGL((window_dkdv_small_kernel<E, D>), dim3((unsigned)p.wgs), dim3(256), 0, s,
                         p);
    if (p.chunk > 0) {
      const int per = kBwdBlock * (D / 8) / 256;  // workgroups per key block
      hipLaunchKernelGGL((window_reduce_kernel<E, D>), dim3((unsigned)(bhk * p.nkb * per)), dim3(256),
                         0, s, p);
    }
  }
  return hipGetLastError();
}

template <class E>
static hipError_t bwd_d(const WindowBwdParams& p, int d, hipStream_t s) {
  switch (d) {
    case 16: return bwd_t<E, 16>(p, s);
    case 32: return bwd_t<E, 32>(p, s);
    case 64: return bwd_t<E, 64>(p, s);
    case 128: return bwd_t<E, 128>(p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_window_bwd(const WindowBwdParams& p, int dtype, int d, hipStream_t s) {
  return dtype == 0 ? bwd_d<F16>(p, d, s) : bwd_d<BF16>(p, d, s);
}

}  // namespace fas
