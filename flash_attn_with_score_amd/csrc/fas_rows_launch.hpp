// Launch of a call's rows (fas_rows.hpp), whatever its tile sources: at most 16
// virtual rows, at most 32, or more, and the merge of split rows.
#pragma once
#include "fas_launch.hpp"
#include "fas_rows.hpp"

namespace fas {

template <class E, int D, int BM, int BN>
hipError_t launch_merge(const RowsParams& p, hipStream_t s) {
  const int64_t groups = (int64_t)p.B * p.Hk, rows = p.G * p.M;
  if (p.nsplit <= kMergeFew) {
    constexpr int RPB = 1024 / D;
    hipLaunchKernelGGL((merge_few_kernel<E, D, BM, BN>),
                       dim3((unsigned)(groups * ((rows + RPB - 1) / RPB))), dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((merge_kernel<E, D, BM, BN>), dim3((unsigned)(groups * rows)), dim3(256), 0, s,
                       p);
  }
  return hipGetLastError();
}

template <class E, int D, class FEW, class MANY>
hipError_t launch_rows(const RowsParams& p, hipStream_t s) {
  const int rows = p.G * p.M;
  const dim3 grid((unsigned)p.grid), block(256);
  if (rows <= 16)
    hipLaunchKernelGGL((few_kernel<E, D, 1, FEW>), grid, block, 0, s, p);
  else if (rows <= kFewRows)
    hipLaunchKernelGGL((few_kernel<E, D, 2, FEW>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((rows_kernel<E, D, MANY>), grid, block, 0, s, p);
  if (p.nsplit > 1)
    return rows <= kFewRows ? launch_merge<E, D, kFewRows, kFewKeys>(p, s)
                            : launch_merge<E, D, kRowsBlock, kRowsKeys>(p, s);
  return hipGetLastError();
}

}  // namespace fas
