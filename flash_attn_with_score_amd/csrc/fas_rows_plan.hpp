// How calls of the row kernels (fas_rows.hpp, fas_cache_attn.hpp) are dealt to
// workgroups.  Host code; depends on sizes only, so a workspace query and the
// launch agree.
#pragma once
#include <algorithm>
#include <cstdint>

#include "fas_check.hpp"
#include "fas_params.hpp"

namespace fas {

struct RowsSplit {
  int64_t nrb, nsplit, min_tiles, rpad;
  size_t part_ml, total;  // workspace: offset of the offsets and sums, bytes
};

// rows: virtual rows of each of `groups` (batch entry, KV head) pairs; keys:
// the most that a sequence can hold; few: few_kernel runs.
inline RowsSplit rows_split(int64_t groups, int64_t rows, int64_t tokens, int64_t keys,
                            int64_t window, int64_t sinks, int64_t D, bool few) {
  RowsSplit w{};
  const int64_t bm = few ? kFewRows : kRowsBlock, bn = few ? kFewKeys : kRowsKeys;
  w.nrb = (rows + bm - 1) / bm;
  w.rpad = w.nrb * bm;
  // Key tiles that a row block can need, whatever the sequences' lengths.
  if (window > 0)
    keys = std::min(keys, std::min(window, keys) + std::min(sinks, keys) + std::min(tokens, bm) +
                              2 * bn);
  const int64_t tiles = (keys + bn - 1) / bn;
  // Two workgroups a CU in one round; fewer keys a workgroup than these cost
  // more in the merge than they save.
  w.min_tiles = few ? 16 : 8;
  constexpr int64_t slots = 2 * kCus;
  const int64_t blocks = groups * w.nrb;
  w.nsplit = 1;
  if (blocks > 0 && blocks < slots)
    w.nsplit = std::max<int64_t>(1, std::min({(slots + blocks - 1) / blocks, tiles / w.min_tiles,
                                              (int64_t)kRowsMaxSplits}));
  if (w.nsplit > 1) {
    const size_t n = (size_t)(groups * w.nsplit * w.rpad);
    w.part_ml = align256(n * (size_t)D * 4);
    w.total = w.part_ml + align256(n * 8);
  }
  return w;
}

inline int check_rows_workspace(const char* fn, size_t need, const void* ws, size_t bytes) {
  if (need > 0 && (ws == nullptr || bytes < need || reinterpret_cast<uintptr_t>(ws) % 256))
    return fail(FAS_ERR_WORKSPACE, fn, "needs %zu bytes of workspace aligned to 256, got %zu at %p",
                need, bytes, ws);
  return FAS_OK;
}

inline void apply_rows_split(RowsParams& p, const RowsSplit& w, void* ws) {
  p.nrb = (int)w.nrb;
  p.nsplit = (int)w.nsplit;
  p.min_tiles = (int)w.min_tiles;
  p.Rpad = (int)w.rpad;
  if (w.nsplit > 1) {
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part_ml);
  }
}

}  // namespace fas
