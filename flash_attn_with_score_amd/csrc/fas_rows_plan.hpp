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
  int64_t nrb, nsplit, min_tiles, rpad, grid;
  bool balance;
  size_t part_ml, part_per, total;  // workspace: offsets, bytes
};
// Workgroups of a call whose row blocks alone leave CUs idle: two a CU.  (Three
// fit, but the third comes at the others' cost: B4 Hk8 N131072 D128 4 bits 105
// us, with 1024 122.)
constexpr int64_t kRowsSlots = 2 * kCus;

// rows: virtual rows of each of the batch's `groups` (batch entry, KV head) pairs; keys:
// the most that a sequence can hold (ragged: they may hold fewer); few:
// few_kernel runs.
inline RowsSplit rows_split(int64_t batch, int64_t groups, int64_t rows, int64_t tokens, int64_t keys,
                            int64_t window, int64_t sinks, int64_t D, bool few, bool ragged) {
  RowsSplit w{};
  const int64_t bm = few ? kFewRows : kRowsBlock, bn = few ? kFewKeys : kRowsKeys;
  w.nrb = (rows + bm - 1) / bm;
  w.rpad = w.nrb * bm;
  // Key tiles that a row block can need, whatever the sequences' lengths.
  if (window > 0)
    keys = std::min(keys, std::min(window, keys) + std::min(sinks, keys) + std::min(tokens, bm) +
                              2 * bn);
  const int64_t tiles = (keys + bn - 1) / bn;
  // few_kernel: its four waves take a tile each per step of about 0.75 us while
  // the loads' latency bounds them, and the merge costs about 4.5 us: a split
  // pays from six steps saved on (B2 Hk8 N1024 D128: 11.5 us, in eight 9.7; B32
  // Hk4 window 1000 D64, in four: 10.8 / 13.0).
  w.min_tiles = few ? 4 : 8;
  const int64_t blocks = groups * w.nrb;
  w.nsplit = 1;
  if (blocks > 0 && blocks < kRowsSlots)
    w.nsplit = std::max<int64_t>(1, std::min({(kRowsSlots + blocks - 1) / blocks,
                                              tiles / w.min_tiles, (int64_t)kRowsMaxSplits}));
  if (few) {
    // Whole steps: the nearest number of them a workgroup.
    const int64_t steps = std::max<int64_t>(1, (tiles + 2 * w.nsplit) / (4 * w.nsplit));
    w.nsplit = std::min<int64_t>(std::max<int64_t>(1, (tiles + 4 * steps - 1) / (4 * steps)),
                                 kRowsMaxSplits);
    if (blocks >= kRowsSlots || tiles / 4 - steps <= 6) w.nsplit = 1;
  }
  w.grid = blocks * w.nsplit;
  // Sequences of unknown lengths (rows_balanced): shorter ones leave workgroups
  // to the longer, up to twice the even share each.  Working it out takes
  // about 1.5 us, so only where a workgroup may run for 12 steps.
  if (few && ragged && batch > 1 && batch <= kBalanceBatch && w.nsplit > 1 &&
      tiles >= 48 * w.nsplit) {
    w.balance = true;
    w.nsplit = std::min({2 * w.nsplit, tiles / w.min_tiles, (int64_t)kRowsMaxSplits});
    w.grid = std::min(kRowsSlots + groups, groups * w.nsplit);
  }
  if (w.nsplit > 1) {
    const size_t n = (size_t)(groups * w.nsplit * w.rpad);
    w.part_ml = align256(n * (size_t)D * 4);
    w.part_per = w.part_ml + align256(n * 8);
    w.total = w.part_per + 256;
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
  p.balance = w.balance ? 1 : 0;
  p.slots = (int)kRowsSlots;
  p.grid = (int)w.grid;
  if (w.nsplit > 1) {
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part_ml);
    p.part_per = reinterpret_cast<int*>(static_cast<char*>(ws) + w.part_per);
  }
}

}  // namespace fas
