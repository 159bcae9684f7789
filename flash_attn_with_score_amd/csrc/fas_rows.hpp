// Attention of rows with a sliding window and sinks: what the kernels of the
// quantised cache (fas_cache_attn.hpp) and of the windowed attention over dense
// keys (fas_window.hpp) share.
//
// A sequence holds len keys; its cnt query rows are its last tokens, row i at
// position len - cnt + i.  A row at position pos sees key j iff 0 <= j <= pos
// and (j > pos - window or j < sinks).  Rows past cnt, and rows that see no key,
// give O = 0 and L = -inf.  (Dense keys: len = N, cnt = M.)
//
// The G query heads of a KV head read the same keys, so a workgroup takes
// their rows together: virtual row v = i * G + j is row i of head h0 + j.
// Besides the shared loads this keeps a block's positions close together: 128
// virtual rows span 128 / G positions, and the window's tiles that only some of
// them see are few.
//
//   few_kernel    at most 32 virtual rows (decoding).  Bound by the bytes of K
//                 and V, so nothing is shared between the waves: each of the
//                 four streams tiles of 32 keys of its own into registers, and
//                 only V passes through a small LDS tile of the wave's, whose
//                 transposing read gives the A operand of O^T += V^T P^T.  The
//                 products are 16x16x32: one or two tiles of 16 rows, so that
//                 few rows take few registers and more waves hide the latency.
//   rows_kernel   128 virtual rows, four waves of 32, over key tiles of 64 that
//                 they share through LDS.  How a tile gets there is the
//                 source's business (dense rows by LDS DMA, codes through
//                 registers); the next tile is under way while the current
//                 one is used.
//   merge_few_kernel, merge_kernel
//                 add up the parts of rows whose keys were dealt to several
//                 workgroups.
//
// Tiles are dealt by the length the device sees, not by the one the host
// knows: every sequence spreads its own tiles evenly over its workgroups.
#pragma once
#include "fas_device.hpp"
#include "fas_params.hpp"

namespace fas {

// The keys that a block of virtual rows [row0, row0 + BM) reads, as a list: the
// first `ns` keys of the sequence (sinks in front of the window), then the keys
// from the first row's window on.  Tile i is entries [BN i, BN i + BN) of the
// list, so the sinks and the window's edge take no tiles of their own.  The tiles
// are dealt to `used` workgroups in runs of `per`.
struct RowsPlan {
  int len, cnt, pos0;  // keys, query rows, position of row 0
  int lo, hi;          // least and greatest position of the block's live rows (hi < lo: none)
  int ns, shift;       // entry e is key e, or e + shift from entry ns on
  int hide;            // entries in front of this one are sinks: the window's edge leaves them
  int tiles, per, used;
  __device__ __forceinline__ int key(int e) const { return e < ns ? e : e + shift; }
  // The key whose row stands in for entry e in memory: entries behind the
  // last key take its row, their weight is 0.
  __device__ __forceinline__ int row(int e) const { return min(key(e), len - 1); }
};
// Sequence b's block rb of the plan, but for how its tiles are dealt.
template <int BM, int BN>
__device__ __forceinline__ RowsPlan rows_tiles(const RowsParams& p, int b, int rb) {
  RowsPlan c;
  c.len = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.capacity) : p.lengths_all;
  c.cnt = p.counts != nullptr ? min(max(p.counts[b], 0), p.M) : p.M;
  c.pos0 = c.len - c.cnt;
  const int i0 = rb * BM / p.G, i1 = min(c.cnt, (rb * BM + BM - 1) / p.G + 1);  // rows [i0, i1)
  c.lo = c.pos0 + i0;
  c.hi = i1 > i0 ? c.pos0 + i1 - 1 : c.lo - 1;
  c.ns = c.shift = c.hide = c.tiles = 0;
  if (c.hi >= max(c.lo, 0)) {
    const int first = max(0, max(c.lo, 0) - p.window + 1);
    c.ns = min(first, p.sinks);
    c.shift = first - c.ns;
    c.hide = c.shift > 0 ? c.ns : p.sinks;
    c.tiles = (c.hi + 1 - c.shift + BN - 1) / BN;
  }
  return c;
}
// How the tiles of one block are dealt: evenly, to at most nsplit workgroups.
template <int BM, int BN>
__device__ __forceinline__ RowsPlan rows_plan(const RowsParams& p, int b, int rb) {
  RowsPlan c = rows_tiles<BM, BN>(p, b, rb);
  c.per = max(p.min_tiles, (c.tiles + p.nsplit - 1) / p.nsplit);
  if (BM == kFewRows) c.per = (c.per + 3) & ~3;  // few_kernel's four waves take turns
  c.used = max(1, (c.tiles + c.per - 1) / c.per);
  return c;
}

// Inclusive scans over the wave's lanes, as six lane shifts of the vector ALU.
template <class F>
__device__ __forceinline__ int wave_scan(int v, F&& f) {
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));  // row_shr:2
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));  // row_shr:4
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));  // row_shr:8
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return v;
}

// Few rows of a batch whose lengths the host does not know (balance: at most
// kBalanceBatch sequences): all take workgroups of about the same length, the
// batch's tiles over about p.slots of them, and the workgroups that have work
// come first in the grid.  Lane i works out sequence i.  Dealt evenly instead, a
// ragged batch waits for its longest sequence.  Returns the workgroup's plan
// and where it stands (split < 0: no work).
template <int BN>
__device__ __forceinline__ RowsPlan rows_balanced(const RowsParams& p, int id, int& b, int& hk,
                                                  int& split) {
  const int lane = (int)threadIdx.x & 63;
  RowsPlan c = rows_tiles<kFewRows, BN>(p, min(lane, p.B - 1), 0);
  const bool mine = lane < p.B;
  const int tiles = mine ? c.tiles : 0;
  auto sum = [](int x) {
    return __builtin_amdgcn_readlane(wave_scan(x, [](int a, int b) { return a + b; }), 63);
  };
  const int64_t total = sum(tiles);
  const int most =
      __builtin_amdgcn_readlane(wave_scan(tiles, [](int x, int y) { return max(x, y); }), 63);
  const int least = max(p.min_tiles, (most + p.nsplit - 1) / p.nsplit);
  int per = (max(least, (int)((total * p.Hk + p.slots - 1) / p.slots)) + 3) & ~3;
  // The sequences' last workgroups are parts of one, half of one in the mean:
  // longer ones until the batch fits the slots, or nearly.
  int used = 0;
#pragma unroll
  for (int it = 0; it < 3; ++it) {
    used = mine ? max(1, (tiles + per - 1) / per) : 0;
    const int over = sum(used) * p.Hk - p.slots;
    if (it == 2 || over <= 0) break;
    per = (per + (int)(((int64_t)per * over + p.slots - 1) / p.slots) + 3) & ~3;
  }
  const int end = wave_scan(used, [](int x, int y) { return x + y; }) * p.Hk;
  b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine && end <= id));
  split = -1;
  if (b < p.B) {
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, b); };
    c = RowsPlan{of(c.len), of(c.cnt), of(c.pos0), of(c.lo), of(c.hi), of(c.ns), of(c.shift),
                 of(c.hide), of(c.tiles), per, of(used)};
    const int rest = id - (of(end) - c.used * p.Hk);
    hk = __builtin_amdgcn_readfirstlane(rest / c.used);
    split = rest - hk * c.used;
    if (id == 0 && threadIdx.x == 0) *p.part_per = per;
  }
  return c;
}

// Which entries of the list the row at position pos sees: all up to
// pos - shift but those in [hide, pos - window - shift].  (Sinks stand in front
// of every row's own position: ns <= lo - shift.)
struct RowMask {
  int last;   // last visible entry
  int first;  // first entry behind `hide` that is not in front of the window
  __device__ __forceinline__ RowMask(const RowsParams& p, const RowsPlan& c, int pos)
      : last(pos - c.shift), first(pos - p.window - c.shift + 1) {}
};
// What a tile of entries [e0, e0 + n) needs for rows at positions [lo, hi]:
// whether some row does not see its end, or its entries in front of a window.
struct TileMask {
  bool end, edge;
  __device__ __forceinline__ TileMask(const RowsParams& p, const RowsPlan& c, int lo, int hi, int e0,
                                      int n)
      : end(e0 + n - 1 > lo - c.shift),
        edge(e0 + n > c.hide && max(e0, c.hide) < hi - p.window - c.shift + 1) {}
};
// Score s of entry e under the masks that its tile needs.
__device__ __forceinline__ float masked_score(float s, int e, const RowMask& m, const RowsPlan& c,
                                              bool end, bool edge) {
  if (end) s = e > m.last ? neg_inf() : s;
  if (edge) s = (uint32_t)(e - c.hide) < (uint32_t)max(0, m.first - c.hide) ? neg_inf() : s;
  return s;
}
__device__ __forceinline__ bool row_sees(const RowMask& m, const RowsPlan& c, int e) {
  return e <= m.last && (e < c.hide || e >= m.first);
}

// Online softmax of one row a lane pair (lanes c and c + 32) over tiles of
// 32 * NB keys; register r of s[kb] is key 32 kb + acc_row(r, g).
template <class E, int D, int NB>
struct SoftRows {
  static constexpr int DB = (D + 31) / 32;
  float m = neg_inf();  // exponent offset (a score), at most 2^8 below the row's maximum
  float l = 0.f;        // this lane's share of the weights' sum
  f32x16 o[DB];
  __device__ __forceinline__ SoftRows() {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  }
  // Weights 2^(qk (s - m)) as B operands of O^T += V^T P^T; their sum (of
  // this lane's keys) is kept in fp32.  They are rounded to the input type
  // for the product alone.
  __device__ __forceinline__ float weights(const f32x16 (&s)[NB], float qk, u32x4 (&pb)[2 * NB]) {
    const float nb = (m == neg_inf() ? 0.f : m) * qk;
    float lt = 0.f;
#pragma unroll
    for (int cs = 0; cs < 2 * NB; ++cs) {
      float pv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = exp2f_fast(fmaf(s[cs >> 1][8 * (cs & 1) + e], qk, -nb));
        lt += pv[e];
      }
      pb[cs] = u32x4{E::pack(pv[0], pv[1]), E::pack(pv[2], pv[3]), E::pack(pv[4], pv[5]),
                     E::pack(pv[6], pv[7])};
    }
    return lt;
  }
  // The weights are formed with the offset as it is; only where a lane's sum
  // passes 2^14 (or is NaN), or a row has no offset yet, does the wave raise
  // the offsets and form them again.  Every weight stays in fp16's range.
  __device__ __forceinline__ void tile(const f32x16 (&s)[NB], float qk, u32x4 (&pb)[2 * NB]) {
    float lt = weights(s, qk, pb);
    const bool redo = !(lt <= 16384.f) || m == neg_inf();
    if (__builtin_amdgcn_ballot_w64(redo) != 0) {
      float mx = neg_inf();
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
      mx = xor32_max(mx);
      if (mx > m && (m == neg_inf() || (mx - m) * qk > 8.f)) {
        const float a = m == neg_inf() ? 0.f : exp2f_fast((m - mx) * qk);
        l *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= a;
        m = mx;
      }
      lt = weights(s, qk, pb);
    }
    l += lt;
  }
};

// NaN blocks: bit `group` of flag(row) says that the V block of tile row `row`
// reads as NaN; rows that see the key are set to NaN there.
template <class E, int D, int NB, class F>
__device__ __forceinline__ void set_nan_rows(SoftRows<E, D, NB>& a, const RowMask& m,
                                             const RowsPlan& plan, int e0, F&& flag) {
  for (int row = 0; row < 32 * NB; ++row) {
    const uint32_t f = flag(row);
    const bool sees = row_sees(m, plan, e0 + row);
#pragma unroll
    for (int db = 0; db < SoftRows<E, D, NB>::DB; ++db)
      if ((f >> db) & 1u)
#pragma unroll
        for (int r = 0; r < 16; ++r) a.o[db][r] = sees ? __builtin_nanf("") : a.o[db][r];
  }
}

// O (and L) of virtual row v, or, with several workgroups a row, its part.
template <class E, int D, int NB>
__device__ __forceinline__ void store_rows(const RowsParams& p, const SoftRows<E, D, NB>& a,
                                            const RowsPlan& c, int b, int hk, int v, int split,
                                            int g) {
  if (v >= p.G * p.M) return;
  const int i = v / p.G, h = hk * p.G + (v - i * p.G);
  const bool live = i < c.cnt;
  const float l = xor32_add(a.l);
  constexpr int DB = SoftRows<E, D, NB>::DB;
  if (c.used > 1) {
    const int64_t row = ((int64_t)(b * p.Hk + hk) * p.nsplit + split) * p.Rpad + v;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int d0 = 32 * db + 16 * hf + 8 * g;
        if (d0 < D) {
          const f32x16& o = a.o[db];
          const int r = 8 * hf;
          float* out = p.part_o + row * D + d0;
          *reinterpret_cast<f32x4*>(out) = f32x4{o[r], o[r + 1], o[r + 2], o[r + 3]};
          *reinterpret_cast<f32x4*>(out + 4) = f32x4{o[r + 4], o[r + 5], o[r + 6], o[r + 7]};
        }
      }
    if (g == 0) *reinterpret_cast<f32x2*>(p.part_ml + 2 * row) =
        f32x2{a.m == neg_inf() ? neg_inf() : a.m * p.qk_scale, l};
    return;
  }
  const float inv = !live || l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = p.o + b * p.so0 + h * p.so1 + (int64_t)i * p.so2;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int d0 = 32 * db + 16 * hf + 8 * g;
      if (d0 < D) {
        const f32x16& o = a.o[db];
        const int r = 8 * hf;
        // (A select: a padding row's lanes may hold infinities.)
        const u32x4 w = {E::pack(o[r] * inv, o[r + 1] * inv), E::pack(o[r + 2] * inv, o[r + 3] * inv),
                         E::pack(o[r + 4] * inv, o[r + 5] * inv),
                         E::pack(o[r + 6] * inv, o[r + 7] * inv)};
        *reinterpret_cast<u32x4*>(out + d0) = live ? w : u32x4{0u, 0u, 0u, 0u};
      }
    }
  if (g == 0 && p.lse != nullptr)
    p.lse[b * p.sl0 + h * p.sl1 + (int64_t)i * p.sl2] =
        !live || l == 0.f ? neg_inf()
                          : (a.m * p.qk_scale + log2f_fast(l)) * 0.69314718055994531f;
}

// Q row of virtual row v from channel d0 on (zeros for rows that do not exist).
template <int D>
__device__ __forceinline__ u32x4 load_q(const RowsParams& p, int b, int hk, int v, int d0) {
  const int i = v / p.G, h = hk * p.G + (v - i * p.G);
  if (v >= p.G * p.M) return u32x4{0u, 0u, 0u, 0u};
  return *reinterpret_cast<const u32x4*>(p.q + b * p.sq0 + h * p.sq1 + (int64_t)i * p.sq2 + d0) ^
         p.qneg;
}

// LDS DMA of tiles of 64 rows of D 16-bit elements by four waves, as dma_tile,
// with the addresses reduced to one add a transfer: the rows that a lane
// fetches lie 2048 / D apart, which the swizzle does not see, so its offset is
// one per-lane part and uniform ones.
template <int D>
struct TileDma {
  static constexpr int BLOCKS = 64 * D / 512, RPB = 512 / D, CPR = D / 8;
  static_assert(BLOCKS <= 4 || swz<D>(0) == swz<D>(4 * RPB), "the swizzle's period");
  int wave, row;   // the lane's first row
  uint32_t lane;   // byte offset of its 16 bytes in a tile
  uint32_t step;   // bytes from one of its rows to the next
  uint32_t pitch;  // bytes of a row
  __device__ __forceinline__ TileDma(int wave_, int l, uint32_t stride)
      : wave(wave_), row(wave_ * RPB + l / CPR), pitch(2u * stride) {
    lane = (uint32_t)row * pitch + (uint32_t)(((l % CPR) ^ swz<D>(row)) << 4);
    step = 4u * RPB * pitch;
  }
  // Entries [e0, e0 + 64) of the list: rows e0 .., or `shift` rows on from
  // entry ns.
  __device__ __forceinline__ void fetch(i32x4 rsrc, int e0, int ns, int shift, uint32_t lds) const {
    const bool mixed = e0 < ns && e0 + 64 > ns;
    const uint32_t base = (uint32_t)(e0 + (e0 >= ns ? shift : 0)) * pitch;
#pragma unroll
    for (int i = 0; i < (BLOCKS + 3) / 4; ++i) {
      if (BLOCKS % 4 == 0 || wave + 4 * i < BLOCKS) {
        uint32_t off = lane + (base + (uint32_t)i * step);
        if (mixed && e0 + row + 4 * RPB * i >= ns) off += (uint32_t)shift * pitch;
        dma16(rsrc, off, __builtin_amdgcn_readfirstlane(lds + (uint32_t)((wave + 4 * i) * 1024)));
      }
    }
  }
};

// ---------------------------------------------------------------- few rows

__device__ __forceinline__ f32x4 mma16(F16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(BF16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// x combined over the four lanes that share a row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return xor32_max(x);
}
__device__ __forceinline__ float quad_add(float x) { return xor32_add(x + __shfl_xor(x, 16)); }

// Byte offset of (row, 16-byte chunk) in a wave's 32 x D tile of values.  The
// rows that a transposing read takes at once (8 rows, two chunks) fall on
// different banks, and so do the rows that lanes write side by side.
template <int D>
__device__ __forceinline__ uint32_t few_off(int row, int chunk) {
  constexpr int CH = D / 8, S = D == 128 ? 0 : D == 64 ? 1 : D == 32 ? 2 : 3;
  return (uint32_t)(row * 2 * D + ((chunk ^ (2 * ((row >> S) & (CH / 2 - 1)))) << 4));
}

// Rows of few_kernel: lane (c, g), c = lane % 16, g = lane / 16, holds row 16 n + c
// of column tile n; of its scores keys 16 t + 4 g + r, of O^T channels
// 16 dt + 4 g + r.
template <class E, int D, int NC>
struct FewRows {
  static constexpr int DT = D / 16;
  float m[NC], l[NC];
  f32x4 o[NC][DT];
  __device__ __forceinline__ FewRows() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      m[n] = neg_inf();
      l[n] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[n][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // As SoftRows::weights and tile.
  __device__ __forceinline__ float weights(int n, const f32x4 (&s)[2], float qk, u32x4& pb) {
    const float nb = (m[n] == neg_inf() ? 0.f : m[n]) * qk;
    float pv[8], lt = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pv[e] = exp2f_fast(fmaf(s[e >> 2][e & 3], qk, -nb));
      lt += pv[e];
    }
    pb = u32x4{E::pack(pv[0], pv[1]), E::pack(pv[2], pv[3]), E::pack(pv[4], pv[5]),
               E::pack(pv[6], pv[7])};
    return lt;
  }
  __device__ __forceinline__ void tile(const f32x4 (&s)[NC][2], float qk, u32x4 (&pb)[NC]) {
    float lt[NC];
    bool redo = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lt[n] = weights(n, s[n], qk, pb[n]);
      redo = redo || !(lt[n] <= 16384.f) || m[n] == neg_inf();
    }
    if (__builtin_amdgcn_ballot_w64(redo) != 0) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float mx = neg_inf();
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[n][e >> 2][e & 3]);
        mx = quad_max(mx);
        if (mx > m[n] && (m[n] == neg_inf() || (mx - m[n]) * qk > 8.f)) {
          const float a = m[n] == neg_inf() ? 0.f : exp2f_fast((m[n] - mx) * qk);
          l[n] *= a;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[n][dt] *= a;
          m[n] = mx;
        }
        lt[n] = weights(n, s[n], qk, pb[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) l[n] += lt[n];
  }
  static constexpr int kSaved = NC * (4 * DT + 2) * 64;  // floats
  __device__ __forceinline__ void save(float* a, int lane) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(a + ((n * DT + dt) * 64 + lane) * 4) = o[n][dt];
      a[(NC * DT * 4 + n) * 64 + lane] = m[n];
      a[(NC * (DT * 4 + 1) + n) * 64 + lane] = l[n];
    }
  }
  // Adds another wave's rows (the same lanes hold the same rows).
  __device__ __forceinline__ void add(const float* a, int lane, float qk) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float mo = a[(NC * DT * 4 + n) * 64 + lane], lo = a[(NC * (DT * 4 + 1) + n) * 64 + lane];
      const float mn = fmaxf(m[n], mo);
      const float a0 = m[n] == neg_inf() ? 0.f : exp2f_fast((m[n] - mn) * qk);
      const float a1 = mo == neg_inf() ? 0.f : exp2f_fast((mo - mn) * qk);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        o[n][dt] = o[n][dt] * a0 +
                   *reinterpret_cast<const f32x4*>(a + ((n * DT + dt) * 64 + lane) * 4) * a1;
      // (Without an offset a sum is 0, or NaN where the scores were.)
      l[n] = (m[n] == neg_inf() ? l[n] : l[n] * a0) + (mo == neg_inf() ? lo : lo * a1);
      m[n] = mn;
    }
  }
};

// SRC (a tile source): fetch(t) starts tile t's loads and take() makes it the
// current one (kAhead: the loop fetches the next tile before it uses the
// current one); key(i, m) is the A operand of keys 16 i .. and k-step m, whose
// channels start at channel(m, g) in lane group g; values(put) hands the value
// rows to put(row, chunk, 16 bytes).
// Waves per SIMD (few_waves): as many as the registers of O^T and of the tiles
// under way leave room for; left free, the compiler spreads over twice as many
// registers.
constexpr int few_waves(int d, int nc) { return d == 128 ? (nc == 1 ? 3 : 2) : nc == 1 ? 4 : 3; }
template <class E, int D, int NC, class SRC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_waves(D, NC))))
void few_kernel(const RowsParams p) {
  constexpr int NW = 4, BN = kFewKeys, KS = D >= 32 ? D / 32 : 1, DT = D / 16;
  using Rows = FewRows<E, D, NC>;
  union Lds {
    uint8_t v[NW][BN * 2 * D];
    float rows[NW / 2][Rows::kSaved];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  int split, b, hk;
  RowsPlan plan;
  if (p.balance) {
    plan = rows_balanced<BN>(p, (int)blockIdx.x, b, hk, split);
    if (split < 0) return;
  } else {
    split = (int)(blockIdx.x % (uint32_t)p.nsplit);
    const int bhk = (int)(blockIdx.x / (uint32_t)p.nsplit);
    b = bhk / p.Hk;
    hk = bhk - b * p.Hk;
    plan = rows_plan<kFewRows, BN>(p, b, 0);
    if (split >= plan.used) return;
  }
  const int bhk = b * p.Hk + hk;
  const int t1 = min(plan.tiles, (split + 1) * plan.per);

  // Rows that do not exist see what the last row sees; nothing of theirs is
  // stored.
  int pos[NC];
  u32x4 q[NC][KS];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int v = 16 * n + c;
    pos[n] = min(plan.pos0 + v / p.G, plan.hi);
#pragma unroll
    for (int m = 0; m < KS; ++m) {
      q[n][m] = load_q<D>(p, b, hk, v, SRC::channel(m, g));
      if (D < 32 && g >= 2) q[n][m] = u32x4{0u, 0u, 0u, 0u};  // half the contraction is padding
    }
  }

  SRC src(p, plan, b, hk, lane);
  Rows a;
  uint8_t* vt = lds.v[wave];
  // Transposing reads: lane j of a 16-lane group fetches 8 bytes of key 4 g + j / 4,
  // channels 4 (j % 4) .., and receives channel j of keys 4 g .. 4 g + 3.
  const int vkey = 4 * g + (c >> 2), vchunk = (c & 3) >> 1, vsub = 8 * (c & 1);
  int t = split * plan.per + wave;
  if (SRC::kAhead && t < t1) src.fetch(t);
  for (; t < t1; t += NW) {
    const int e0 = t * BN;
    if constexpr (!SRC::kAhead) src.fetch(t);
    src.take();
    if (SRC::kAhead && t + NW < t1) src.fetch(t + NW);
    f32x4 s[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < KS; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x4 k = src.key(i, m);
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][i] = mma16(E{}, k, q[n][m], s[n][i]);
      }
    const TileMask need(p, plan, plan.lo, plan.hi, e0, BN);
    if (need.end || need.edge) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s[n][e >> 2][e & 3] =
              masked_score(s[n][e >> 2][e & 3], e0 + 16 * (e >> 2) + 4 * g + (e & 3),
                           RowMask(p, plan, pos[n]), plan, true, true);
    }
    // A wave's LDS accesses run in issue order: only the compiler must keep the
    // last tile's reads, these writes and the reads below in theirs.
    __builtin_amdgcn_wave_barrier();
    src.values([&](int row, int chunk, u32x4 x) __attribute__((always_inline)) {
      *reinterpret_cast<u32x4*>(vt + few_off<D>(row, chunk)) = x;
    });
    u32x4 pb[NC];
    a.tile(s, p.qk_scale, pb);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      // Contraction index 8 g + e is key 4 g + e, or 16 + 4 g + e - 4: the order
      // of the weights.
      const fp16x4_lds r0 = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
          (FAS_LDS fp16x4_lds*)(vt + few_off<D>(vkey, 2 * dt + vchunk) + vsub));
      const fp16x4_lds r1 = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
          (FAS_LDS fp16x4_lds*)(vt + few_off<D>(vkey + 16, 2 * dt + vchunk) + vsub));
      const u32x2 x = __builtin_bit_cast(u32x2, r0), y = __builtin_bit_cast(u32x2, r1);
#pragma unroll
      for (int n = 0; n < NC; ++n) a.o[n][dt] = mma16(E{}, u32x4{x.x, x.y, y.x, y.y}, pb[n], a.o[n][dt]);
    }
    if constexpr (SRC::kNanBlocks) {
      const uint32_t nan = src.nan();
      if (__builtin_amdgcn_ballot_w64(nan != 0) != 0) {
        for (int row = 0; row < BN; ++row) {
          const uint32_t f = SRC::nan_row(nan, row);
          if (f == 0) continue;
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            const bool sees = row_sees(RowMask(p, plan, pos[n]), plan, e0 + row);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
              if ((f >> (dt / 2)) & 1u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  a.o[n][dt][r] = sees ? __builtin_nanf("") : a.o[n][dt][r];
          }
        }
      }
    }
  }
  // The four waves' rows, pairwise.
  __syncthreads();
  if (wave >= 2) a.save(lds.rows[wave - 2], lane);
  __syncthreads();
  if (wave < 2) a.add(lds.rows[wave], lane, p.qk_scale);
  __syncthreads();
  if (wave == 1) a.save(lds.rows[0], lane);
  __syncthreads();
  if (wave != 0) return;
  a.add(lds.rows[0], lane, p.qk_scale);
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int v = 16 * n + c;
    const float l = quad_add(a.l[n]);
    if (v >= p.G * p.M) continue;
    const int i = v / p.G, h = hk * p.G + (v - i * p.G);
    const bool live = i < plan.cnt;
    if (plan.used > 1) {
      const int64_t row = ((int64_t)bhk * p.nsplit + split) * p.Rpad + v;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(p.part_o + row * D + 16 * dt + 4 * g) = a.o[n][dt];
      if (g == 0)
        *reinterpret_cast<f32x2*>(p.part_ml + 2 * row) =
            f32x2{a.m[n] == neg_inf() ? neg_inf() : a.m[n] * p.qk_scale, l};
      continue;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = p.o + b * p.so0 + h * p.so1 + (int64_t)i * p.so2;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const f32x4 o = a.o[n][dt] * inv;
      *reinterpret_cast<u32x2*>(out + 16 * dt + 4 * g) =
          live ? u32x2{E::pack(o[0], o[1]), E::pack(o[2], o[3])} : u32x2{0u, 0u};
    }
    if (g == 0 && p.lse != nullptr)
      p.lse[b * p.sl0 + h * p.sl1 + (int64_t)i * p.sl2] =
          !live || l == 0.f ? neg_inf()
                            : (a.m[n] * p.qk_scale + log2f_fast(l)) * 0.69314718055994531f;
  }
}

// ---------------------------------------------------------------- many rows

// SRC (a tile source): fetch(t, stage) starts tile t on its way to an LDS
// stage, land(stage) completes it for this thread; keys(stage) and
// values(stage) are its swizzled tiles; nan_blocks(stage, lane) says which of
// tile row `lane`'s V blocks read as NaN (kNanBlocks sources: those blocks are
// staged as zeros).
constexpr uint32_t kMi355Cus = 256;
template <class E, int D, class SRC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void rows_kernel(const RowsParams p) {
  constexpr int BM = kRowsBlock, BN = kRowsKeys, KS = D / 16, DB = (D + 31) / 32;
  __shared__ __attribute__((aligned(16))) typename SRC::Lds lds;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, g = lane >> 5;
  uint32_t id = blockIdx.x;
  const int split = (int)(id % (uint32_t)p.nsplit);
  id /= (uint32_t)p.nsplit;
  const int nbh = p.B * p.Hk;
  const int bhk = (int)(id % (uint32_t)nbh);
  const int rb = p.nrb - 1 - (int)(id / (uint32_t)nbh);  // longest first
  const int b = __builtin_amdgcn_readfirstlane(bhk / p.Hk), hk = bhk - b * p.Hk;
  const RowsPlan plan = rows_plan<BM, BN>(p, b, rb);
  if (split >= plan.used) return;
  const int t0 = split * plan.per, t1 = min(plan.tiles, t0 + plan.per);

  // Rows that do not exist see what the last row sees; nothing of theirs is
  // stored.
  const int row0 = rb * BM + 32 * wave, v = row0 + c;
  const int pos = min(plan.pos0 + v / p.G, plan.hi);
  // Positions of the wave's live rows (none: whi = -1); it skips tiles that
  // none of them sees.
  const int wlo = plan.pos0 + row0 / p.G;
  const int whi = row0 / p.G < plan.cnt ? min(plan.pos0 + (row0 + 31) / p.G, plan.hi) : -1;
  u32x4 q[KS];
#pragma unroll
  for (int m = 0; m < KS; ++m) q[m] = load_q<D>(p, b, hk, v, 16 * m + 8 * g);

  const RowMask mask(p, plan, pos);
  // In tiles of the list: the wave's rows see nothing from tile w_end on nor in
  // tiles [w_hide, w_first); tiles before w_edge may cross a row's window, those
  // from w_last on a row's own position; the others need no mask.
  const int first = wlo - p.window - plan.shift + 1;
  const int w_end = whi < 0 ? 0 : (whi - plan.shift) / BN + 1;
  const int w_hide = (plan.hide + BN - 1) / BN, w_first = max(0, first) / BN;
  const int w_edge = (max(0, whi - p.window - plan.shift + 1) + BN - 1) / BN;
  const int w_last = max(0, wlo - plan.shift + 1) / BN;

  SRC src(p, plan, b, hk, lds);
  SoftRows<E, D, 2> a;
  if (t0 < t1) {
    src.fetch(t0, 0);
    src.land(0);
  }
  lds_barrier();
  auto step = [&](int t, auto stage_tag) __attribute__((always_inline)) {
    constexpr int stage = decltype(stage_tag)::value;
    const int e0 = t * BN;
    if (t + 1 < t1) src.fetch(t + 1, stage ^ 1);
    if (t < w_end && !(t >= w_hide && t < w_first)) {
      const uint16_t *kt = src.keys(stage), *vt = src.values(stage);
      f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        s[0] = E::mma(lds_row_chunk<D>(kt, perm_row(c), m, g), q[m], s[0]);
        s[1] = E::mma(lds_row_chunk<D>(kt, 32 + perm_row(c), m, g), q[m], s[1]);
      }
      sched_score_tile<KS, 0>();
      // (A copy of the step without these branches needs more registers than
      // two waves a SIMD have.)
      auto apply = [&](bool end, bool edge) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[kb][r] = masked_score(s[kb][r], e0 + 32 * kb + acc_row(r, g), mask, plan, end, edge);
      };
      if (t >= w_last) apply(true, false);
      if (t < w_edge) apply(false, true);
      u32x4 pb[4];
      a.tile(s, p.qk_scale, pb);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int cs = 0; cs < 4; ++cs)
          a.o[db] = E::mma(lds_vt_operand<D>(vt, db, cs, lane), pb[cs], a.o[db]);
      if constexpr (SRC::kNanBlocks) {
        const uint32_t nan = src.nan_blocks(stage, lane);
        if (__builtin_amdgcn_ballot_w64(nan != 0) != 0)
          set_nan_rows(a, mask, plan, e0, [&](int row) {
            return (uint32_t)__builtin_amdgcn_readlane((int)nan, row);
          });
      }
    }
    if (t + 1 < t1) src.land(stage ^ 1);
    lds_barrier();
  };
  // Two workgroups share a CU and the older one's waves go first: where the grid is
  // one round, it ended after 110 us and the younger one, alone then, after 140 (B2
  // H32/8 M512 N8000 D128 4 bits, in two parts).  So the younger one goes first for
  // half its tiles: the call 157.8 us, so 153; B4 M256 N4000 D64 57.8, 55.0.  (In
  // grids of several rounds the next workgroups even it out: B1 H32/8 S8192 window
  // 256 62 us, with this 70.)
  const bool younger = gridDim.x <= 2 * kMi355Cus && blockIdx.x >= kMi355Cus;
  const int half = younger ? t0 + (t1 - t0) / 2 : t1;
  if (younger) __builtin_amdgcn_s_setprio(1);
  for (int t = t0; t < t1; t += 2) {
    if (t >= half) __builtin_amdgcn_s_setprio(0);
    step(t, std::integral_constant<int, 0>{});
    if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
  }
  store_rows<E, D, 2>(p, a, plan, b, hk, v, split, g);
}

// ---------------------------------------------------------------- merge

// The plan of virtual row v, as the kernel that wrote its parts had it.
template <int BM, int BN>
__device__ __forceinline__ RowsPlan merge_plan(const RowsParams& p, int b, int v) {
  RowsPlan c = rows_plan<BM, BN>(p, b, v / BM);
  if (BM == kFewRows && p.balance) {
    c.per = *p.part_per;
    c.used = max(1, (c.tiles + c.per - 1) / c.per);
  }
  return c;
}
// O (four channels from d0 on) and L of virtual row v, from the parts' sum acc
// and l relative to the base-2 offset mx.
template <class E>
__device__ __forceinline__ void merge_store(const RowsParams& p, const RowsPlan& c, int b, int hk,
                                            int v, int d0, f32x4 acc, float mx, float l) {
  const int i = v / p.G, h = hk * p.G + (v - i * p.G);
  const bool live = i < c.cnt;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(p.o + b * p.so0 + h * p.so1 + (int64_t)i * p.so2 + d0) =
      live ? u32x2{E::pack(acc[0] * inv, acc[1] * inv), E::pack(acc[2] * inv, acc[3] * inv)}
           : u32x2{0u, 0u};
  if (d0 == 0 && p.lse != nullptr)
    p.lse[b * p.sl0 + h * p.sl1 + (int64_t)i * p.sl2] =
        !live || l == 0.f ? neg_inf() : (mx + log2f_fast(l)) * 0.69314718055994531f;
}

// Row v of KV head bhk: offset M = max of the parts' offsets, weights
// 2^(m - M), L = sum w l, O = sum w O / L.  (A part without an offset has l = 0,
// or NaN where its scores were.)
//
// At most kMergeFew parts a row: D / 4 threads a row, four channels each, all
// parts' loads under way together.  (A workgroup a row, as below, took 53 us for
// the 32768 rows in two parts of B2 H32 M512.)
template <class E, int D, int BM, int BN>
__global__ __launch_bounds__(256) void merge_few_kernel(const RowsParams p) {
  constexpr int CH = D / 4, RPB = 256 / CH;
  const int rows = p.G * p.M, blocks = (rows + RPB - 1) / RPB;
  const int bhk = (int)(blockIdx.x / (uint32_t)blocks);
  const int v = (int)(blockIdx.x - (uint32_t)bhk * (uint32_t)blocks) * RPB + (int)threadIdx.x / CH;
  if (v >= rows) return;
  const int b = bhk / p.Hk, hk = bhk - b * p.Hk, d0 = 4 * ((int)threadIdx.x % CH);
  const RowsPlan plan = merge_plan<BM, BN>(p, b, v);
  if (plan.used == 1) return;
  const int64_t row0 = (int64_t)bhk * p.nsplit * p.Rpad + v;
  f32x2 ml[kMergeFew];
  f32x4 x[kMergeFew];
  float mx = neg_inf();
#pragma unroll
  for (int s = 0; s < kMergeFew; ++s) {
    const bool has = s < plan.used;
    const int64_t row = row0 + (int64_t)(has ? s : 0) * p.Rpad;
    ml[s] = *reinterpret_cast<const f32x2*>(p.part_ml + 2 * row);
    x[s] = *reinterpret_cast<const f32x4*>(p.part_o + row * D + d0);
    if (!has) ml[s] = f32x2{neg_inf(), 0.f};
    mx = fmaxf(mx, ml[s].x);
  }
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll
  for (int s = 0; s < kMergeFew; ++s) {
    if (s >= plan.used) continue;
    const float w = ml[s].x == neg_inf() ? 0.f : exp2f_fast(ml[s].x - mx);
    l += ml[s].x == neg_inf() ? ml[s].y : w * ml[s].y;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, x[s][e], acc[e]);
  }
  merge_store<E>(p, plan, b, hk, v, d0, acc, mx, l);
}

// More parts: one workgroup a row.  Thread s holds part s's weight, then
// 1024 / D threads share the parts of each group of four channels.
template <class E, int D, int BM, int BN>
__global__ __launch_bounds__(256) void merge_kernel(const RowsParams p) {
  constexpr int CH = D / 4, WAYS = 256 / CH;
  __shared__ float wgt[kRowsMaxSplits];
  __shared__ float red[2][4];
  __shared__ f32x4 part[WAYS][CH];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int rows = p.G * p.M;
  const int bhk = (int)(blockIdx.x / (uint32_t)rows), v = (int)(blockIdx.x - (uint32_t)bhk * (uint32_t)rows);
  const int b = bhk / p.Hk, hk = bhk - b * p.Hk;
  const RowsPlan plan = merge_plan<BM, BN>(p, b, v);
  if (plan.used == 1) return;
  const int64_t row0 = (int64_t)bhk * p.nsplit * p.Rpad + v;
  static_assert(kRowsMaxSplits == 256, "one part a thread");
  f32x2 ml{neg_inf(), 0.f};
  if (tid < plan.used) ml = *reinterpret_cast<const f32x2*>(p.part_ml + 2 * (row0 + (int64_t)tid * p.Rpad));
  float mx = ml.x;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
  if ((tid & 63) == 0) red[0][wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float w = ml.x == neg_inf() ? 0.f : exp2f_fast(ml.x - mx);
  wgt[tid] = w;
  float l = ml.x == neg_inf() ? ml.y : w * ml.y;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) l += __shfl_xor(l, i);
  if ((tid & 63) == 0) red[1][wave] = l;
  __syncthreads();
  l = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  const int ch = tid % CH, way = tid / CH;
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = way; s < plan.used; s += WAYS) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + (row0 + (int64_t)s * p.Rpad) * D + 4 * ch);
    const float ws = wgt[s];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(ws, x[e], acc[e]);
  }
  part[way][ch] = acc;
  __syncthreads();
  if (way != 0) return;
  for (int s = 1; s < WAYS; ++s) acc += part[s][ch];
  merge_store<E>(p, plan, b, hk, v, 4 * ch, acc, mx, l);
}

}  // namespace fas
