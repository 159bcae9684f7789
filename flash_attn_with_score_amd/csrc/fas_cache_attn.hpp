// gfx950 attention over the quantised KV cache (fas_cache.hpp: its form;
// fas_rows.hpp: which keys a row sees, and what is shared with dense keys).
//
// few_kernel runs with CacheFewSource: a wave's codes come straight from memory
// into registers, one tile ahead.  K codes become the A operand of S^T = K Q^T in
// place: the contraction runs over the channels in the order in which a lane
// holds them, a quarter of a row each (one scale at D = 128), and Q is loaded in
// the same order.  V codes are converted on their way into the wave's LDS tile.
// rows_kernel runs with CacheSource: the codes of the next tile are fetched
// before the products of the current one and converted into LDS after them.
//
// Keys past len are never taken as values: their row index is clamped to the
// last key and their weight is 0.  A weight of 0 would still turn a NaN value
// into NaN, and values of partly visible tiles may be NaN for rows that do not
// see them, so V blocks that read as NaN (scale byte 255) enter the product as
// zeros, and the rows that see such a block are set to NaN afterwards.
#pragma once
#include "fas_cache.hpp"
#include "fas_rows.hpp"

namespace fas {

// ---------------------------------------------------------------- few rows

// Tiles of 32 cache rows for few_kernel, in registers, one tile ahead.
template <class E, int D, int BITS>
struct CacheFewSource {
  static constexpr bool kAhead = true, kNanBlocks = true;
  static constexpr int KL = D >= 32 ? 4 : 2;   // lanes that share a key row
  static constexpr int KC = D / KL;            // channels a lane holds of it
  static constexpr int VL = KL, VR = VL / 2;   // value rows a lane holds parts of
  static constexpr int WPL = KC * BITS / 32;   // words of codes of such a part
  struct Tile {
    uint32_t kw[2][WPL], vw[VR][WPL], ks[2], vs[VR];
  };
  Tile cur, next;
  const RowsPlan& plan;
  const uint8_t *kc, *ks, *vc, *vs;
  const int64_t skc, sks, svc, svs;
  const int c, kpart, vrow, vpart;

  __device__ __forceinline__ CacheFewSource(const RowsParams& p, const RowsPlan& plan_, int b,
                                            int hk, int lane)
      : plan(plan_), skc(p.sk2), sks(p.sks2), svc(p.sv2), svs(p.svs2), c(lane & 15),
        kpart((lane >> 4) % KL), vrow(lane / VL), vpart(lane % VL) {
    kc = p.k + b * p.sk0 + hk * p.sk1 + 4 * WPL * kpart;
    ks = p.ks + b * p.sks0 + hk * p.sks1 + kpart * KC / 32;
    vc = p.v + b * p.sv0 + hk * p.sv1 + 4 * WPL * vpart;
    vs = p.vs + b * p.svs0 + hk * p.svs1 + vpart * KC / 32;
  }
  static __device__ __forceinline__ void words(uint32_t (&w)[WPL], const uint8_t* src) {
    if constexpr (WPL >= 4) {
#pragma unroll
      for (int i = 0; i < WPL / 4; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4*>(src)[i];
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else if constexpr (WPL == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(src);
      w[0] = x.x; w[1] = x.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
  }
  __device__ __forceinline__ void fetch(int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = plan.row(t * kFewKeys + 16 * i + c);
      words(next.kw[i], kc + r * skc);
      next.ks[i] = ks[r * sks];
    }
#pragma unroll
    for (int i = 0; i < VR; ++i) {
      const int64_t r = plan.row(t * kFewKeys + 16 * i + vrow);
      words(next.vw[i], vc + r * svc);
      next.vs[i] = vs[r * svs];
    }
  }
  __device__ __forceinline__ void take() { cur = next; }
  // Channel of k-step m that lane group g contributes first.
  static __device__ __forceinline__ int channel(int m, int g) { return (g % KL) * KC + 8 * m; }
  __device__ __forceinline__ u32x4 key(int i, int m) const {
    return cache_unpack8<E, BITS>(cur.kw[i] + m * BITS / 4, cache_scale(cur.ks[i]));
  }
  // Bit i: this lane's part of value row 16 i + vrow reads as NaN.
  __device__ __forceinline__ uint32_t nan() const {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < VR; ++i) n |= cur.vs[i] == 0xffu ? 1u << i : 0u;
    return n;
  }
  // The tile's value rows, NaN blocks as zeros.
  template <class PUT>
  __device__ __forceinline__ void values(PUT&& put) const {
#pragma unroll
    for (int i = 0; i < VR; ++i)
#pragma unroll
      for (int m = 0; m < KC / 8; ++m) {
        const u32x4 x = cache_unpack8<E, BITS>(cur.vw[i] + m * BITS / 4, cache_scale(cur.vs[i]));
        put(16 * i + vrow, vpart * (KC / 8) + m,
            cur.vs[i] == 0xffu ? u32x4{0u, 0u, 0u, 0u} : x);
      }
  }
  // Which 32-channel blocks of value row `row` read as NaN, from the lanes' nan().
  static __device__ __forceinline__ uint32_t nan_row(uint32_t n, int row) {
    uint32_t f = 0;
#pragma unroll
    for (int j = 0; j < VL; ++j)
      f |= (((uint32_t)__builtin_amdgcn_readlane((int)n, (row % (64 / VL)) * VL + j) >>
             (row / (64 / VL))) & 1u)
           << (j * KC / 32);
    return f;
  }
};

// ---------------------------------------------------------------- many rows

// Tiles of 64 cache rows for rows_kernel: 256 threads, each with a run of up to
// 32 channels of one row.
template <class E, int D, int BITS>
struct CacheSource {
  static constexpr bool kNanBlocks = true;
  static constexpr int TILE = kRowsKeys * D;
  static constexpr int UPT = D >= 32 ? D / 32 : 1;  // units of 8 channels a thread converts
  static constexpr int UPR = D / 8;                 // units per row
  static constexpr int WPT = UPT * BITS / 4;        // words of codes
  static constexpr int GROUPS = D >= 32 ? D / 32 : 1;
  struct Lds {
    uint16_t kv[2][2][TILE];
    uint8_t nan[2][kRowsKeys][4];
  };
  Lds& lds;
  const RowsPlan& plan;
  const int row, unit;
  const bool stager;
  const uint8_t *kc, *ks, *vc, *vs;
  const int64_t skc, sks, svc, svs;
  uint32_t kw[WPT], vw[WPT], ksb = 0, vsb = 0;

  // The row of the j-th group of threads: neighbours take rows whose chunks the
  // swizzle puts on different banks (in order, four of the threads that write
  // at once hit each bank at D = 128: B2 H32/8 M512 N8000 4 bits 233 us, so 210;
  // two at D = 64, where another order measured the same).
  static __device__ __forceinline__ int row_of(int j) {
    return D == 128 ? (j & ~15) | ((j & 3) << 2) | ((j >> 2) & 3) : j;
  }
  __device__ __forceinline__ CacheSource(const RowsParams& p, const RowsPlan& plan_, int b, int hk,
                                         Lds& lds_)
      : lds(lds_), plan(plan_), row(row_of((int)threadIdx.x * UPT / UPR)),
        unit((int)threadIdx.x * UPT % UPR),
        stager(D >= 32 || (int)threadIdx.x < kRowsKeys * UPR),
        kc(p.k + b * p.sk0 + hk * p.sk1 + unit * BITS),
        ks(p.ks + b * p.sks0 + hk * p.sks1 + unit / 4),
        vc(p.v + b * p.sv0 + hk * p.sv1 + unit * BITS),
        vs(p.vs + b * p.svs0 + hk * p.svs1 + unit / 4),
        skc(p.sk2), sks(p.sks2), svc(p.sv2), svs(p.svs2) {}

  static __device__ __forceinline__ void words(uint32_t (&w)[WPT], const uint8_t* src) {
    if constexpr (WPT >= 4) {
#pragma unroll
      for (int i = 0; i < WPT / 4; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4*>(src)[i];
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else if constexpr (WPT == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(src);
      w[0] = x.x; w[1] = x.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
  }
  __device__ __forceinline__ void fetch(int t, int) {
    if (!stager) return;
    const int64_t r = plan.row(t * kRowsKeys + row);
    words(kw, kc + r * skc);
    words(vw, vc + r * svc);
    ksb = ks[r * sks];
    vsb = vs[r * svs];
  }
  __device__ __forceinline__ void land(int stage) {
    if (!stager) return;
    const bool nan = vsb == 0xffu;
    const float fk = cache_scale(ksb), fv = cache_scale(nan ? 0x7fu : vsb);
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int off = tile_off<D>(row, unit + i);
      *reinterpret_cast<u32x4*>(&lds.kv[stage][0][off]) =
          cache_unpack8<E, BITS>(kw + i * BITS / 4, fk);
      const u32x4 x = cache_unpack8<E, BITS>(vw + i * BITS / 4, fv);
      *reinterpret_cast<u32x4*>(&lds.kv[stage][1][off]) = nan ? u32x4{0u, 0u, 0u, 0u} : x;
    }
    // (Where a block spans two threads both write the same byte.)
    lds.nan[stage][row][unit / 4] = nan ? 1 : 0;
    if (GROUPS < 4 && unit == 0)
      for (int i = GROUPS; i < 4; ++i) lds.nan[stage][row][i] = 0;
  }
  __device__ __forceinline__ const uint16_t* keys(int stage) const { return lds.kv[stage][0]; }
  __device__ __forceinline__ const uint16_t* values(int stage) const { return lds.kv[stage][1]; }
  __device__ __forceinline__ uint32_t nan_blocks(int stage, int lane) const {
    const uint32_t n = *reinterpret_cast<const uint32_t*>(lds.nan[stage][lane]);
    return (n & 1u) | ((n >> 7) & 2u) | ((n >> 14) & 4u) | ((n >> 21) & 8u);
  }
};

}  // namespace fas
