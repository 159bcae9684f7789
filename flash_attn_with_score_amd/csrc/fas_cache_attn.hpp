// gfx950 attention over the quantised KV cache (fas_cache.hpp: its form;
// fas_rows.hpp: which keys a row sees, and what is shared with dense keys).
//
//   cache_few_kernel    at most 32 virtual rows (decoding).  Bound by the
//                       cache's bytes, so nothing is shared between the waves:
//                       each wave streams tiles of 32 keys of its own straight
//                       from memory into registers, one tile ahead.  K codes
//                       become the A operand of S^T = K Q^T in place (the
//                       contraction runs over the channels in the order in
//                       which a lane holds them, half a row each, and Q is
//                       loaded in the same order); V codes become rows of a
//                       small LDS tile of the wave's, which the transposing
//                       read turns into the A operand of O^T += V^T P^T.
//   rows_kernel         more rows (a chunk of a prompt), with CacheSource: the
//                       codes of the next tile are fetched before the products
//                       of the current one and converted into LDS after them.
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

// Half a row of codes (lane half g: channels g D/2 ..) and its scale bytes.
template <int D, int BITS>
struct HalfRow {
  static constexpr int kWords = D * BITS / 64;
  uint32_t w[kWords];
  uint32_t s;  // one byte, or two (D = 128)
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int g) {
    const uint8_t* src = codes + 4 * kWords * g;
    if constexpr (kWords >= 4) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4*>(src)[i];
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else if constexpr (kWords == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(src);
      w[0] = x.x; w[1] = x.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
    if constexpr (D == 128)
      s = reinterpret_cast<const uint16_t*>(scales)[g];
    else
      s = scales[D == 64 ? g : 0];
  }
  // Channels 8 m .. 8 m + 7 of the half.
  template <class E>
  __device__ __forceinline__ u32x4 get(int m) const {
    return cache_unpack8<E, BITS>(w + m * BITS / 4,
                                  cache_scale(D == 128 ? (s >> (8 * (m / 4))) & 0xffu : s));
  }
};

template <class E, int D, int BITS>
__global__ __launch_bounds__(256) void cache_few_kernel(const RowsParams p) {
  constexpr int NW = 4, BN = kCacheFewKeys, KS = D / 16, DB = (D + 31) / 32;
  constexpr int kChunk0 = D / 16;  // 16-byte chunks of half a row of values
  using Rows = SoftRows<E, D, 1>;
  union Lds {
    uint16_t v[NW][BN * D];
    float rows[NW / 2][Rows::kSaved];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, g = lane >> 5;
  const int split = (int)(blockIdx.x % (uint32_t)p.nsplit), bhk = (int)(blockIdx.x / (uint32_t)p.nsplit);
  const int b = bhk / p.Hk, hk = bhk - b * p.Hk;
  const RowsPlan plan = rows_plan<kCacheFewRows, BN>(p, b, 0);
  if (split >= plan.used) return;
  const int t1 = min(plan.tiles, (split + 1) * plan.per);

  // Rows that do not exist see what the last row sees; nothing of theirs is
  // stored.
  const int pos = min(plan.pos0 + c / p.G, plan.hi);
  u32x4 q[KS];
#pragma unroll
  for (int m = 0; m < KS; ++m) q[m] = load_q<D>(p, b, hk, c, g * (D / 2) + 8 * m);

  const uint8_t* kc = p.k + b * p.sk0 + hk * p.sk1;
  const uint8_t* ks = p.ks + b * p.sks0 + hk * p.sks1;
  const uint8_t* vc = p.v + b * p.sv0 + hk * p.sv1;
  const uint8_t* vs = p.vs + b * p.svs0 + hk * p.svs1;
  HalfRow<D, BITS> kn, vn;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int k0 = plan.tile(t) * BN;
    const int64_t kr = min(k0 + perm_row(c), plan.len - 1), vr = min(k0 + c, plan.len - 1);
    kn.load(kc + kr * p.sk2, ks + kr * p.sks2, g);
    vn.load(vc + vr * p.sv2, vs + vr * p.svs2, g);
  };
  Rows a;
  uint16_t* vt = lds.v[wave];
  int t = split * plan.per + wave;
  if (t < t1) fetch(t);
  for (; t < t1; t += NW) {
    const int k0 = plan.tile(t) * BN;
    const HalfRow<D, BITS> kr = kn;
    HalfRow<D, BITS> vr = vn;
    if (t + NW < t1) fetch(t + NW);
    f32x16 s[1] = {f32x16{}};
#pragma unroll
    for (int m = 0; m < KS; ++m) s[0] = E::mma(kr.template get<E>(m), q[m], s[0]);
    if (!rows_full(p, plan, k0, BN)) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!row_sees(p, pos, k0 + acc_row(r, g))) s[0][r] = neg_inf();
    }
    // This lane's NaN blocks as bits of the row's blocks.
    uint32_t nan = 0;
    if constexpr (D == 128) {
      nan = ((vr.s & 0xffu) == 0xffu ? 1u : 0u) | ((vr.s >> 8) == 0xffu ? 2u : 0u);
      nan <<= 2 * g;
    } else {
      nan = vr.s == 0xffu ? (D == 64 ? 1u << g : 1u) : 0u;
    }
    const bool any_nan = __builtin_amdgcn_ballot_w64(nan != 0) != 0;
    if (any_nan) {
#pragma unroll
      for (int m = 0; m < KS; ++m)
        if ((nan >> (D == 128 ? 2 * g + m / 4 : D == 64 ? g : 0)) & 1u)
#pragma unroll
          for (int i = 0; i < BITS / 4; ++i) vr.w[m * BITS / 4 + i] = 0u;
      if constexpr (D == 128)
        vr.s = ((vr.s & 0xffu) == 0xffu ? 0x7fu : vr.s & 0xffu) |
               ((vr.s >> 8) == 0xffu ? 0x7f00u : vr.s & 0xff00u);
      else
        vr.s = vr.s == 0xffu ? 0x7fu : vr.s;
    }
    // V rows into the wave's tile.  A wave's LDS accesses run in issue order:
    // only the compiler must keep the last tile's reads, these writes and the
    // reads below in theirs.
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m = 0; m < KS; ++m)
      *reinterpret_cast<u32x4*>(vt + tile_off<D>(c, kChunk0 * g + m)) = vr.template get<E>(m);
    u32x4 pb[2];
    a.tile(s, p.qk_scale, pb);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int cs = 0; cs < 2; ++cs)
        a.o[db] = E::mma(lds_vt_operand<D>(vt, db, cs, lane), pb[cs], a.o[db]);
    if (any_nan)
      set_nan_rows(a, p, pos, k0, [&](int row) {
        return (uint32_t)(__builtin_amdgcn_readlane((int)nan, row) |
                          __builtin_amdgcn_readlane((int)nan, row + 32));
      });
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
  store_rows<E, D, 1>(p, a, plan, b, hk, c, split, g);
}

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

  __device__ __forceinline__ CacheSource(const RowsParams& p, const RowsPlan& plan_, int b, int hk,
                                         Lds& lds_)
      : lds(lds_), plan(plan_), row((int)threadIdx.x * UPT / UPR), unit((int)threadIdx.x * UPT % UPR),
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
    const int64_t r = min(plan.tile(t) * kRowsKeys + row, plan.len - 1);
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
