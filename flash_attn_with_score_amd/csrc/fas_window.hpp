// gfx950 windowed attention over dense keys, forward (rows_kernel and few_kernel
// of fas_rows.hpp with DenseSource and DenseFewSource) and backward.
//
// Query row i is at position p = (N - M) + i and sees key j iff j <= p and
// (j > p - window or j < sinks).  The backward has attention()'s products
// (fas_bwd.hpp: the operand layouts) over the visible pairs alone:
//
//   window_dq_kernel      query-block outer, over tiles of 64 entries of the key
//                         list that RowsPlan describes: S^T, P^T, dS^T,
//                         dQ^T += K^T dS^T.  It first forms its rows' delta and
//                         exponent offsets and leaves them for the next kernel.
//   window_dkdv_kernel    key-block outer: S, P, dP, dS, dV^T += dO^T P,
//                         dK^T += Q^T dS.  The rows that see a block of 128
//                         keys are one run: those at most `window` behind its
//                         last key, or, where the block holds sinks, all later
//                         ones, which is M / (window + 128) times as long.
//                         So the row tiles of all blocks (of all heads) are one
//                         list, block after block, and every workgroup takes
//                         an equal run of it (p.chunk units): parts of a block
//                         at its ends, whole blocks between.  Parts go to fp32
//                         slabs, two a workgroup, that window_reduce_kernel
//                         adds in order.  Where whole blocks are even enough
//                         (p.chunk 0) a workgroup takes one.
//
// A pair that a row does not see has P = 0 and so dS = 0; P and dS are rounded
// to the input type for their products, everything else is fp32.
#pragma once
#include "fas_bwd.hpp"
#include "fas_rows.hpp"

namespace fas {

// Tiles of 64 dense rows by LDS DMA (rows past the last key read as zeros).
template <class E, int D>
struct DenseSource {
  static constexpr bool kNanBlocks = false;
  static constexpr int TILE = kRowsKeys * D;
  struct Lds {
    uint16_t kv[2][2][TILE];
  };
  Lds& lds;
  const RowsPlan& plan;
  const i32x4 wk, wv;
  const TileDma<D> dk, dv;
  static __device__ __forceinline__ i32x4 uniform(i32x4 w) {
    return i32x4{__builtin_amdgcn_readfirstlane(w.x), __builtin_amdgcn_readfirstlane(w.y),
                 __builtin_amdgcn_readfirstlane(w.z), __builtin_amdgcn_readfirstlane(w.w)};
  }
  __device__ __forceinline__ DenseSource(const RowsParams& p, const RowsPlan& plan_, int b, int hk,
                                         Lds& lds_)
      : lds(lds_), plan(plan_),
        wk(make_rsrc_words(p.k + b * p.sk0 + hk * p.sk1, p.k_bytes)),
        wv(make_rsrc_words(p.v + b * p.sv0 + hk * p.sv1, p.v_bytes)),
        dk(__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), (int)threadIdx.x & 63,
           (uint32_t)(p.sk2 >> 1)),
        dv(dk.wave, (int)threadIdx.x & 63, (uint32_t)(p.sv2 >> 1)) {}
  __device__ __forceinline__ void fetch(int t, int stage) {
    // (The descriptors are uniform, but at D = 16, where half the waves load,
    // the compiler moves them to vector registers.)
    dk.fetch(uniform(wk), t * kRowsKeys, plan.ns, plan.shift, lds_addr(lds.kv[stage][0]));
    dv.fetch(uniform(wv), t * kRowsKeys, plan.ns, plan.shift, lds_addr(lds.kv[stage][1]));
  }
  __device__ __forceinline__ void land(int) { vm_wait_all(); }
  __device__ __forceinline__ const uint16_t* keys(int stage) const { return lds.kv[stage][0]; }
  __device__ __forceinline__ const uint16_t* values(int stage) const { return lds.kv[stage][1]; }
};

// Tiles of 32 dense rows for few_kernel, in registers.  (No tile ahead: a
// tile of 32 keys takes 64 registers at D = 128, and the other waves' loads
// cover the wait.)
template <class E, int D>
struct DenseFewSource {
  static constexpr bool kAhead = false, kNanBlocks = false;
  static constexpr int KS = D >= 32 ? D / 32 : 1, VL = D / 16;
  u32x4 k[2][KS], v[VL];
  const RowsPlan& plan;
  const uint8_t *kp, *vp;
  const int64_t sk, sv;
  const int c, lane;
  __device__ __forceinline__ DenseFewSource(const RowsParams& p, const RowsPlan& plan_, int b,
                                            int hk, int lane_)
      : plan(plan_), kp(p.k + b * p.sk0 + hk * p.sk1 + 2 * channel(0, lane_ >> 4)),
        vp(p.v + b * p.sv0 + hk * p.sv1 + 16 * (lane_ % (D / 8))), sk(p.sk2), sv(p.sv2),
        c(lane_ & 15), lane(lane_) {}
  static __device__ __forceinline__ int channel(int m, int g) {
    return D >= 32 ? 32 * m + 8 * g : 8 * (g & 1);
  }
  __device__ __forceinline__ void fetch(int t) {
    const int e0 = t * kFewKeys;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* row = kp + (int64_t)plan.row(e0 + 16 * i + c) * sk;
#pragma unroll
      for (int m = 0; m < KS; ++m) k[i][m] = *reinterpret_cast<const u32x4*>(row + 64 * m);
    }
#pragma unroll
    for (int j = 0; j < VL; ++j)
      v[j] = *reinterpret_cast<const u32x4*>(
          vp + (int64_t)plan.row(e0 + value_row(j)) * sv);
  }
  __device__ __forceinline__ int value_row(int j) const { return (64 * j + lane) / (D / 8); }
  __device__ __forceinline__ void take() {}
  __device__ __forceinline__ u32x4 key(int i, int m) const { return k[i][m]; }
  template <class PUT>
  __device__ __forceinline__ void values(PUT&& put) const {
#pragma unroll
    for (int j = 0; j < VL; ++j) put(value_row(j), lane % (D / 8), v[j]);
  }
};

// 64-row tiles (of one query head) that see key block kb: [lo, lo + n).
__device__ __forceinline__ void window_tiles(const WindowBwdParams& p, int kb, int& lo, int& n) {
  const int k0 = kb * kBwdBlock, rlo = max(0, k0 - p.causal_off);
  const int rhi = k0 < p.sinks ? p.M
                               : (int)min((int64_t)p.M, (int64_t)k0 + kBwdBlock - 1 + p.window -
                                                            p.causal_off);
  lo = rlo / 64;
  n = max(0, (rhi + 63) / 64 - lo);
}
// A block's share of the list in units: its row tiles (of G heads), and
// kBlockUnits for what it costs beside them: K and V, the first tile's way, the
// results.  (Without these a head's last workgroups, whose blocks are short and
// so more, ended at 160 to 169 us where the others took 150: the backward of B1
// H32/8 S4096 D128 window 1024 327 us, with three 315, with one or five 316 to 320.)
__device__ __forceinline__ int window_units(const WindowBwdParams& p, int kb) {
  int lo, n;
  window_tiles(p, kb, lo, n);
  return n > 0 ? n * p.G + kBlockUnits : 0;
}
// Units of key blocks [0, kb) of a KV head, worked out 64 blocks at a time;
// `find` instead: the block that unit `at` falls into, and the units before it.
__device__ __forceinline__ int64_t window_before(const WindowBwdParams& p, int kb) {
  const int lane = (int)threadIdx.x & 63;
  int64_t sum = 0;
  for (int k = 0; k < kb; k += 64) {
    const int n = k + lane < kb ? window_units(p, k + lane) : 0;
    sum += __builtin_amdgcn_readlane(wave_scan(n, [](int x, int y) { return x + y; }), 63);
  }
  return sum;
}
__device__ __forceinline__ int window_find(const WindowBwdParams& p, int64_t at, int64_t& before) {
  const int lane = (int)threadIdx.x & 63;
  before = 0;
  for (int k = 0;; k += 64) {
    const int n = k + lane < p.nkb ? window_units(p, k + lane) : 0;
    const int end = wave_scan(n, [](int x, int y) { return x + y; });
    const int total = __builtin_amdgcn_readlane(end, 63);
    if (at < before + total || k + 64 >= p.nkb) {
      const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before + end <= at));
      if (i > 0) before += __builtin_amdgcn_readlane(end, min(i, 64) - 1);
      return min(k + i, p.nkb - 1);
    }
    before += total;
  }
}

// ---------------------------------------------------------------- dK, dV

// A workgroup's run of the list: block after block, tiles [s0, s1) of each.
struct WindowRun {
  int wg, bhk, kb;
  int tlo, tiles;  // the block's 64-row tiles [tlo, tlo + tiles) of every head
  int s0, s1;      // of its G * tiles, in head order
  int64_t at, stop, before, start;  // units of the list: the run's, those before the block
                                    // in its KV head, and the block's first
  // The run's first block (false: no tiles left for this workgroup).  Runs that
  // follow each other go to one XCD (workgroup i runs on XCD i % 8): they share
  // query rows in its L2.
  __device__ __forceinline__ bool begin(const WindowBwdParams& p) {
    wg = blockIdx.x;
    at = stop = before = 0;
    if (p.chunk > 0) {
      wg = (wg & 7) * ((int)gridDim.x >> 3) + (wg >> 3);
      at = (int64_t)wg * p.chunk;
      stop = min(at + p.chunk, (int64_t)p.B * p.Hk * p.head_units);
      if (at >= stop) return false;
      bhk = (int)(at / p.head_units);
      kb = window_find(p, at - (int64_t)bhk * p.head_units, before);
    } else {
      kb = wg / (p.B * p.Hk);  // longest first: blocks with sinks
      bhk = wg - kb * (p.B * p.Hk);
    }
    set(p);
    return true;
  }
  __device__ __forceinline__ void set(const WindowBwdParams& p) {
    bhk = __builtin_amdgcn_readfirstlane(bhk);
    kb = __builtin_amdgcn_readfirstlane(kb);
    window_tiles(p, kb, tlo, tiles);
    s0 = 0;
    s1 = p.G * tiles;
    start = (int64_t)bhk * p.head_units + before;
    if (p.chunk > 0) {
      s0 = __builtin_amdgcn_readfirstlane((int)max((int64_t)0, at - start - kBlockUnits));
      s1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)s1, stop - start - kBlockUnits));
    }
  }
  __device__ __forceinline__ bool whole(const WindowBwdParams& p) const {
    return s0 == 0 && s1 == p.G * tiles;
  }
  // The next block with rows (blocks that no row sees take no units), if the
  // run reaches its tiles.
  __device__ __forceinline__ bool next(const WindowBwdParams& p) {
    const int units = p.G * tiles + kBlockUnits;
    at = start + units;
    if (p.chunk == 0 || at + kBlockUnits >= stop) return false;
    before += units;
    do {
      if (++kb == p.nkb) {
        kb = 0;
        before = 0;
        ++bhk;
      }
      window_tiles(p, kb, tlo, tiles);
    } while (tiles == 0);
    set(p);
    return true;
  }
  // Slab of this workgroup's part: 2 wg of its run's first block, else 2 wg + 1.
  __device__ __forceinline__ int slab(const WindowBwdParams& p) const {
    return 2 * wg + (start > (int64_t)wg * p.chunk ? 1 : 0);
  }
};

// Which keys of the wave's 32, from key0 on, a run of 32 rows sees, from
// position p0 on: some of them, all of them; and per lane (key key0 + c) the
// row position - key below which it does (a key past N: never).
struct WindowSight {
  int key0, N, window, sinks;
  __device__ __forceinline__ bool live(int p0) const {
    return p0 + 31 >= key0 && (key0 + 31 > p0 - window || key0 < sinks);
  }
  __device__ __forceinline__ bool full(int p0) const {
    return p0 >= key0 + 31 && key0 + 31 < N && (key0 > p0 + 31 - window || key0 + 32 <= sinks);
  }
  __device__ __forceinline__ int reach(int c) const {
    return key0 + c >= N ? 0 : key0 + c < sinks ? 0x7fffffff : window;
  }
};

// dV^T (dv) or dK^T of the wave's keys, register r of block db: key `key`, head
// dim 32 db + acc_row(r, g): to its place, or into the part's slab.
template <class E, int D, int DB>
__device__ __forceinline__ void window_store(const WindowBwdParams& p, const WindowRun& run, bool dv,
                                             const f32x16 (&acc)[DB], int key, int g) {
  const int b = run.bhk / p.Hk, hk = run.bhk - b * p.Hk;
  const float scale = dv ? 1.f : p.scale_signed;
  if (run.whole(p)) {
    if (key >= p.N) return;
    uint16_t* out = dv ? p.dv + b * p.sdv0 + hk * p.sdv1 + (int64_t)key * p.sdv2
                       : p.dk + b * p.sdk0 + hk * p.sdk1 + (int64_t)key * p.sdk2;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int d0 = 32 * db + 16 * hf + 8 * g;
        if (d0 < D) *reinterpret_cast<u32x4*>(out + d0) = pack_b<E>(acc[db] * scale, hf);
      }
    return;
  }
  float* out = p.part + ((int64_t)run.slab(p) * kBwdBlock + key % kBwdBlock) * (2 * D) + (dv ? D : 0);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int d0 = 32 * db + 16 * hf + 8 * g;
      if (d0 < D) {
        const f32x16 x = acc[db] * scale;
        const int r = 8 * hf;
        *reinterpret_cast<f32x4*>(out + d0) = f32x4{x[r], x[r + 1], x[r + 2], x[r + 3]};
        *reinterpret_cast<f32x4*>(out + d0 + 4) = f32x4{x[r + 4], x[r + 5], x[r + 6], x[r + 7]};
      }
    }
}

// dK, dV up to D = 64, and at D = 128 in fp16: four waves, each with both products
// of its 32 keys.  Up to D = 64 two workgroups a CU cover each other's waits (the
// split of the work between two waves that window_dkdv_kernel makes costs them
// more than it gives, their LDS holding one workgroup a CU: B1 H32 S8192 D64
// window 1024, backward, 401 / 477 us).
template <class E, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 128 ? 1 : 2)))
void window_dkdv_small_kernel(const WindowBwdParams p) {
  constexpr int KS = D / 16;
  constexpr int DB = D >= 32 ? D / 32 : 1;
  constexpr int NW = 4;
  constexpr int BK = 32 * NW;  // keys per workgroup
  constexpr int TQ = 64;       // query rows per tile
  constexpr int TILE = TQ * D;

  __shared__ __attribute__((aligned(16))) uint16_t qlds[2][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t glds[2][TILE];  // dO
  __shared__ __attribute__((aligned(16))) float nlds[2][TQ];
  __shared__ __attribute__((aligned(16))) float xlds[2][TQ];       // -delta

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, g = lane >> 5;
  WindowRun run;
  if (!run.begin(p)) return;
  const float qk = p.qk_scale;
  const uint32_t q_base = lds_addr(&qlds[0][0]), g_base = lds_addr(&glds[0][0]);
  const TileDma<D> qdma(wave, lane, (uint32_t)p.sq2), gdma(wave, lane, (uint32_t)p.sg2);

  do {  // one key block, or the part of it in this workgroup's run
    const int b = run.bhk / p.Hk, hk = run.bhk % p.Hk;
    const int h0 = hk * p.G;
    const int key0 = run.kb * BK + 32 * wave;  // this wave's keys [key0, key0 + 32)
    const WindowSight sight{key0, p.N, p.window, p.sinks};
    const int reach = sight.reach(c), tlo = run.tlo, tiles = run.tiles;

    const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.k + b * p.sk0 + hk * p.sk1, p.k_bytes);
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.v + b * p.sv0 + hk * p.sv1, p.v_bytes);
    u32x4 kreg[KS], vreg[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kreg[ks] = buf_load16(rk, (uint32_t)(((key0 + c) * p.sk2 + 16 * ks + 8 * g) * 2)) ^ p.qneg;
      vreg[ks] = buf_load16(rv, (uint32_t)(((key0 + c) * p.sv2 + 16 * ks + 8 * g) * 2));
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kreg[ks]), "+v"(vreg[ks]));

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      dk[db] = f32x16{};
      dv[db] = f32x16{};
    }

    const VtOff vto = vt_offsets<D>(lane);
    const uint32_t rco = row_chunk_offset<D>(perm_row(c), g);

    for (int hh = 0; hh < p.G; ++hh) {
      const int t0 = tlo + max(0, run.s0 - hh * tiles), t1 = tlo + min(tiles, run.s1 - hh * tiles);
      if (t0 >= t1) continue;
      const int h = h0 + hh;
      const int64_t bh = (int64_t)b * p.H + h;
      const i32x4 wq = make_rsrc_words(p.q + b * p.sq0 + h * p.sq1, p.q_bytes);
      const i32x4 wg = make_rsrc_words(p.dout + b * p.sg0 + h * p.sg1, p.g_bytes);
      const float* nlg = p.nl + bh * p.Mpad;
      const float* xg = p.delta + bh * p.Mpad;
      float nst = 0.f, xst = 0.f;
      auto fetch = [&](int t, int s) __attribute__((always_inline)) {
        qdma.fetch(wq, t * TQ, 0, 0, q_base + (uint32_t)(s * TILE * 2));
        gdma.fetch(wg, t * TQ, 0, 0, g_base + (uint32_t)(s * TILE * 2));
        if (tid < TQ) {
          nst = nlg[t * TQ + tid];
          xst = xg[t * TQ + tid];
        }
      };
      auto stash = [&](int s) __attribute__((always_inline)) {
        if (tid < TQ) {
          nlds[s][tid] = nst;
          xlds[s][tid] = xst;
        }
      };
      fetch(t0, 0);
      vm_wait_all();
      stash(0);
      __syncthreads();
      auto step = [&](int t, auto stage_tag) __attribute__((always_inline)) {
        constexpr int stage = decltype(stage_tag)::value;
        const bool more = t + 1 < t1;
        if (more) fetch(t + 1, stage ^ 1);
        const uint16_t* qt = qlds[stage];
        const uint16_t* gt = glds[stage];
        // One 32-row block; masked and unmasked copies of the elementwise part
        // join before the dV / dK products.
        auto body = [&](int qb, bool full) __attribute__((always_inline)) {
          const int r0 = t * TQ + 32 * qb;
          // Register r holds query row r0 + acc_row(r, g) and key key0 + c.
          // Operand fetches go two k-steps ahead of the products that take them,
          // and S and dP alternate.
          __builtin_amdgcn_sched_barrier(0);
          uint32_t ro = rco;
          opaque(ro);
          f32x16 s = f32x16{}, dp, nl;
          load8(dp, &xlds[stage][32 * qb + 8 * g], 0, 0);
          load8(dp, &xlds[stage][32 * qb + 16 + 8 * g], 0, 1);
          u32x4 aq[KS], ag[KS];
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            aq[ks] = lds_row_chunk(qt + 32 * qb * D, ro, ks);
            ag[ks] = lds_row_chunk(gt + 32 * qb * D, ro, ks);
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            s = E::mma(aq[ks], kreg[ks], s);
            dp = E::mma(ag[ks], vreg[ks], dp);
          }
          load8(nl, &nlds[stage][32 * qb + 8 * g], 0, 0);
          load8(nl, &nlds[stage][32 * qb + 16 + 8 * g], 0, 1);
          {
            constexpr int PD = KS < 3 ? KS : 3;
            __builtin_amdgcn_sched_group_barrier(0x100, 4 + 2 * PD, 0);  // DS read
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);  // MFMA
              if (i + PD < KS)
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
              else if (i + PD == KS)
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          VtOff vo = vto;
          opaque(vo);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = exp2f_fast(fmaf(s[r], qk, nl[r]));
          if (!full) {
            int diff = p.causal_off + r0 - (key0 + c);
            asm volatile("" : "+v"(diff));  // (a branch, not 32 selects on every block)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if ((uint32_t)(diff + acc_row(r, g)) >= (uint32_t)reach) s[r] = 0.f;
          }
          u32x4 tg[2 * DB], tq[2 * DB];
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tg[2 * db + h] = lds_vt_operand<D>(gt, vo, db, 2 * qb + h);
              tq[2 * db + h] = lds_vt_operand<D>(qt, vo, db, 2 * qb + h);
            }
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= s[r];
          const u32x4 pb[2] = {pack_b<E>(s, 0), pack_b<E>(s, 1)};
          const u32x4 sb[2] = {pack_b<E>(dp, 0), pack_b<E>(dp, 1)};
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              dv[db] = E::mma(tg[2 * db + h], pb[h], dv[db]);
              dk[db] = E::mma(tq[2 * db + h], sb[h], dk[db]);
            }
          {
            constexpr int PD = 2;  // operand pairs ahead
            __builtin_amdgcn_sched_group_barrier(0x100, 4 * PD, 0);
#pragma unroll
            for (int i = 0; i < 2 * DB; ++i) {
              __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
              if (i + PD < 2 * DB) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            }
          }
        };
        const int p0 = p.causal_off + t * TQ;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
          if (sight.live(p0 + 32 * qb)) body(qb, sight.full(p0 + 32 * qb));
        if (more) {
          vm_wait_all();
          stash(stage ^ 1);
        }
        __syncthreads();
      };
      for (int t = t0; t < t1; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
      }
    }

    window_store<E, D>(p, run, false, dk, key0 + c, g);
    window_store<E, D>(p, run, true, dv, key0 + c, g);
  } while (run.next(p));
}

// dK, dV at D = 128 in bf16: eight waves, two for each 32 keys: one turns S into P and
// accumulates dV, the other turns dP into dS and accumulates dK, a tile later,
// with the P that the first left in LDS.  Each does half the products and holds
// half the accumulators, so two waves a SIMD fit (one that did both took 350
// registers), and one's exponentials and waits run beside the other's products
// (the backward of B1 H32/8 S8192 D128 window 4096: 1533 us, with one wave for
// both 1647).  P passes in fp16: within 2^-11 of its value, and 2^-25 below fp16's
// normal range, an eighth of what rounding dS to bf16 takes.
template <int D>
struct WindowDkdvLds {
  uint16_t q[3][64 * D], g[3][64 * D];  // Q and dO
  u32x4 p[2][4][2][2][64];              // P of two tiles: key wave, 32-row block, half, lane
  float nl[3][64], x[3][64];            // -L log2(e), -delta
};
// One role (FIRST: S, P, dV; else dP, dS, dK), in code of its own: where the two
// shared a loop their accumulators were moved at every join.
template <class E, int D, bool first>
__device__ __forceinline__ void window_dkdv(const WindowBwdParams& p, WindowDkdvLds<D>& lds) {
  constexpr int KS = D / 16;
  constexpr int DB = D >= 32 ? D / 32 : 1;
  constexpr int BK = kBwdBlock;  // keys per workgroup
  constexpr int TQ = 64;         // query rows per tile
  constexpr int TILE = TQ * D;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, g = lane >> 5;
  const int kw = wave & 3;
  WindowRun run;
  if (!run.begin(p)) return;
  const float qk = p.qk_scale;
  // The first waves fetch Q, the second ones dO.
  const TileDma<D> dma(kw, lane, (uint32_t)(first ? p.sq2 : p.sg2));
  const uint32_t dma_base = lds_addr(first ? &lds.q[0][0] : &lds.g[0][0]);
  const VtOff vto = vt_offsets<D>(lane);
  const uint32_t rco = row_chunk_offset<D>(perm_row(c), g);

  do {  // one key block, or the part of it in this workgroup's run
    const int b = __builtin_amdgcn_readfirstlane(run.bhk / p.Hk), hk = run.bhk - b * p.Hk;
    const int h0 = hk * p.G;
    const int key0 = run.kb * BK + 32 * kw;  // this wave's keys [key0, key0 + 32)
    const WindowSight sight{key0, p.N, p.window, p.sinks};
    const int reach = sight.reach(c);

    // K or V (B operand of S = Q K^T or dP = dO V^T): lane holds row key0 + c.
    // K carries the sign of a negative sm_scale.
    u32x4 kv[KS];
    {
      const __amdgpu_buffer_rsrc_t r =
          first ? make_rsrc(p.k + b * p.sk0 + hk * p.sk1, p.k_bytes)
                : make_rsrc(p.v + b * p.sv0 + hk * p.sv1, p.v_bytes);
      const int64_t stride = first ? p.sk2 : p.sv2;
      const uint32_t flip = first ? p.qneg : 0u;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kv[ks] = buf_load16(r, (uint32_t)(((key0 + c) * stride + 16 * ks + 8 * g) * 2)) ^ flip;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kv[ks]));
    }
    f32x16 acc[DB];  // dV^T or dK^T
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
    // The head whose tiles are fetched: its rows of Q or dO, and of nl or -delta.
    i32x4 rsrc;
    const float* rowv;
    auto head = [&](int hh) __attribute__((always_inline)) {
      const int h = h0 + hh;
      rsrc = first ? make_rsrc_words(p.q + b * p.sq0 + h * p.sq1, p.q_bytes)
                   : make_rsrc_words(p.dout + b * p.sg0 + h * p.sg1, p.g_bytes);
      rowv = (first ? p.nl : p.delta) + ((int64_t)b * p.H + h) * p.Mpad + lane;
    };
    // Its tile `t` on its way to stage st; the row values into a register of the
    // waves' first (nl) and fifth (-delta).
    float rv = 0.f;
    auto fetch = [&](int t, int st) __attribute__((always_inline)) {
      dma.fetch(rsrc, t * TQ, 0, 0, dma_base + (uint32_t)(st * TILE * 2));
      if (kw == 0) rv = rowv[t * TQ];
    };
    auto land = [&](int st) __attribute__((always_inline)) {
      vm_wait_all();
      if (kw == 0) (first ? lds.nl[st] : lds.x[st])[lane] = rv;
    };
    // One product pair's schedule: operand fetches two k-steps (pairs) ahead.
    auto row_products = [&](const uint16_t* tile, f32x16 x) __attribute__((always_inline)) {
      uint32_t ro = rco;
      opaque(ro);
      u32x4 a[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) a[ks] = lds_row_chunk(tile, ro, ks);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x = E::mma(a[ks], kv[ks], x);
      return x;
    };
    auto col_products = [&](const uint16_t* tile, int qb, const u32x4 (&w)[2])
                            __attribute__((always_inline)) {
      VtOff vo = vto;
      opaque(vo);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[db] = E::mma(lds_vt_operand<D>(tile, vo, db, 2 * qb + h), w[h], acc[db]);
    };
    auto sched_rows = [&]() __attribute__((always_inline)) {
      constexpr int PD = KS < 4 ? KS : 4;
      __builtin_amdgcn_sched_group_barrier(0x100, 4 + PD, 0);  // DS read
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        if (i + PD < KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    };
    auto sched_cols = [&]() __attribute__((always_inline)) {
      constexpr int PD = 2 * DB < 3 ? 2 * DB : 3;
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * PD, 0);
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + PD < 2 * DB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
    };
    // P of a 32-row block (register r: query row acc_row(r, g), key key0 + c).
    auto weights = [&](int st, int buf, int t) __attribute__((always_inline)) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int p0 = p.causal_off + t * TQ + 32 * qb;
        if (!sight.live(p0)) continue;
        __builtin_amdgcn_sched_barrier(0);
        f32x16 nl;
        load8(nl, &lds.nl[st][32 * qb + 8 * g], 0, 0);
        load8(nl, &lds.nl[st][32 * qb + 16 + 8 * g], 0, 1);
        f32x16 s = row_products(&lds.q[st][32 * qb * D], f32x16{});
        sched_rows();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = exp2f_fast(fmaf(s[r], qk, nl[r]));
        if (!sight.full(p0)) {
          int diff = p0 - (key0 + c);
          asm volatile("" : "+v"(diff));  // (a branch, not 32 selects on every block)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((uint32_t)(diff + acc_row(r, g)) >= (uint32_t)reach) s[r] = 0.f;
        }
        const u32x4 pb[2] = {pack_b<E>(s, 0), pack_b<E>(s, 1)};
#pragma unroll
        for (int h = 0; h < 2; ++h) lds.p[buf][kw][qb][h][lane] = pack_b<F16>(s, h);
        col_products(lds.g[st], qb, pb);
        sched_cols();
      }
    };
    auto grads = [&](int st, int buf, int t) __attribute__((always_inline)) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int p0 = p.causal_off + t * TQ + 32 * qb;
        if (!sight.live(p0)) continue;
        __builtin_amdgcn_sched_barrier(0);
        f32x16 dp;
        load8(dp, &lds.x[st][32 * qb + 8 * g], 0, 0);
        load8(dp, &lds.x[st][32 * qb + 16 + 8 * g], 0, 1);
        dp = row_products(&lds.g[st][32 * qb * D], dp);
        sched_rows();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[8];
          unpack8<F16>(lds.p[buf][kw][qb][h][lane], w);
#pragma unroll
          for (int r = 0; r < 8; ++r) dp[8 * h + r] *= w[r];
        }
        const u32x4 sb[2] = {pack_b<E>(dp, 0), pack_b<E>(dp, 1)};
        col_products(lds.q[st], qb, sb);
        sched_cols();
      }
    };

    // Step i: the first waves take tile i, the second ones tile i - 1, while tile
    // i + 1 arrives: three stages, two buffers of P.
    const int n = run.s1 - run.s0;
    int hh = n > 0 ? run.s0 / run.tiles : 0, tt = run.s0 - hh * run.tiles;  // the tile to fetch next
    int t_prev = 0, t_cur = run.tlo + tt, t_next;
    head(hh);
    if (n > 0) {
      fetch(run.tlo + tt, 0);
      land(0);
    }
    lds_barrier();
    int st_prev = 2, st_cur = 0, st_next = 1;
    for (int i = 0; i <= n && n > 0; ++i) {
      if (++tt == run.tiles) {
        tt = 0;
        head(++hh);
      }
      t_next = run.tlo + tt;
      const bool more = i + 1 < n;
      if (more) fetch(t_next, st_next);
      if constexpr (first) {
        if (i < n) weights(st_cur, i & 1, t_cur);
      } else {
        if (i > 0) grads(st_prev, (i & 1) ^ 1, t_prev);
      }
      if (more) land(st_next);
      lds_barrier();
      t_prev = t_cur;
      t_cur = t_next;
      const int s = st_prev;
      st_prev = st_cur;
      st_cur = st_next;
      st_next = s;
    }

    window_store<E, D>(p, run, first, acc, key0 + c, g);
  } while (run.next(p));
}
template <class E, int D>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void window_dkdv_kernel(const WindowBwdParams p) {
  __shared__ __attribute__((aligned(16))) WindowDkdvLds<D> lds;
  if (__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) < 4)
    window_dkdv<E, D, true>(p, lds);
  else
    window_dkdv<E, D, false>(p, lds);
}

// Key blocks that were dealt to several workgroups: dK, dV as the sum of their
// parts, in order; and blocks that no row sees: zeros.  A workgroup per 256 / (D
// / 8) keys of a block.
template <class E, int D>
__global__ __launch_bounds__(256) void window_reduce_kernel(const WindowBwdParams p) {
  constexpr int CPR = D / 8, KEYS = 256 / CPR, PER = kBwdBlock / KEYS;
  const int sub = (int)(blockIdx.x % PER), item = (int)(blockIdx.x / PER);
  const int bhk = item / p.nkb, kb = item - bhk * p.nkb;
  const int units = window_units(p, kb);
  const int64_t start = (int64_t)bhk * p.head_units + window_before(p, kb);
  const int64_t w0 = (start + kBlockUnits) / p.chunk, w1 = (start + units - 1) / p.chunk;
  if (units > 0 && w0 == w1) return;  // written by its only workgroup
  const int row = sub * KEYS + (int)threadIdx.x / CPR, d0 = 8 * ((int)threadIdx.x % CPR);
  const int key = kb * kBwdBlock + row;
  if (key >= p.N) return;
  float a[8] = {}, v[8] = {};
  if (units > 0) {
#pragma unroll 4
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t slab = 2 * w + (start > w * p.chunk ? 1 : 0);
      const float* src = p.part + (slab * kBwdBlock + row) * (2 * D) + d0;
      const f32x4 a0 = *reinterpret_cast<const f32x4*>(src);
      const f32x4 a1 = *reinterpret_cast<const f32x4*>(src + 4);
      const f32x4 v0 = *reinterpret_cast<const f32x4*>(src + D);
      const f32x4 v1 = *reinterpret_cast<const f32x4*>(src + D + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] += a0[e];
        a[4 + e] += a1[e];
        v[e] += v0[e];
        v[4 + e] += v1[e];
      }
    }
  }
  const int hk = bhk % p.Hk, b = bhk / p.Hk;
  *reinterpret_cast<u32x4*>(p.dk + b * p.sdk0 + hk * p.sdk1 + (int64_t)key * p.sdk2 + d0) =
      u32x4{E::pack(a[0], a[1]), E::pack(a[2], a[3]), E::pack(a[4], a[5]), E::pack(a[6], a[7])};
  *reinterpret_cast<u32x4*>(p.dv + b * p.sdv0 + hk * p.sdv1 + (int64_t)key * p.sdv2 + d0) =
      u32x4{E::pack(v[0], v[1]), E::pack(v[2], v[3]), E::pack(v[4], v[5]), E::pack(v[6], v[7])};
}

// ---------------------------------------------------------------- dQ

template <class E, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void window_dq_kernel(const WindowBwdParams p) {
  constexpr int KS = D / 16;
  constexpr int DB = D >= 32 ? D / 32 : 1;
  constexpr int NW = 4;
  constexpr int BM = 32 * NW;  // query rows per workgroup
  constexpr int BN = 64;       // keys per tile
  constexpr int TILE = BN * D;

  __shared__ __attribute__((aligned(16))) uint16_t klds[2][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t vlds[2][TILE];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, g = lane >> 5;
  const int nbh = p.B * p.H;
  const int bh = blockIdx.x % nbh;
  const int rb = p.nrb - 1 - blockIdx.x / nbh;  // longest row blocks first
  const int b = bh / p.H, h = bh % p.H, hk = h / p.G;
  const int row0 = rb * BM, wrow0 = row0 + 32 * wave, qrow = wrow0 + c;

  const __amdgpu_buffer_rsrc_t rq = make_rsrc(p.q + b * p.sq0 + h * p.sq1, p.q_bytes);
  const __amdgpu_buffer_rsrc_t rg = make_rsrc(p.dout + b * p.sg0 + h * p.sg1, p.g_bytes);
  u32x4 qreg[KS], greg[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qreg[ks] = buf_load16(rq, (uint32_t)((qrow * p.sq2 + 16 * ks + 8 * g) * 2)) ^ p.qneg;
    greg[ks] = buf_load16(rg, (uint32_t)((qrow * p.sg2 + 16 * ks + 8 * g) * 2));
  }
  // nl = -L log2(e), the base-2 exponent offset of the row's weights (-inf, so
  // that P is 0, for rows that see no key and for the padding past M), and
  // -delta = -sum_d O dO, here and for the dK/dV kernel, which runs next.  (A pass
  // of its own over O and dO took 14 us of 339 at B1 H32/8 S4096 D128.)
  float nl = neg_inf(), xl = 0.f;
  if (qrow < p.M) {
    const float L = p.lse[b * p.sl0 + h * p.sl1 + (int64_t)qrow * p.sl2];
    if (L != neg_inf()) nl = -L * kLog2e;
  }
  // O is rounded to the type, from weights that were.  In rows of few keys O is
  // as large as V and that is most of the gradients' error (dQ's norm: 1.6 to
  // 1.77 times a mere rounding's over 100 to 512 causal rows, 1.40 to 1.46 with an
  // exact delta), so a block whose first row sees 128 keys or fewer forms delta =
  // sum_j P dP instead, in a sweep of its own over its keys: the first block of a
  // sequence, which has the shortest list, and all blocks of short windows (the
  // backward of B1 H32/8 S8192 D64: window 129 94 us, window 128 114 us).  At D = 16,
  // where rounding dS for its product costs dQ the most, up to 256 keys.
  const int lo = p.causal_off + row0, hi = min(p.N - 1, lo + BM - 1);
  constexpr int kFew = D == 16 ? 256 : 128;
  const bool sweep = lo < p.window ? lo < kFew : min(lo + 1 - p.window, p.sinks) + p.window <= kFew;
  if (!sweep) {
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(p.o + b * p.so0 + h * p.so1, p.o_bytes);
    u32x4 oreg[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      oreg[ks] = buf_load16(ro, (uint32_t)((qrow * p.so2 + 16 * ks + 8 * g) * 2));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float x[8], y[8];
      unpack8<E>(oreg[ks], x);
      unpack8<E>(greg[ks], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) xl = fmaf(x[e], y[e], xl);
    }
    xl = -xor32_add(xl);
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qreg[ks]), "+v"(greg[ks]));

  // The block's keys as a list, as RowsPlan has it: ns sinks, then the window.
  int ns = 0, shift = 0, hide = 0, ntiles = 0;
  if (hi >= 0) {
    const int first = max(0, lo - p.window + 1);
    ns = min(first, p.sinks);
    shift = first - ns;
    hide = shift > 0 ? ns : p.sinks;
    ntiles = (hi + 1 - shift + BN - 1) / BN;
  }
  auto key_of = [&](int e) __attribute__((always_inline)) { return e < ns ? e : e + shift; };
  const int wlo = p.causal_off + wrow0, whi = wrow0 < p.M ? min(p.N - 1, wlo + 31) : -1;
  const int pos = p.causal_off + qrow;

  const i32x4 wk = make_rsrc_words(p.k + b * p.sk0 + hk * p.sk1, p.k_bytes);
  const i32x4 wv = make_rsrc_words(p.v + b * p.sv0 + hk * p.sv1, p.v_bytes);
  const uint32_t k_base = lds_addr(&klds[0][0]), v_base = lds_addr(&vlds[0][0]);
  const TileDma<D> dk(wave, lane, (uint32_t)p.sk2), dv(wave, lane, (uint32_t)p.sv2);
  auto fetch = [&](int t, int s) __attribute__((always_inline)) {
    dk.fetch(wk, t * BN, ns, shift, k_base + (uint32_t)(s * TILE * 2));
    dv.fetch(wv, t * BN, ns, shift, v_base + (uint32_t)(s * TILE * 2));
  };

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = f32x16{};
  float sum = 0.f;
  const float qk = p.qk_scale;
  const VtOff vto = vt_offsets<D>(lane);
  const uint32_t rco = row_chunk_offset<D>(perm_row(c), g);

  // One tile, towards dQ or (`sums`) towards delta.
  auto step = [&](int t, auto stage_tag, auto sums_tag) __attribute__((always_inline)) {
    constexpr int stage = decltype(stage_tag)::value;
    constexpr bool sums = decltype(sums_tag)::value;
    const bool more = t + 1 < ntiles;
    if (more) fetch(t + 1, stage ^ 1);
    const uint16_t* kt = klds[stage];
    const uint16_t* vt = vlds[stage];
    const int e0 = t * BN;
    // One 32-key sub-block (bwd_dq_kernel has the reasons for its fences).
    auto body = [&](int kb2, bool end, bool edge) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      uint32_t ro = rco;
      opaque(ro);
      u32x4 ak[KS], av[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        ak[ks] = lds_row_chunk(kt + 32 * kb2 * D, ro, ks);
        av[ks] = lds_row_chunk(vt + 32 * kb2 * D, ro, ks);
      }
      // Register r holds list entry e0 + 32 kb2 + acc_row(r, g) for query row qrow.
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = xl;
      s = E::mma(ak[0], qreg[0], f32x16{});
      dp = E::mma(av[0], greg[0], dp);
#pragma unroll
      for (int ks = 1; ks < KS; ++ks) {
        s = E::mma(ak[ks], qreg[ks], s);
        dp = E::mma(av[ks], greg[ks], dp);
      }
      {
        constexpr int PD = KS < 2 ? KS : 2;
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * PD, 0);  // DS read
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);  // MFMA
          if (i + PD < KS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
      }
      // RowMask in entries of the sub-block: those past `last`, and those in
      // [hide, hide + span).  (A branch: with selects on every sub-block the
      // backward of B1 H32/8 S8192 D64 window 1024 took 352 us, so 326; D128 window
      // 4096 1484, 1436.)
      if (end || edge) {
        const int ebase = e0 + 32 * kb2, below = ebase - hide;
        const int span = max(0, pos - p.window - shift + 1 - hide);
        int last = pos - shift - ebase;
        asm volatile("" : "+v"(last));
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (acc_row(r, g) > last || (uint32_t)(acc_row(r, g) + below) < (uint32_t)span)
            s[r] = neg_inf();
      }
      float pr[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) pr[r] = exp2f_fast(fmaf(s[r], qk, nl));
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = pr[r] * dp[r];
      if constexpr (sums) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += dp[r];
        return;
      }
      const u32x4 sb0 = pack_b<E>(dp, 0), sb1 = pack_b<E>(dp, 1);
      __builtin_amdgcn_sched_barrier(0);
      VtOff o = vto;
      opaque(o);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dq[db] = E::mma(lds_vt_operand<D>(kt, o, db, 2 * kb2), sb0, dq[db]);
        dq[db] = E::mma(lds_vt_operand<D>(kt, o, db, 2 * kb2 + 1), sb1, dq[db]);
      }
      {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (i + 2 < 2 * DB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
      }
    };
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      // The sub-block's first and last keys (one that the sinks end in holds
      // keys of both kinds), and the masks that it needs (TileMask).
      const int e = e0 + 32 * kb2, ka = key_of(e), kz = key_of(e + 31);
      if (ka > whi || (kz <= wlo - p.window && ka >= p.sinks)) continue;
      const bool end = e + 31 > wlo - shift;
      const bool edge = e + 32 > hide && max(e, hide) < whi - p.window - shift + 1;
      body(kb2, end, edge);
    }
    if (more) vm_wait_all();
    __syncthreads();
  };
  auto all = [&](auto sums_tag) __attribute__((always_inline)) {
    if (ntiles == 0) return;
    fetch(0, 0);
    vm_wait_all();
    __syncthreads();
    for (int t = 0; t < ntiles; t += 2) {
      step(t, std::integral_constant<int, 0>{}, sums_tag);
      if (t + 1 < ntiles) step(t + 1, std::integral_constant<int, 1>{}, sums_tag);
    }
  };
  if (sweep) {  // (xl is 0: the products are dP itself)
    all(std::true_type{});
    xl = -xor32_add(sum);
  }
  if (g == 0) {
    p.nl[(int64_t)bh * p.Mpad + qrow] = nl;
    p.delta[(int64_t)bh * p.Mpad + qrow] = xl;
  }
  all(std::false_type{});

  // Lane (c, g), register r of block db: row qrow, head dim 32db + acc_row(r, g).
  if (qrow >= p.M) return;
  uint16_t* dqr = p.dq + b * p.sdq0 + h * p.sdq1 + (int64_t)qrow * p.sdq2;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int d0 = 32 * db + 16 * hf + 8 * g;
      if (d0 < D) {
        const f32x16 x = dq[db] * p.scale_signed;
        *reinterpret_cast<u32x4*>(dqr + d0) = pack_b<E>(x, hf);
      }
    }
}

}  // namespace fas
