// wattn_bwd.cu — windowed attention with sinks, backward, on tcgen05 (what wattn.cu takes).
//
// With P = 2^(c S - lse2) from the saved log-sum-exp, delta_i = sum_d dO O and dP = dO v^T:
//   dS = P (dP - delta),  dQ = scale dS k,  dK = scale dS^T q,  dV = P^T dO.
// Two kinds of block of one shape: 128 rows stay (two operand tiles A1, A2), tiles of 64 rows stream by
// (B1, B2). Per streamed tile, T1 = A1 B1^T and T2 = A2 B2^T (fp32, TMEM); two softmax warpgroups,
// each with half of the tile's columns, make P and dS from them and put them back to TMEM in the IO
// dtype (a product's operands have one type): P rounded, dS as its rounding and the rounding of what
// that leaves, multiplied one after the other; then
//   KV: rows are keys (A = k, v; B = q, dO):    dV += P B2,  dK += dS B1
//   Q : rows are queries (A = q, dO; B = k, v): dQ += dS B1
// accumulate in TMEM. T1 and T2 have two buffers, so the MMAs of one tile run under the softmax of
// the other, and each product has a warp of its own to issue it, all of its lanes together (a lane on its
// own takes some 90 cycles an MMA: 219 us for 204 at 2 x 4096 queries, 16 heads of 128, window 512).
// Bound by the softmax warps' chain (TMEM load, exponentials, store, barrier): some 2 k cycles a streamed
// tile, of which the tensor pipe works half. 2 x 4096 queries, 16 heads of 128 on 4, window 512, 4 sinks: 216 us
// with the two small kernels around it, 676 TFLOP/s of its products, dS's twice.
// S and dP are computed in both (7 products for the 5 of one that adds dQ up in memory by
// atomics): nothing is added in an order that changes, and dS is not stored.
//
// delta comes from `out` as the forward stored it: O's rounding to the IO dtype enters dS, times P.
//
// KV walks the query heads of its key head one after the other, so the sum over a shared head's
// queries stays in TMEM. The queries that see a tile's sinks only as sinks, all those past its window,
// are the work of further, shorter blocks behind the tiles' own (a quarter of their length, so that
// they fill the SMs that the last round of tiles leaves idle); their fp32 sums, and the tile's
// own for these rows, are added in order by a last kernel.
//
// f16 has nothing below 2^-24 and ends at 65504, while dS is of the gradients' size. So in f16 both are held
// at a power of two of their size: P at 2^14 times, which its exponent takes along, and dS at 2^14 / 2^e
// times with 2^e above the largest |dP - delta| that there can be, 2 max |dO_i| max |v_j| over the queries
// that see a key and the keys that a query may see; the statistics' kernel finds both. The results'
// factors take the powers out again (2 x 4096 queries as above: 214 us without, 221 so; 1024 queries of 4
// heads 9.7 and 13.6, the clearing of the two maxima being one more node). bf16 has the range of the sums.
//
// Masked keys: P and dS are replaced by 0, and (Q) their rows of the k tile zeroed in shared memory
// before dS k, so that what they hold reaches nothing. A query that sees nothing, and one past the
// end, has -lse2 = -inf, so that its P is 0; (KV, with a mask) its rows of the q and dO tiles are zeroed likewise.
#include <algorithm>
#include "sm100.cuh"
#include "wattn.h"

namespace tops {

struct WattnBwdArgs {
  int Nq, Nk, Hq, Hkv, group, D;
  int left, right, sinks;
  int q_tiles, tiles;    // query tiles, key tiles
  int kv_blocks;         // blocks of KV; Q's are behind them
  int own;               // KV: blocks of the tiles themselves; behind them, for the sinks' late queries,
  int nsb, nx, per;      // of nsb tiles and each query head, nx blocks of `per` streamed tiles
  int keep;              // rows of a part
  int nqp;               // row length of lse2 and delta
  const uint8_t* mask;
  float c, scale;
  const float *lse2, *delta;  // [B][Hq][nqp], negated
  const unsigned* top;        // f16: the largest |dO_i|^2 and |v_j|^2, as bits
  void *dq, *dk, *dv;
  float* part;                // [B][Hkv][nsb][1 + group nx][2][keep][DT]
};

template <int DT>
struct WattnBwdCfg {
  static constexpr int SUB = DT / 64;
  static constexpr int RES = SUB * 128 * 128;  // bytes of a resident tile
  static constexpr int STR = SUB * 64 * 128;   // bytes of a streamed tile
  static constexpr int NST = 4;                // stages of streamed tiles
  static constexpr int ACC = 256;              // TMEM: T1, T2 of buffer s at 128 s and 128 s + 64
  static constexpr int THREADS = 416;
};

template <int DT>
struct WattnBwdSmem {
  using Cfg = WattnBwdCfg<DT>;
  alignas(1024) uint8_t a1[Cfg::RES];
  alignas(1024) uint8_t a2[Cfg::RES];
  alignas(1024) uint8_t b1[Cfg::NST][Cfg::STR];
  alignas(1024) uint8_t b2[Cfg::NST][Cfg::STR];
  alignas(16) float st[Cfg::NST][2][64];  // KV: lse2 and delta of the streamed queries
  uint64_t res_full, full[Cfg::NST], empty[Cfg::NST];
  uint64_t t_full[2], p_full[2], ds_full[2], p_free[2], ds_free[2], acc_done;  // of tile it at it & 1
  uint32_t tmem_base;
  int abort;
};

// f16: P is held at 2^kWattnLift times its size (in the statistics' -lse2)
constexpr float kWattnLift = 14.f;
template <typename T>
__device__ __forceinline__ float wattn_lift() {
  return Elem<T>::kFmt == 0 ? kWattnLift : 0.f;
}
// What dS is multiplied with (f16: P is held at 2^14 times its size; |dP - delta| times `down` is below 1),
// and the factors of dV and, before the scale, of dQ and dK that undo it.
struct WattnScales {
  float down = 1.f, dv = 1.f, ds = 1.f;
};
template <typename T>
__device__ __forceinline__ WattnScales wattn_scales(const unsigned* top) {
  WattnScales s;
  if constexpr (Elem<T>::kFmt == 0) {
    const float most = 2.f * sqrtf(__uint_as_float(top[0])) * sqrtf(__uint_as_float(top[1]));
    const int e = most > 0.f ? ilogbf(most) + 1 : 0;
    s.down = ldexpf(1.f, -e);
    s.dv = ldexpf(1.f, -static_cast<int>(kWattnLift));
    s.ds = ldexpf(s.dv, e);
  }
  return s;
}

// The walk of one block: which tiles stream by.
template <bool KV>
struct WattnWalk {
  int b, hk, row0, total;  // first resident row (key or query), streamed tiles
  int head;                // KV: first query head; Q: the query head
  int qlo, nqb;            // KV: first streamed query, streamed tiles of a head
  int kb, slot;            // KV: the tile, and which of its parts this is (0: its own)
  int late;                // KV: first query that sees the tile's sinks only as sinks
  WattnBlocks<6> blk;      // Q: the key tiles
  __device__ WattnWalk(const WattnBwdArgs& a) : blk(0, 1, 1, 0, 0, 0) {
    if constexpr (KV) {
      const int off = a.Nk - a.Nq;
      int bh, u = blockIdx.x;
      if (u < a.own) {
        bh = u / a.tiles;
        kb = u % a.tiles;
        slot = 0;
      } else {
        u -= a.own;
        slot = 1 + u % (a.nx * a.group);
        u /= a.nx * a.group;
        kb = u % a.nsb;
        bh = u / a.nsb;
      }
      b = bh / a.Hkv;
      hk = bh % a.Hkv;
      row0 = kb * 128;
      late = max(0, min(a.Nq, min(row0 + 127, a.Nk - 1) + a.left + 1 - off));
      head = hk * a.group;
      if (slot == 0) {
        qlo = max(0, row0 - a.right - off) & ~7;
        nqb = (max(0, late - qlo) + 63) >> 6;
        total = nqb * a.group;
      } else {
        head += (slot - 1) / a.nx;
        qlo = (late & ~7) + (slot - 1) % a.nx * a.per * 64;
        total = nqb = min(a.per, (max(0, a.Nq - qlo) + 63) >> 6);
      }
    } else {
      const int u = blockIdx.x - a.kv_blocks, tile = u % a.q_tiles;
      head = u / a.q_tiles % a.Hq;
      b = u / a.q_tiles / a.Hq;
      hk = head / a.group;
      row0 = tile * 128;
      blk = WattnBlocks<6>(row0, a.Nq, a.Nk, a.left, a.right, a.sinks);
      total = blk.n;
      qlo = nqb = kb = slot = late = 0;
    }
  }
  // first row of streamed tile `it`, and its query head
  __device__ int row(int it) const {
    if constexpr (KV) return qlo + it % nqb * 64;
    return blk.key(it);
  }
  // and that of the tile after it (without the division that a walk over several heads takes)
  __device__ int row_after(int row, int it) const {
    if constexpr (KV) return row + 64 == qlo + nqb * 64 ? qlo : row + 64;
    return blk.key(it + 1);
  }
  __device__ int qhead(int it) const {
    if constexpr (KV) return head + it / nqb;
    return head;
  }
};

template <typename T, int DT, bool KV, bool MASK>
__device__ __forceinline__ void wattn_backward_block(const CUtensorMap& map_a1, const CUtensorMap& map_a2,
                                                     const CUtensorMap& map_b1, const CUtensorMap& map_b2,
                                                     const WattnBwdArgs& a) {
  using Cfg = WattnBwdCfg<DT>;
  using E = Elem<T>;
  constexpr int NST = Cfg::NST, SUB = Cfg::SUB;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<WattnBwdSmem<DT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;
  const WattnWalk<KV> walk(a);

  if (threadIdx.x == 0) {
    mbar_init(&sm.res_full, 1);
    for (int s = 0; s < NST; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], KV ? 2 : 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.t_full[s], 2);
      mbar_init(&sm.p_full[s], 8);
      mbar_init(&sm.ds_full[s], 8);
      mbar_init(&sm.p_free[s], 1);
      mbar_init(&sm.ds_free[s], 1);
    }
    mbar_init(&sm.acc_done, KV ? 2 : 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem_base;
  if (a.nsb > 0) pdl_trigger();
  pdl_wait();  // the rows' lse2 and delta come from the kernel before this one

  if (warp == 0) {
    if (lane == 0 && walk.total > 0) {
      const int res_head = KV ? walk.hk : walk.head;
      mbar_expect_tx(&sm.res_full, 2 * Cfg::RES);
#pragma unroll
      for (int s = 0; s < 2 * SUB; ++s) {
        const int sub = s >> 1, half = (s & 1) * 64, at = sub * 128 * 128 + half * 128;
        tma_load_4d(sm.a1 + at, &map_a1, &sm.res_full, sub * 64, res_head, walk.row0 + half, walk.b);
        tma_load_4d(sm.a2 + at, &map_a2, &sm.res_full, sub * 64, res_head, walk.row0 + half, walk.b);
      }
      for (int it = 0; it < walk.total; ++it) {
        const int r = it % NST;
        if (!mbar_wait(&sm.empty[r], ((it / NST) & 1) ^ 1, abort, 521)) break;
        const int row = walk.row(it), h = KV ? walk.qhead(it) : walk.hk;
        mbar_expect_tx(&sm.full[r], 2 * Cfg::STR + (KV ? 512 : 0));
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          tma_load_4d(sm.b1[r] + s * 64 * 128, &map_b1, &sm.full[r], s * 64, h, row, walk.b);
          tma_load_4d(sm.b2[r] + s * 64 * 128, &map_b2, &sm.full[r], s * 64, h, row, walk.b);
        }
        if constexpr (KV) {
          const int64_t at = (static_cast<int64_t>(walk.b) * a.Hq + h) * a.nqp + row;
          bulk_load(sm.st[r][0], a.lse2 + at, 256, &sm.full[r]);
          bulk_load(sm.st[r][1], a.delta + at, 256, &sm.full[r]);
        }
      }
    }
  } else if (warp <= 2) {
    // T1 (warp 1) and T2 (warp 2); a buffer is free once the product that read P (KV: T1's) or dS
    // out of it is done. (Q keeps no P: T1's goes with dS.)
    if (walk.total > 0) {
      const uint32_t idesc = make_idesc_f16(128, 64, E::kFmt, false, false);
      const int ksteps = (a.D + 15) >> 4;
      const uint32_t ra = smem_u32(warp == 1 ? sm.a1 : sm.a2);
      uint64_t* const free = KV && warp == 1 ? sm.p_free : sm.ds_free;
      bool ok = mbar_wait_warp(&sm.res_full, 0, abort, 523);
      for (int it = 0; ok && it < walk.total; ++it) {
        const int r = it % NST, s = it & 1;
        if (!mbar_wait_warp(&sm.full[r], (it / NST) & 1, abort, 522)) break;
        if (!mbar_wait_warp(&free[s], ((it >> 1) & 1) ^ 1, abort, 524)) break;
        tc_fence_after();
        const uint32_t rb = smem_u32(warp == 1 ? sm.b1[r] : sm.b2[r]), t = tbase + s * 128 + (warp - 1) * 64;
        if (elect_lane()) {
#pragma unroll
          for (int kk = 0; kk < DT / 16; ++kk)
            if (kk < ksteps)
              mma_ss(t, make_smem_desc(ra + (kk / 4) * 128 * 128 + (kk % 4) * 32, 16, 1024, kSw128),
                     make_smem_desc(rb + (kk / 4) * 64 * 128 + (kk % 4) * 32, 16, 1024, kSw128), idesc, kk > 0);
          mma_commit(&sm.t_full[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp <= 4) {
    // KV: dV += P B2 (warp 3), dK += dS B1 (warp 4); Q: dQ += dS B1 (warp 4)
    if (KV || warp == 4) {
      const uint32_t idesc = make_idesc_f16(128, DT, E::kFmt, false, true);
      const bool of_p = warp == 3;
      const uint32_t acc = tbase + Cfg::ACC + (KV && !of_p ? DT : 0);
      for (int it = 0; it < walk.total; ++it) {
        const int r = it % NST, s = it & 1;
        if (!mbar_wait_warp(of_p ? &sm.p_full[s] : &sm.ds_full[s], (it >> 1) & 1, abort, 528)) break;
        tc_fence_after();
        const uint32_t t = tbase + s * 128 + (of_p ? 0 : 64), rb = smem_u32(of_p ? sm.b2[r] : sm.b1[r]);
        if (elect_lane()) {
          // a warpgroup leaves its 32 columns, packed to 16, where they were: at 0 and 32
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts(acc, t + (kk >> 1) * 32 + (kk & 1) * 8, make_smem_desc(rb + kk * 2048, 64 * 128, 1024, kSw128), idesc,
                   it > 0 || kk > 0);
          if (!of_p)  // what dS's rounding leaves, in the 16 columns behind each
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ts(acc, t + (kk >> 1) * 32 + (kk & 1) * 8 + 16, make_smem_desc(rb + kk * 2048, 64 * 128, 1024, kSw128),
                     idesc, true);
          mma_commit(of_p ? &sm.p_free[s] : &sm.ds_free[s]);
          mma_commit(&sm.empty[r]);
          if (it + 1 == walk.total) mma_commit(&sm.acc_done);
        }
        __syncwarp();
      }
    }
  } else {
    const int g = (warp - 5) >> 2;  // warpgroup: columns 32 g .. of every tile
    const int wq = warp & 3;
    const int row = wq * 32 + lane;
    const uint32_t lane_addr = tbase + (static_cast<uint32_t>(wq * 32) << 16);
    const int off = a.Nk - a.Nq;
    // KV: this thread's key, and the positions [plo, phi) that see it; Q: its query's position and
    // the keys [lo, hi) of its window
    const int at = walk.row0 + row;
    int lo, hi, upto = 0;
    bool keep = true;
    float lse2 = 0.f, delta = 0.f;
    if constexpr (KV) {
      lo = at - a.right;
      hi = at + a.left + 1;
      if (at < a.sinks) hi = walk.slot == 0 ? walk.late + off : a.Nk;
      if (walk.slot > 0) lo = max(lo, walk.late + off);
      if (MASK && at < a.Nk) keep = a.mask[static_cast<int64_t>(walk.b) * a.Nk + at] != 0;
    } else {
      const int p = at + off;
      lo = p - a.left;
      hi = min(p + a.right + 1, a.Nk);
      upto = a.sinks;
      // nqp reaches past the last tile's rows: those hold -inf and 0
      const int64_t q = (static_cast<int64_t>(walk.b) * a.Hq + walk.head) * a.nqp + at;
      lse2 = a.lse2[q];
      delta = a.delta[q];
    }
    const f2 c2 = f2_both(a.c);
    const WattnScales scales = wattn_scales<T>(a.top);
    bool ok = true;
    int next = walk.total > 0 ? walk.row(0) : 0;
    for (int it = 0; it < walk.total; ++it) {
      const int r = it % NST, s = it & 1, r0 = next + 32 * g;  // this warpgroup's first streamed row
      next = walk.row_after(next, it);
      uint32_t kept = 0xffffffffu;
      bool whole = keep;
      if (!KV && MASK) {
        const int k = r0 + lane;
        const uint8_t byte = k < a.Nk ? a.mask[static_cast<int64_t>(walk.b) * a.Nk + k] : 0;
        kept = __ballot_sync(0xffffffffu, byte != 0);
        whole = kept == 0xffffffffu;
      }
      if (KV && !mbar_wait(&sm.full[r], (it / NST) & 1, abort, 525)) { ok = false; break; }
      if (!mbar_wait(&sm.t_full[s], (it >> 1) & 1, abort, 526)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[32], y[32];
      const uint32_t t1 = lane_addr + s * 128 + 32 * g, t2 = t1 + 64;
      tmem_ld32(t1, x);
      bool inside;
      if constexpr (KV) {
        const int p0 = r0 + off;
        inside = p0 >= walk.row0 + 127 - a.right && p0 + 31 <= walk.row0 + a.left;
      } else {
        const int p0 = walk.row0 + off;
        inside = r0 + 32 <= min(p0 + a.right + 1, a.Nk) && !walk.blk.sink(it) &&
                 (r0 >= p0 + walk.blk.rows - 1 - a.left || r0 + 32 <= a.sinks);
      }
      uint32_t see = 0xffffffffu;
      const bool edge = __any_sync(0xffffffffu, !inside || !whole);
      if (edge) {
        if constexpr (KV) {
          const int b0 = r0 + off;
          see = keep ? bits_below(hi - b0) & ~bits_below(lo - b0) : 0u;
        } else {
          const bool snk = walk.blk.sink(it);
          const int f = snk ? walk.blk.nse : lo, u = snk ? walk.blk.nse : upto, e = snk ? min(hi, walk.blk.nse) : hi;
          see = bits_below(e - r0) & (~bits_below(f - r0) | bits_below(u - r0)) & kept;
        }
      }
      // x: P. The statistics wait negated, in pairs, 16 bytes a load
      const ulonglong2* s_lse = reinterpret_cast<const ulonglong2*>(sm.st[r][0] + 32 * g);
      const ulonglong2* s_del = reinterpret_cast<const ulonglong2*>(sm.st[r][1] + 32 * g);
      auto pair = [](const uint32_t* v, int i) { return f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])); };
      auto unpair = [](f2 e, uint32_t* v, int i) {
        float e0, e1;
        f2_unpack(e, e0, e1);
        v[2 * i] = __float_as_uint(e0);
        v[2 * i + 1] = __float_as_uint(e1);
      };
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        ulonglong2 n = make_ulonglong2(f2_both(lse2), f2_both(lse2));
        if constexpr (KV) n = s_lse[i / 2];
        unpair(f2_fma(pair(x, i), c2, n.x), x, i);
        unpair(f2_fma(pair(x, i + 1), c2, n.y), x, i + 1);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(ex2_approx(__uint_as_float(x[i])));
      if (edge) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(see >> i & 1)) x[i] = 0u;
      }
      if constexpr (KV) {
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = E::pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        tmem_st16(t1, pk);
        if (MASK && edge && wq == 0) {
          // T1 and T2 of this tile are done: rows of queries that see nothing may be zeroed for P^T dO and
          // dS^T q, so that no NaN there meets a P of 0 (without an edge each of them sees the warp's keys).
          // Here, where few registers are in use: before P it cost a spill
          const bool none = sm.st[r][0][32 * g + lane] == -INFINITY;
          if (__any_sync(0xffffffffu, none)) {
            if (none)
#pragma unroll 1
              for (int i = 0; i < 8 * SUB; ++i) {
                const int to = (i >> 3) * 64 * 128 + (32 * g + lane) * 128 + (i & 7) * 16;
                *reinterpret_cast<uint4*>(sm.b1[r] + to) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(sm.b2[r] + to) = make_uint4(0, 0, 0, 0);
              }
            fence_proxy_async_smem();
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[s]);
      }
      // y: dS
      tmem_ld32(t2, y);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        ulonglong2 n = make_ulonglong2(f2_both(delta), f2_both(delta));
        if constexpr (KV) n = s_del[i / 2];
        f2 d0 = f2_add(pair(y, i), n.x), d1 = f2_add(pair(y, i + 1), n.y);
        if constexpr (E::kFmt == 0) d0 = f2_mul(d0, f2_both(scales.down)), d1 = f2_mul(d1, f2_both(scales.down));
        unpair(f2_mul(d0, pair(x, i)), y, i);
        unpair(f2_mul(d1, pair(x, i + 1)), y, i + 1);
      }
      if (edge) {  // (what an unseen pair's product holds may be NaN)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(see >> i & 1)) y[i] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = E::pack2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
      tmem_st16(t2, pk);
      // dS with twice the dtype's digits: its differences P (dP - delta) cancel in the sums of dQ and dK, and
      // rounded once they put these 1.5 to 1.8 times as far from the 64-bit values as the results' own
      // rounding does (bf16: 0.0024 in the 2-norm, so 0.0017). 2 x 4096 queries, window 512: 193 us rounded
      // once, 216 so; P, which only dV and the forward read, is rounded once (dV: 0.0024).
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const f2 r = f2_fma(f2_pack(E::lo(pk[i]), E::hi(pk[i])), f2_both(-1.f), pair(y, i));
        float r0, r1;
        f2_unpack(r, r0, r1);
        pk[i] = E::pack2(r0, r1);
      }
      tmem_st16(t2 + 16, pk);
      if (!KV && MASK && !whole && wq == 0) {
        // T1 of this tile is done: its masked keys' rows may be zeroed for dS k
        if (!(kept >> lane & 1)) {
#pragma unroll
          for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint4*>(sm.b1[r] + u * 64 * 128 + (32 * g + lane) * 128)[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.ds_full[s]);
    }
    // ---------------- epilogue ----------------
    // KV: warpgroup 0 writes dV, 1 dK; Q: each half of dQ's channels
    if (walk.total > 0 && (!ok || !mbar_wait(&sm.acc_done, 0, abort, 527))) ok = false;
    if (ok) {
      tc_fence_after();
      const float f = KV && g == 0 ? scales.dv : scales.ds * a.scale;
      const bool zero = walk.total == 0;
      constexpr int COLS = KV ? DT : DT / 2;
      const int col0 = KV ? 0 : g * COLS;
      const uint32_t acc = lane_addr + Cfg::ACC + (KV ? g * DT : col0);
      float* part = nullptr;
      int parts = 0;  // rows of the tile whose sums go to the parts
      T* dst;
      int64_t pitch;
      const int at0 = walk.row0 + wq * 32;
      if constexpr (KV) {
        if (a.nx > 0 && walk.kb < a.nsb) parts = min(a.keep, a.sinks - walk.row0);
        if (row < parts)
          part = a.part + ((((static_cast<int64_t>(walk.b) * a.Hkv + walk.hk) * a.nsb + walk.kb) *
                                (1 + a.group * a.nx) + walk.slot) * 2 + g) * a.keep * DT + row * DT;
        pitch = static_cast<int64_t>(a.Hkv) * a.D;
        dst = static_cast<T*>(g == 0 ? a.dv : a.dk) + (static_cast<int64_t>(walk.b) * a.Nk + at0) * pitch + walk.hk * a.D;
      } else {
        pitch = static_cast<int64_t>(a.Hq) * a.D;
        dst = static_cast<T*>(a.dq) + (static_cast<int64_t>(walk.b) * a.Nq + at0) * pitch + walk.head * a.D;
      }
      // rows of this warp that leave for the result itself: [from, to)
      const int from = max(0, parts - wq * 32), to = KV && walk.slot > 0 ? 0 : (KV ? a.Nk : a.Nq) - at0;
      uint8_t* buf = sm.a1 + (warp - 5) * 2048;  // (all products that read the tile are done)
#pragma unroll
      for (int c0 = 0; c0 < COLS; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(acc + c0, o);
        if (zero)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        if (KV && part != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(part + c0 + 4 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = E::pack2(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f);
        store_rows(buf, lane, pk, [&](int r, int ch) -> void* {
          const int col = col0 + c0 + ch;
          return r >= from && r < to && col < a.D ? dst + r * pitch + col : nullptr;
        });
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tbase, 512);
}

// Both kinds of block in one launch, KV's first: Q's fill the SMs that the last KV blocks leave. Maps:
// boxes of 64 rows. MASK: there is a key mask (its code in the way of a call without one costs 0.3 us of
// 16.5, 1024 queries of 4 heads forward and backward).
template <typename T, int DT, bool MASK>
__global__ void __launch_bounds__(WattnBwdCfg<DT>::THREADS, 1)
    wattn_backward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_d,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ WattnBwdArgs a) {
  if (static_cast<int>(blockIdx.x) < a.kv_blocks)
    wattn_backward_block<T, DT, true, MASK>(map_k, map_v, map_q, map_d, a);
  else
    wattn_backward_block<T, DT, false, MASK>(map_q, map_d, map_k, map_v, a);
}

// -delta, delta = sum_d dO O, and -lse2 = -lse log2(e) (f16: + 14) per query, in rows of nqp: queries past
// Nq, and those that see nothing, get -inf and 0. f16: the largest |dO|^2 of those that see something, and
// (blocks behind the queries') the largest |v|^2 of the keys that the mask keeps, of `keys` from `key0` on
// and of the sinks before them. Eight threads a row, 16-byte loads. Blocks: 32 rows in x, heads in y,
// sequences in z, of which a grid has 65535 at most: these go on by the grid. (All three in x, taken apart by
// divisions, cost 0.9 us a call, of 21 for 1024 queries of 4 heads forward and backward.)
template <typename T, int DT>
__global__ void __launch_bounds__(256) wattn_stats_kernel(WattnArgs a, const T* __restrict__ dout, int64_t s0,
                                                          int64_t s1, int64_t s2, const T* __restrict__ out,
                                                          const float* __restrict__ lse, int nqp, int key0, int keys,
                                                          float* __restrict__ lse2, float* __restrict__ delta,
                                                          unsigned* __restrict__ top) {
  using E = Elem<T>;
  constexpr bool TOP = E::kFmt == 0;
  pdl_trigger();
  const int part = threadIdx.x & 7, in = threadIdx.x >> 3;
  auto load = [&](const T* p, bool there, uint4* u) {
#pragma unroll
    for (int k = 0; k < DT / 64; ++k) {
      const int c = part * 8 + 64 * k;
      u[k] = make_uint4(0, 0, 0, 0);
      if (there && c < a.D) u[k] = *reinterpret_cast<const uint4*>(p + c);
    }
  };
  auto dot = [&](const uint4* u, const uint4* w) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < DT / 64; ++k) {
      const uint32_t *p = &u[k].x, *q = &w[k].x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x = fmaf(E::lo(p[e]), E::lo(q[e]), fmaf(E::hi(p[e]), E::hi(q[e]), x));
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  };
  const int q_blocks = nqp / 32, block = blockIdx.x;
  const bool of_v = TOP && block >= q_blocks;
  const int i = (of_v ? block - q_blocks : block) * 32 + in, heads = of_v ? a.Hkv : a.Hq;
  const int sinks = min(a.sinks, key0), j = i < sinks ? i : key0 + i - sinks;
  unsigned bits = 0;
  for (int b = blockIdx.z; b < a.B; b += gridDim.z)
    for (int h = blockIdx.y; h < heads; h += gridDim.y) {
      uint4 u[DT / 64], w[DT / 64];
      float size = 0.f;  // |dO|^2 or |v|^2 of the row
      if (!of_v) {
        const int64_t bh = static_cast<int64_t>(b) * a.Hq + h;
        const bool there = i < a.Nq;
        load(dout + b * s0 + i * s1 + h * s2, there, u);
        load(out + ((static_cast<int64_t>(b) * a.Nq + i) * a.Hq + h) * a.D, there, w);
        const float v = there && part == 0 ? lse[bh * a.Nq + i] : -INFINITY, x = dot(u, w);
        if (TOP) size = dot(u, u);
        if (v == -INFINITY) size = 0.f;  // (the row's other threads count nothing)
        if (part == 0) {
          lse2[bh * nqp + i] = v == -INFINITY ? -INFINITY : wattn_lift<T>() - v * kLog2e;
          delta[bh * nqp + i] = v == -INFINITY ? 0.f : -x;
        }
      } else {
        const bool there = i < keys && (a.mask == nullptr || a.mask[static_cast<int64_t>(b) * a.Nk + j] != 0);
        load(static_cast<const T*>(a.v) + b * a.vs[0] + j * a.vs[1] + h * a.vs[2], there, u);
        size = dot(u, u);
      }
      // what is not finite makes the results so wherever it goes, and says nothing of the others' size
      if (TOP && size < INFINITY) bits = max(bits, __float_as_uint(size));
    }
  if constexpr (TOP) {
    bits = __reduce_max_sync(0xffffffffu, bits);
    __shared__ unsigned most[8];
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = bits;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int k = 1; k < 8; ++k) bits = max(bits, most[k]);
      unsigned* t = top + of_v;
      if (bits > *reinterpret_cast<volatile unsigned*>(t)) atomicMax(t, bits);  // (a maximum has no order)
    }
  }
}

// Adds the parts of the sinks' rows, in an order of its own. One block: a (b, key head), tile, output and
// two rows, whose parts SHARES groups of its threads add up.
template <int DT>
struct WattnParts {
  static constexpr int PER = DT / 8, ROWS = 2, SHARES = 256 / PER / ROWS;  // threads a row, 8 channels each
};
template <typename T, int DT>
__global__ void __launch_bounds__(256) wattn_parts_kernel(const WattnBwdArgs a) {
  using E = Elem<T>;
  using W = WattnParts<DT>;
  __shared__ float sum[W::SHARES][W::ROWS * W::PER][9];
  const int at = threadIdx.x % (W::PER * W::ROWS), share = threadIdx.x / (W::PER * W::ROWS);
  const unsigned pairs = (a.keep + W::ROWS - 1) / W::ROWS, unit = blockIdx.x / pairs;
  const int row = blockIdx.x % pairs * W::ROWS + at / W::PER, col = at % W::PER * 8;
  const unsigned nsb = a.nsb, which = unit & 1;
  const int kb = static_cast<int>((unit >> 1) % nsb);
  const int64_t bh = (unit >> 1) / nsb;
  const int key = kb * 128 + row;
  const bool live = row < a.keep && key < a.sinks && col < a.D;
  const int n = live ? 1 + a.group * a.nx : 0;
  const float* p = a.part + ((bh * a.nsb + kb) * (1 + a.group * a.nx) * 2 + which) * a.keep * DT + row * DT + col;
  float v[8] = {};
  pdl_wait();
#pragma unroll 4
  for (int i = share; i < n; i += W::SHARES) {
    const float* q = p + static_cast<int64_t>(i) * 2 * a.keep * DT;
    const float4 u = *reinterpret_cast<const float4*>(q), w = *reinterpret_cast<const float4*>(q + 4);
    v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
    v[4] += w.x, v[5] += w.y, v[6] += w.z, v[7] += w.w;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) sum[share][at][k] = v[k];
  __syncthreads();
  if (share != 0 || !live) return;
#pragma unroll
  for (int s = 1; s < W::SHARES; ++s)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += sum[s][at][k];
  const WattnScales scales = wattn_scales<T>(a.top);
  const float f = which == 0 ? scales.dv : scales.ds * a.scale;
  const int64_t b = bh / a.Hkv, hk = bh % a.Hkv;
  T* dst = static_cast<T*>(which == 0 ? a.dv : a.dk) + ((b * a.Nk + key) * a.Hkv + hk) * a.D + col;
  *reinterpret_cast<uint4*>(dst) = make_uint4(E::pack2(v[0] * f, v[1] * f), E::pack2(v[2] * f, v[3] * f),
                                              E::pack2(v[4] * f, v[5] * f), E::pack2(v[6] * f, v[7] * f));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct WattnBwdPlan {
  int nqp, nsb, nx, per, keep;
  int64_t stats, part;  // elements of each of lse2 and delta (and 4 for the largest sizes); of the sinks' parts
};

inline WattnBwdPlan wattn_bwd_plan(const WattnArgs& a, int64_t Nq) {
  WattnBwdPlan p;
  // a streamed tile starts at a multiple of 8 below Nq and reads 64, a resident one 128
  p.nqp = static_cast<int>((Nq + 127) / 128 * 128 + 64);
  p.stats = static_cast<int64_t>(a.B) * a.Hq * p.nqp;
  const int group = a.Hq / a.Hkv;
  p.nsb = (a.sinks + 127) / 128;
  p.keep = a.sinks < 128 ? a.sinks : 128;
  // queries past the first tile's window, in tiles of 64; a block takes a quarter of a tile's own walk
  const int64_t last = a.Nk - 1 < 127 ? a.Nk - 1 : 127;
  int64_t late = last + a.left + 1 - (a.Nk - Nq);
  late = late < 0 ? 0 : late > Nq ? Nq : late;
  const int64_t blocks = p.nsb > 0 && late < Nq ? (Nq - late / 8 * 8 + 63) / 64 : 0;
  const int64_t own = group * ((static_cast<int64_t>(a.left) + a.right + 128 + 63) / 64);
  int64_t per = own / 4 < 4 ? 4 : own / 4;
  // ..but no more blocks than 8 for each SM, where that many sinks alone do not make them: each leaves a
  // fp32 part of up to 128 KB (8192 sinks, a window of 2, 4 query heads to a key head, 131072 queries: 17 GB
  // a key head without this, 142 MB so)
  const int64_t units = static_cast<int64_t>(a.B) * a.Hkv * p.nsb * group, room = units > 0 ? 8 * sm_count() / units : 0;
  if (room < 1)
    per = blocks > per ? blocks : per;
  else if (per * room < blocks)
    per = (blocks + room - 1) / room;
  p.per = static_cast<int>(per);
  p.nx = static_cast<int>((blocks + per - 1) / per);
  if (p.nx == 0) p.nsb = 0;
  const int64_t DT = a.D <= 64 ? 64 : 128;
  p.part = static_cast<int64_t>(a.B) * a.Hkv * p.nsb * (1 + static_cast<int64_t>(group) * p.nx) * 2 * p.keep * DT;
  return p;
}

template <typename T, int DT, bool MASK>
static int launch_wattn_backward(int dtype, const WattnArgs& a, const void* dout, const int64_t* ds, const void* out,
                          const float* lse, float* ws, void* dq, void* dk, void* dv, cudaStream_t st) {
  bind_context();
  const WattnBwdPlan p = wattn_bwd_plan(a, a.Nq);
  float *lse2 = ws, *delta = ws + p.stats;
  CUtensorMap mq, mk, mv, md;
  if (!wattn_map(&mq, dtype, a.q, a.qs, a.B, a.Nq, a.Hq, a.D, 64) ||
      !wattn_map(&md, dtype, dout, ds, a.B, a.Nq, a.Hq, a.D, 64) ||
      !wattn_map(&mk, dtype, a.k, a.ks, a.B, a.Nk, a.Hkv, a.D, 64) ||
      !wattn_map(&mv, dtype, a.v, a.vs, a.B, a.Nk, a.Hkv, a.D, 64))
    return TOPS_ERR_TMAP;
  WattnBwdArgs f;
  f.Nq = a.Nq, f.Nk = a.Nk, f.Hq = a.Hq, f.Hkv = a.Hkv, f.group = a.Hq / a.Hkv, f.D = a.D;
  f.left = a.left, f.right = a.right, f.sinks = a.sinks;
  f.nsb = p.nsb, f.nx = p.nx, f.per = p.per, f.keep = p.keep, f.nqp = p.nqp, f.mask = a.mask;
  f.c = a.scale * kLog2e, f.scale = a.scale, f.lse2 = lse2, f.delta = delta;
  f.part = ws + 2 * p.stats + 4;
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
  f.tiles = (a.Nk + 127) / 128, f.q_tiles = (a.Nq + 127) / 128;
  const int64_t own = heads * f.tiles, kv = own + heads * p.nsb * f.group * p.nx;
  const int64_t grid = kv + static_cast<int64_t>(f.q_tiles) * a.Hq * a.B;
  // f16: the keys from the first query's window on and the sinks before them, for their largest value
  unsigned* top = reinterpret_cast<unsigned*>(ws + 2 * p.stats);
  const bool f16 = dtype == TOPS_F16;
  const int key0 = std::max(0, a.Nk - a.Nq - a.left), keys = a.Nk - key0 + std::min(a.sinks, key0);
  const dim3 stats(p.nqp / 32 + (f16 ? (keys + 31) / 32 : 0), std::min(a.Hq, 65535), std::min(a.B, 65535));
  constexpr int ROWS = WattnParts<DT>::ROWS;
  const int64_t parts = heads * 2 * p.nsb * ((p.keep + ROWS - 1) / ROWS);
  if (std::max(grid, parts) >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  f.own = static_cast<int>(own), f.kv_blocks = static_cast<int>(kv), f.dq = dq, f.dk = dk, f.dv = dv;
  if (f16 && cudaMemsetAsync(top, 0, 8, st) != cudaSuccess) return TOPS_ERR_CUDA;
  f.top = top;
  wattn_stats_kernel<T, DT><<<stats, 256, 0, st>>>(
      a, static_cast<const T*>(dout), ds[0], ds[1], ds[2], static_cast<const T*>(out), lse, p.nqp, key0, keys, lse2,
      delta, top);
  const size_t smem = sizeof(WattnBwdSmem<DT>) + 1024;
  auto kern = wattn_backward_kernel<T, DT, MASK>;
  static std::atomic<uint64_t> done{0};
  set_smem_once(kern, smem, done);
  launch_pdl(kern, static_cast<unsigned>(grid), WattnBwdCfg<DT>::THREADS, smem, st, mq, md, mk, mv, f);
  if (f.nsb > 0) launch_pdl(wattn_parts_kernel<T, DT>, static_cast<unsigned>(parts), 256, 0, st, f);
  return launch_status();
}

template <typename T>
int run_wattn_backward(int dtype, const WattnArgs& a, const void* dout, const int64_t* ds, const void* out,
                       const float* lse, float* ws, void* dq, void* dk, void* dv, cudaStream_t st) {
  const auto run = [&](auto dt, auto mask) {
    return launch_wattn_backward<T, decltype(dt)::value, decltype(mask)::value>(dtype, a, dout, ds, out, lse, ws, dq, dk, dv,
                                                                                st);
  };
  using std::integral_constant;
  if (a.D <= 64)
    return a.mask ? run(integral_constant<int, 64>(), std::true_type()) : run(integral_constant<int, 64>(), std::false_type());
  return a.mask ? run(integral_constant<int, 128>(), std::true_type()) : run(integral_constant<int, 128>(), std::false_type());
}

}  // namespace tops
