// wattn.cu — windowed attention with sinks, forward, on tcgen05 (16-bit IO, D a multiple of 8 up
// to 128, 16-byte aligned rows, scale > 0).
//
//   S = q k^T,  P = 2^(c (S - m)) with c = scale log2(e),  O = P v / sum P,  lse = ln2 (c m + log2 sum P)
// over the keys that a query sees (wattn.h), in one walk over them with a running maximum m and sum.
//
// A block (CTA) takes 128 queries of one head and walks over 64-key blocks: the sinks, where the
// window has left them behind, then the window, which starts exactly at the first key that the
// tile's first query sees (a TMA row coordinate needs no alignment), so a window of W costs
// ceil((W + 127) / 64) blocks. Only blocks on the edge of the window, or with a masked key, test
// their keys; the others run without. Up to 32 left-behind sinks are a block of 32 keys.
//
// One warp loads (TMA; keys past the end and channels past D arrive as zeros), one issues the MMAs
// of S and another those of P v, all of its lanes together (a lane on its own takes some 85 cycles
// to issue one: 61 us for 57.7 at 2 x 4096 queries, 16 heads of 128, window 512), four hold the
// softmax: a thread owns a query row (a TMEM lane), so row maximum and sum need no exchange. S is a
// fp32 TMEM tile, P takes its place rounded to the IO dtype (the product's operand type; its sum is
// taken before the rounding), O accumulates in TMEM and is rescaled only when the maximum has grown
// by 2^8 (f16: 2^7). S has two buffers: q k^T of the next block runs under the softmax of this one. Two CTAs
// share an SM and its 512 TMEM columns (S 2 x 64, O up to 128 each). CTAs are persistent: the loads
// and S of the next tile run under the end of the present one (8192 queries, 16 heads, window 1024:
// 87.5 us with a CTA a tile, 83.6 so).
//
// Bound by the exponentials and the products together: 8192 queries, 16 heads of 128 on 4, window 1024:
// 77.5 us from a CUDA graph with its inputs in the cache, 836 TFLOP/s of the products that a query's own
// keys take; 92 us a call from Python with inputs that come from memory.
//
// Masked keys: their score is replaced by -inf, and their rows of the V tile are zeroed in shared
// memory before P v, so that a NaN there does not pass through 0 * NaN.
#include <atomic>
#include "sm100.cuh"
#include "wattn.h"

namespace tops {

struct WattnFwdArgs {
  int Nq, Nk, Hq, group, D;  // group: query heads to a key head
  int left, right, sinks, tiles, units;  // units: (tile of queries, head, sequence)
  int step[3];                           // the grid in those
  const uint8_t* mask;
  float c;  // scale * log2(e)
  void* out;
  float* lse;
};

template <int DT>
struct WattnFwdCfg {
  static constexpr int SUB = DT / 64;            // 64-channel sub-tiles (128-byte rows, 128B swizzle)
  static constexpr int BK = 64;                  // keys a block
  static constexpr int Q_TILE = SUB * 128 * 128;
  static constexpr int TILE = SUB * BK * 128;    // bytes of a K or V tile
  static constexpr int NS = 2;                   // K and V stages
  static constexpr int O_COL = 128;              // TMEM: S (and P) of block j at 64 (j & 1), O
  static constexpr int THREADS = 224;
};

template <int DT>
struct WattnFwdSmem {
  using Cfg = WattnFwdCfg<DT>;
  alignas(1024) uint8_t q[Cfg::Q_TILE];
  alignas(1024) uint8_t k[Cfg::NS][Cfg::TILE];
  alignas(1024) uint8_t v[Cfg::NS][Cfg::TILE];
  alignas(16) uint8_t o[4][2048];  // a warp's part of the result on its way out
  uint64_t q_full, q_empty, o_empty, k_full[2], k_empty[2], v_full[2];
  uint64_t s_full[2], p_full[2], pv_done[2];  // of block j at j & 1
  uint32_t tmem_base;
  int abort;
};

// bits j of 0..31 with base + j < n
__device__ __forceinline__ uint32_t bits_below(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// A warp's 32 rows of 32 channels, lane's row in pk, to where at(row, channel) says (null: nowhere) in
// 64-byte pieces, through 2 KB of shared memory: a lane that stores its own row writes half a sector of
// 32 lines at once (2 x 4096 queries, 16 heads of 128, window 512: forward 57.7 us with that, 55.4 so,
// backward 204 and 198).
template <typename F>
__device__ __forceinline__ void store_rows(uint8_t* buf, int lane, const uint32_t* pk, F&& at) {
  __syncwarp();
#pragma unroll
  for (int v = 0; v < 4; ++v)
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((v ^ (lane >> 1 & 3)) << 4)) =
        make_uint4(pk[4 * v], pk[4 * v + 1], pk[4 * v + 2], pk[4 * v + 3]);
  __syncwarp();
  const int v = lane & 3;
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    w[i] = *reinterpret_cast<const uint4*>(buf + row * 64 + ((v ^ (row >> 1 & 3)) << 4));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (void* p = at(8 * i + (lane >> 2), 8 * v)) *static_cast<uint4*>(p) = w[i];
}

// The blocks of 2^LOG keys that a tile of 128 query rows walks over: nsb of sinks, then the window's.
template <int LOG>
struct WattnBlocks {
  static constexpr int W = 1 << LOG;
  int p0, rows;      // position of the first query, queries in the tile
  int start, end;    // keys of the window part
  int nse, nsb, n;   // sinks before it, their blocks, all blocks
  __device__ WattnBlocks(int q0, int Nq, int Nk, int left, int right, int sinks) {
    rows = min(128, Nq - q0);
    p0 = q0 + Nk - Nq;
    start = max(0, p0 - left);
    end = min(p0 + rows + right, Nk);
    nse = min(sinks, start);
    if (start <= sinks) start = nse = 0;
    nsb = (nse + W - 1) >> LOG;
    n = nsb + ((end - start + W - 1) >> LOG);
  }
  __device__ bool sink(int j) const { return j < nsb; }
  __device__ bool narrow(int j) const { return j < nsb && nse <= 32; }
  __device__ int key(int j) const { return j < nsb ? j << LOG : start + ((j - nsb) << LOG); }
};

template <typename T, int DT, bool MASK>
__global__ void __launch_bounds__(WattnFwdCfg<DT>::THREADS, 2)
    wattn_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k32,
                         const __grid_constant__ CUtensorMap map_v32, const WattnFwdArgs a) {
  using Cfg = WattnFwdCfg<DT>;
  using E = Elem<T>;
  constexpr int SUB = Cfg::SUB;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<WattnFwdSmem<DT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;

  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    mbar_init(&sm.o_empty, 4);
    for (int s = 0; s < Cfg::NS; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.pv_done[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.p_full[s], 4);
    }
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 256);
    tmem_relinquish();  // the SM's other CTA allocates too
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem_base;

  // Persistent: a CTA takes units blockIdx.x, + gridDim.x, .. Blocks of keys are counted on across
  // units (g: block j of unit lu is block g + j), so loads and S of the next unit run under the end
  // of the present one.
  int g = 0, lu = 0;
  int tile = blockIdx.x % a.tiles, h = blockIdx.x / a.tiles % a.Hq, b = blockIdx.x / a.tiles / a.Hq;
  auto next = [&] {
    tile += a.step[0], h += a.step[1], b += a.step[2], ++lu;
    if (tile >= a.tiles) tile -= a.tiles, ++h;
    if (h >= a.Hq) h -= a.Hq, ++b;
  };
  auto blocks = [&](int tile) { return WattnBlocks<6>(tile * 128, a.Nq, a.Nk, a.left, a.right, a.sinks); };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x, next()) {
        const WattnBlocks<6> blk = blocks(tile);
        const int hk = h / a.group;
        auto load = [&](const CUtensorMap* m, uint8_t* dst, uint64_t* bar, int head, int row, int rows, int sub) {
          mbar_expect_tx(bar, SUB * rows * 128);
#pragma unroll
          for (int s = 0; s < SUB; ++s) tma_load_4d(dst + s * sub, m, bar, s * 64, head, row, b);
        };
        if (!mbar_wait(&sm.q_empty, (lu & 1) ^ 1, abort, 516)) break;  // the unit before has no more S
        load(&map_q, sm.q, &sm.q_full, h, tile * 128, 128, 128 * 128);
        for (int j = 0; j < blk.n; ++j, ++g) {
          const int s = g & 1;
          const uint32_t ph = ((g >> 1) & 1) ^ 1;
          const bool nar = blk.narrow(j);
          const int rows = nar ? 32 : Cfg::BK;
          ok = mbar_wait(&sm.k_empty[s], ph, abort, 501);
          if (!ok) break;
          load(nar ? &map_k32 : &map_k, sm.k[s], &sm.k_full[s], hk, blk.key(j), rows, Cfg::BK * 128);
          ok = mbar_wait(&sm.pv_done[s], ph, abort, 502);  // P v of the block before in this stage
          if (!ok) break;
          load(nar ? &map_v32 : &map_v, sm.v[s], &sm.v_full[s], hk, blk.key(j), rows, Cfg::BK * 128);
        }
      }
    }
  } else if (warp == 1) {
    // S of block g; its buffer held P of block g - 2
    const int ksteps = (a.D + 15) >> 4;
    const uint32_t qa = smem_u32(sm.q);
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x, next()) {
      const WattnBlocks<6> blk = blocks(tile);
      if (!mbar_wait_warp(&sm.q_full, lu & 1, abort, 504)) break;
      for (int j = 0; j < blk.n; ++j, ++g) {
        const int s = g & 1;
        ok = mbar_wait_warp(&sm.k_full[s], (g >> 1) & 1, abort, 503) &&
             mbar_wait_warp(&sm.pv_done[s], ((g >> 1) & 1) ^ 1, abort, 505);
        if (!ok) break;
        tc_fence_after();
        const uint32_t idesc = make_idesc_f16(128, blk.narrow(j) ? 32 : Cfg::BK, E::kFmt, false, false);
        const uint32_t ka = smem_u32(sm.k[s]);
        if (elect_lane()) {
#pragma unroll
          for (int kk = 0; kk < DT / 16; ++kk)
            if (kk < ksteps)
              mma_ss(tbase + s * 64, make_smem_desc(qa + (kk / 4) * 128 * 128 + (kk % 4) * 32, 16, 1024, kSw128),
                     make_smem_desc(ka + (kk / 4) * Cfg::BK * 128 + (kk % 4) * 32, 16, 1024, kSw128), idesc, kk > 0);
          mma_commit(&sm.s_full[s]);
        }
        __syncwarp();
      }
      if (elect_lane()) mma_commit(&sm.q_empty);
      __syncwarp();
    }
  } else if (warp == 6) {
    const uint32_t idesc_pv = make_idesc_f16(128, DT, E::kFmt, false, true);
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x, next()) {
      const WattnBlocks<6> blk = blocks(tile);
      for (int j = 0; j < blk.n; ++j, ++g) {
        const int s = g & 1;
        ok = mbar_wait_warp(&sm.v_full[s], (g >> 1) & 1, abort, 506) &&
             mbar_wait_warp(&sm.p_full[s], (g >> 1) & 1, abort, 507) &&
             // the first product overwrites O: the unit before must have read it
             (j > 0 || lu == 0 || mbar_wait_warp(&sm.o_empty, (lu - 1) & 1, abort, 517));
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_u32(sm.v[s]);
        const int steps = blk.narrow(j) ? 2 : 4;
        if (elect_lane()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < steps)
              mma_ts(tbase + Cfg::O_COL, tbase + s * 64 + kk * 8,
                     make_smem_desc(va + kk * 2048, Cfg::BK * 128, 1024, kSw128), idesc_pv, j > 0 || kk > 0);
          mma_commit(&sm.pv_done[s]);
        }
        __syncwarp();
      }
    }
  } else {
    const int wq = warp & 3;
    const int row = wq * 32 + lane;  // TMEM lane = query row of the tile
    const uint32_t lane_addr = tbase + (static_cast<uint32_t>(wq * 32) << 16);
    // f16 ends at 2^-24: P is held at 2^8 times its size, the sum with it, and the maximum may lag by 2^7
    // there: a key keeps all its digits down to 2^-22 of the largest and counts down to 2^-33 (without
    // it the many small probabilities of a window, beside a sink that takes most, are zeros). Lags of 7,
    // 6 and 4 that leave more room take 54.2, 55.5 and 68 us for 2 x 4096 queries, 16 heads of 128,
    // window 512 (8 without the factor: 54.2). bf16 has the range.
    constexpr bool F16 = E::kFmt == 0;
    constexpr float kLift = F16 ? 8.f : 0.f;
    const float c = a.c, grow = (F16 ? 7.f : 8.f) / c;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x, next()) {
    const WattnBlocks<6> blk = blocks(tile);
    const int p = blk.p0 + row;
    const int lo = p - a.left, hi = min(p + a.right + 1, a.Nk);  // window keys [lo, hi)
    float m = -INFINITY, l = 0.f;

    // One block of NCOL keys; EDGE: some of them may not be seen.
    auto work = [&](auto ncol_c, auto edge_c, int j, int key, const uint32_t* kept) {
      constexpr int NCOL = decltype(ncol_c)::value;
      constexpr bool EDGE = decltype(edge_c)::value;
      const uint32_t s_addr = lane_addr + ((g + j) & 1) * 64;
      uint32_t x[NCOL];
      if constexpr (NCOL == 64)
        tmem_ld64(s_addr, x);
      else
        tmem_ld32(s_addr, x);
      if constexpr (EDGE) {
        const bool snk = blk.sink(j);
        const int first = snk ? blk.nse : lo, upto = snk ? blk.nse : a.sinks, end = snk ? min(hi, blk.nse) : hi;
#pragma unroll
        for (int w = 0; w < NCOL / 32; ++w) {
          const int k0 = key + w * 32;
          uint32_t see = bits_below(end - k0) & (~bits_below(first - k0) | bits_below(upto - k0));
          if (MASK) see &= kept[w];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see >> i & 1)) x[w * 32 + i] = 0xff800000u;  // -inf
        }
      }
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = __uint_as_float(x[i]);
#pragma unroll
      for (int i = 4; i < NCOL; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[e] = fmaxf(fmaxf(t[e], __uint_as_float(x[i + e])), i + 4 + e < NCOL ? __uint_as_float(x[i + 4 + e]) : t[e]);
      const float mx = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      const bool need = m == -INFINITY ? mx > -INFINITY : mx > m + grow;
      if (__any_sync(0xffffffffu, need)) {
        const float mn = need ? mx : m;
        if (j > 0) {
          // O is stable once P v of the block before is done
          if (!mbar_wait(&sm.pv_done[(g + j - 1) & 1], ((g + j - 1) >> 1) & 1, abort, 508)) return false;
          tc_fence_after();
          const float f = need ? ex2_approx((m - mn) * c) : 1.0f;
          l *= f;
#pragma unroll
          for (int c0 = 0; c0 < DT; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(lane_addr + Cfg::O_COL + c0, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(lane_addr + Cfg::O_COL + c0, o);
          }
        }
        m = mn;
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      const f2 c2 = f2_both(c), d2 = f2_both(kLift - mc);
      f2 sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c0 = 0; c0 < NCOL; c0 += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f2 e = f2_fma(f2_pack(__uint_as_float(x[c0 + 2 * i]), __uint_as_float(x[c0 + 2 * i + 1])), c2, d2);
          float e0, e1;
          f2_unpack(e, e0, e1);
          e0 = ex2_approx(e0);
          e1 = ex2_approx(e1);
          sum[i & 1] = f2_add(sum[i & 1], f2_pack(e0, e1));
          pk[i] = E::pack2(e0, e1);
        }
        tmem_st16(s_addr + c0 / 2, pk);
      }
      float s0, s1;
      f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_wait_st();
      return true;
    };

    // the key mask, 64 bytes a block, the next block's on their way
    uint8_t byte[2];
    auto load_mask = [&](int j) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int k = blk.key(j) + w * 32 + lane;
        byte[w] = k < a.Nk ? a.mask[static_cast<int64_t>(b) * a.Nk + k] : 0;
      }
    };
    if (MASK) load_mask(0);
    for (int j = 0; j < blk.n; ++j) {
      const int key = blk.key(j), s = (g + j) & 1;
      const uint32_t ph = ((g + j) >> 1) & 1;
      const bool nar = blk.narrow(j);
      uint32_t kept[2];
      bool whole = true;
      if constexpr (MASK) {
        kept[0] = __ballot_sync(0xffffffffu, byte[0] != 0);
        kept[1] = __ballot_sync(0xffffffffu, byte[1] != 0);
        whole = (kept[0] & kept[1]) == 0xffffffffu;
        if (j + 1 < blk.n) load_mask(j + 1);
      }
      if (!mbar_wait(&sm.s_full[s], ph, abort, 510)) { ok = false; break; }
      if (warp == 2 && lane == 0) mbar_arrive(&sm.k_empty[s]);  // q k^T of the block is done
      tc_fence_after();
      // every row sees the whole block: up to the first row's end, from the last row's start
      const bool inside = key + Cfg::BK <= min(blk.p0 + a.right + 1, a.Nk) && !blk.sink(j) &&
                          (key >= blk.p0 + blk.rows - 1 - a.left || key + Cfg::BK <= a.sinks);
      using std::integral_constant;
      const bool done =
          nar ? work(integral_constant<int, 32>(), integral_constant<bool, true>(), j, key, kept)
          : inside && whole ? work(integral_constant<int, 64>(), integral_constant<bool, false>(), j, key, kept)
                            : work(integral_constant<int, 64>(), integral_constant<bool, true>(), j, key, kept);
      if (!done) { ok = false; break; }
      if constexpr (MASK) {
        if (!whole) {
          // masked keys' rows of V: zero (the swizzle moves 16-byte chunks within a row only)
          if (!mbar_wait(&sm.v_full[s], ph, abort, 511)) { ok = false; break; }
          const uint32_t word = wq & 1 ? kept[1] : kept[0];
          if (row < (nar ? 32 : 64) && !(word >> lane & 1)) {
#pragma unroll
            for (int e = 0; e < SUB; ++e)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(sm.v[s] + e * Cfg::BK * 128 + row * 128)[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[s]);
    }
    // ---------------- O / l -> out, lse ----------------
    const int e = g + blk.n - 1;  // the unit's last block
    g += blk.n;
    if (!ok || !mbar_wait(&sm.pv_done[e & 1], (e >> 1) & 1, abort, 512)) {
      ok = false;
      break;
    }
    tc_fence_after();
    const int i = tile * 128 + row;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const int i0 = tile * 128 + wq * 32;
    T* dst = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.Nq + i0) * a.Hq + h) * a.D;
    const int64_t pitch = static_cast<int64_t>(a.Hq) * a.D;
#pragma unroll
    for (int c0 = 0; c0 < DT; c0 += 32) {
      uint32_t o[32], pk[16];
      tmem_ld32(lane_addr + Cfg::O_COL + c0, o);
      if (c0 + 32 == DT) {  // O has been read: the next unit's products may overwrite it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        pk[e] = l == 0.f ? 0u : E::pack2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
      store_rows(sm.o[wq], lane, pk, [&](int r, int ch) -> void* {
        const int col = c0 + ch;
        return i0 + r < a.Nq && col < a.D ? dst + r * pitch + col : nullptr;
      });
    }
    if (a.lse && i < a.Nq)
      a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i] =
          l == 0.f ? -INFINITY : (fmaf(m, c, log2f(l) - kLift)) * 0.69314718055994531f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tbase, 256);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// A thread that has not used its device yet (autograd has threads of its own) has no current context,
// without which a tensor map cannot be encoded. cudaSetDevice makes it current, and is open while a stream
// is captured, as memory calls are not.
static void bind_context() {
  static thread_local uint64_t bound = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (bound & bit) return;
  cudaSetDevice(dev);
  bound |= bit;
}

// (B, N, H, D) with channel rows of D elements: boxes of 64 channels x `rows` tokens of one head,
// 128B swizzle. A place of size 1 gets a stride of one row whatever the tensor says.
inline bool wattn_map(CUtensorMap* m, int dtype, const void* p, const int64_t* st, int64_t B, int64_t N, int64_t H,
                      int64_t D, uint32_t rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H), static_cast<uint64_t>(N),
                            static_cast<uint64_t>(B)};
  auto bytes = [&](int64_t n, int64_t s) { return static_cast<uint64_t>(n > 1 ? s : (D + 7) / 8 * 8) * 2; };
  const uint64_t str[3] = {bytes(H, st[2]), bytes(N, st[1]), bytes(B, st[0])};
  const uint32_t box[4] = {64, 1, rows, 1};
  return make_tmap(m, tmap_dtype(dtype), 4, p, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// What the TMA maps ask of a tensor: 16-byte rows, no stride of zero over more than one place.
inline bool wattn_fits(const void* p, const int64_t* st, int64_t B, int64_t N, int64_t H) {
  const int64_t n[3] = {B, N, H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] % 8 != 0 || st[i] <= 0 || st[i] >= (int64_t(1) << 38))) return false;
  return aligned16(p);
}

// Whether the tensor-core kernels take a call (the others run on the CUDA cores). A scale of zero
// or below would turn -inf, a masked score, into NaN or +inf.
inline bool wattn_tensor(int dtype, const WattnArgs& a) {
  return (dtype == TOPS_BF16 || dtype == TOPS_F16) && a.D % 8 == 0 && a.D <= 128 && a.scale > 0.f &&
         wattn_fits(a.q, a.qs, a.B, a.Nq, a.Hq) && wattn_fits(a.k, a.ks, a.B, a.Nk, a.Hkv) &&
         wattn_fits(a.v, a.vs, a.B, a.Nk, a.Hkv);
}

// The kernel's shared memory limit, raised once a device (the call costs as much as a launch).
template <typename K>
inline void set_smem_once(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  set_smem(kernel, bytes);
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename T, int DT, bool MASK>
static int launch_wattn_forward(int dtype, const WattnArgs& a, void* out, float* lse, cudaStream_t st) {
  bind_context();
  CUtensorMap mq, mk, mv, mk32, mv32;
  if (!wattn_map(&mq, dtype, a.q, a.qs, a.B, a.Nq, a.Hq, a.D, 128) ||
      !wattn_map(&mk, dtype, a.k, a.ks, a.B, a.Nk, a.Hkv, a.D, 64) ||
      !wattn_map(&mv, dtype, a.v, a.vs, a.B, a.Nk, a.Hkv, a.D, 64))
    return TOPS_ERR_TMAP;
  if (a.sinks == 0)  // no block of left-behind sinks
    mk32 = mk, mv32 = mv;
  else if (!wattn_map(&mk32, dtype, a.k, a.ks, a.B, a.Nk, a.Hkv, a.D, 32) ||
           !wattn_map(&mv32, dtype, a.v, a.vs, a.B, a.Nk, a.Hkv, a.D, 32))
    return TOPS_ERR_TMAP;
  WattnFwdArgs f;
  f.Nq = a.Nq, f.Nk = a.Nk, f.Hq = a.Hq, f.group = a.Hq / a.Hkv, f.D = a.D;
  f.left = a.left, f.right = a.right, f.sinks = a.sinks, f.tiles = (a.Nq + 127) / 128;
  f.mask = a.mask, f.c = a.scale * kLog2e, f.out = out, f.lse = lse;
  const int64_t units = static_cast<int64_t>(f.tiles) * a.Hq * a.B, most = 2 * static_cast<int64_t>(sm_count());
  if (units >= (int64_t(1) << 30)) return TOPS_ERR_SHAPE;
  f.units = static_cast<int>(units);
  const int64_t grid = units < most ? units : most;
  f.step[0] = static_cast<int>(grid % f.tiles), f.step[1] = static_cast<int>(grid / f.tiles % a.Hq);
  f.step[2] = static_cast<int>(grid / f.tiles / a.Hq);
  const size_t smem = sizeof(WattnFwdSmem<DT>) + 1024;
  auto kern = wattn_forward_kernel<T, DT, MASK>;
  static std::atomic<uint64_t> done{0};
  set_smem_once(kern, smem, done);
  kern<<<static_cast<unsigned>(grid), WattnFwdCfg<DT>::THREADS, smem, st>>>(mq, mk, mv, mk32, mv32, f);
  return launch_status();
}

template <typename T>
int run_wattn_forward(int dtype, const WattnArgs& a, void* out, float* lse, cudaStream_t st) {
  if (a.D <= 64)
    return a.mask ? launch_wattn_forward<T, 64, true>(dtype, a, out, lse, st)
                  : launch_wattn_forward<T, 64, false>(dtype, a, out, lse, st);
  return a.mask ? launch_wattn_forward<T, 128, true>(dtype, a, out, lse, st)
                : launch_wattn_forward<T, 128, false>(dtype, a, out, lse, st);
}

}  // namespace tops
