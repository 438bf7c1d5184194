// wattn.cu — windowed attention with sinks, forward, on tcgen05 (16-bit IO, D a multiple of 8 up
// to 128, 16-byte aligned rows, scale > 0).
//
//   S = q k^T,  P = 2^(c (S - m)) with c = scale log2(e),  O = P v / sum P,  lse = ln2 (c m + log2 sum P)
// over the keys that a query sees (wattn.h), in one walk over them with a running maximum m and sum.
//
// A block (CTA) takes 128 queries of one head and walks over 128-key blocks: the sinks, where the
// window has left them behind, then the window, which starts exactly at the first key that the
// tile's first query sees (a TMA row coordinate needs no alignment), so a window of W costs
// ceil((W + 127) / 128) blocks. Only blocks on the edge of the window, or with a masked key, test
// their keys; the others run without. Up to 32 left-behind sinks are a block of 32 keys.
//
// One warp loads (TMA; keys past the end and channels past D arrive as zeros), one issues the
// MMAs, four hold the softmax: a thread owns a query row (a TMEM lane), so row maximum and sum need
// no exchange. S is a fp32 TMEM tile, P goes back to TMEM rounded to the IO dtype (the product's
// operand type; its sum is taken before the rounding), O accumulates in TMEM and is rescaled only
// when the maximum has grown by 2^8. Two CTAs share an SM and its 512 TMEM columns, so that one's
// MMAs run under the other's softmax. D > 64: P takes S's columns and S of the next block follows
// P v of this one; D <= 64: P has its own columns and S of the next block is computed under the
// softmax of this one.
//
// Masked keys: their score is replaced by -inf, and their rows of the V tile are zeroed in shared
// memory before P v, so that a NaN there does not pass through 0 * NaN.
#include "sm100.cuh"
#include "wattn.h"

namespace tops {

struct WattnFwdArgs {
  int Nq, Nk, Hq, group, D;  // group: query heads to a key head
  int left, right, sinks, tiles;
  const uint8_t* mask;
  float c;  // scale * log2(e)
  void* out;
  float* lse;
};

template <int DT>
struct WattnFwdCfg {
  static constexpr int SUB = DT / 64;             // 64-channel sub-tiles (128-byte rows, 128B swizzle)
  static constexpr int TILE = SUB * 128 * 128;    // bytes of a 128-row tile
  static constexpr int NS = DT == 128 ? 1 : 2;    // K and V stages
  static constexpr int S_COL = 0;
  static constexpr int P_COL = DT == 128 ? 0 : 128;
  static constexpr int O_COL = DT == 128 ? 128 : 192;
  static constexpr bool AHEAD = P_COL != S_COL;   // S of the next block before P v of this one
  static constexpr int THREADS = 192;
};

template <int DT>
struct WattnFwdSmem {
  using Cfg = WattnFwdCfg<DT>;
  alignas(1024) uint8_t q[Cfg::TILE];
  alignas(1024) uint8_t k[Cfg::NS][Cfg::TILE];
  alignas(1024) uint8_t v[Cfg::NS][Cfg::TILE];
  uint64_t q_full, k_full[Cfg::NS], k_empty[Cfg::NS], v_full[Cfg::NS], v_empty[Cfg::NS];
  uint64_t s_full, s_free, p_full, pv_done;
  uint32_t tmem_base;
  int abort;
};

// bits j of 0..31 with base + j < n
__device__ __forceinline__ uint32_t bits_below(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
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
  constexpr int NS = Cfg::NS, SUB = Cfg::SUB;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<WattnFwdSmem<DT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;

  const int tile = blockIdx.x % a.tiles;
  const int h = blockIdx.x / a.tiles % a.Hq;
  const int b = blockIdx.x / a.tiles / a.Hq;
  const int q0 = tile * 128;
  const WattnBlocks<7> blk(q0, a.Nq, a.Nk, a.left, a.right, a.sinks);

  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], 1);
    }
    mbar_init(&sm.s_full, 1);
    mbar_init(&sm.s_free, 4);
    mbar_init(&sm.p_full, 4);
    mbar_init(&sm.pv_done, 1);
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

  if (warp == 0) {
    if (lane == 0) {
      const int hk = h / a.group;
      auto load = [&](const CUtensorMap* m, uint8_t* dst, uint64_t* bar, int head, int row, int rows) {
        mbar_expect_tx(bar, SUB * rows * 128);
#pragma unroll
        for (int s = 0; s < SUB; ++s) tma_load_4d(dst + s * 128 * 128, m, bar, s * 64, head, row, b);
      };
      load(&map_q, sm.q, &sm.q_full, h, q0, 128);
      for (int j = 0; j < blk.n; ++j) {
        const int s = j % NS;
        const uint32_t ph = ((j / NS) & 1) ^ 1;
        const bool nar = blk.narrow(j);
        const int rows = nar ? 32 : 128;
        if (!mbar_wait(&sm.k_empty[s], ph, abort, 501)) break;
        load(nar ? &map_k32 : &map_k, sm.k[s], &sm.k_full[s], hk, blk.key(j), rows);
        if (!mbar_wait(&sm.v_empty[s], ph, abort, 502)) break;
        load(nar ? &map_v32 : &map_v, sm.v[s], &sm.v_full[s], hk, blk.key(j), rows);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc_pv = make_idesc_f16(128, DT, E::kFmt, false, true);
      const int ksteps = (a.D + 15) >> 4;
      const uint32_t qa = smem_u32(sm.q);
      auto issue_s = [&](int j) {
        const int s = j % NS;
        if (!mbar_wait(&sm.k_full[s], (j / NS) & 1, abort, 503)) return false;
        tc_fence_after();
        const uint32_t idesc = make_idesc_f16(128, blk.narrow(j) ? 32 : 128, E::kFmt, false, false);
        const uint32_t ka = smem_u32(sm.k[s]);
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
          const uint32_t off = (kk / 4) * 128 * 128 + (kk % 4) * 32;
          if (kk < ksteps)
            mma_ss(tbase + Cfg::S_COL, make_smem_desc(qa + off, 16, 1024, kSw128),
                   make_smem_desc(ka + off, 16, 1024, kSw128), idesc, kk > 0);
        }
        mma_commit(&sm.s_full);
        mma_commit(&sm.k_empty[s]);
        return true;
      };
      bool ok = mbar_wait(&sm.q_full, 0, abort, 504) && issue_s(0);
      for (int j = 0; ok && j < blk.n; ++j) {
        if (Cfg::AHEAD && j + 1 < blk.n) {
          if (!mbar_wait(&sm.s_free, j & 1, abort, 505)) break;
          if (!issue_s(j + 1)) break;
        }
        const int s = j % NS;
        if (!mbar_wait(&sm.v_full[s], (j / NS) & 1, abort, 506)) break;
        if (!mbar_wait(&sm.p_full, j & 1, abort, 507)) break;
        tc_fence_after();
        const uint32_t va = smem_u32(sm.v[s]);
        const int steps = blk.narrow(j) ? 2 : 8;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (kk < steps)
            mma_ts(tbase + Cfg::O_COL, tbase + Cfg::P_COL + kk * 8, make_smem_desc(va + kk * 2048, 16384, 1024, kSw128),
                   idesc_pv, j > 0 || kk > 0);
        mma_commit(&sm.pv_done);
        mma_commit(&sm.v_empty[s]);
        if (!Cfg::AHEAD && j + 1 < blk.n && !issue_s(j + 1)) break;
      }
    }
  } else {
    const int wq = warp & 3;
    const int row = wq * 32 + lane;  // TMEM lane = query row of the tile
    const uint32_t lane_addr = tbase + (static_cast<uint32_t>(wq * 32) << 16);
    const int p = blk.p0 + row;
    const int lo = p - a.left, hi = min(p + a.right + 1, a.Nk);  // window keys [lo, hi)
    const float c = a.c, grow = 8.0f / c;
    float m = -INFINITY, l = 0.f;
    bool ok = true;

    // one block of NCOL keys
    auto work = [&](auto ncol_c, int j, int key, bool edge, const uint32_t* kept) {
      constexpr int NCOL = decltype(ncol_c)::value;
      uint32_t x[NCOL];
      if constexpr (NCOL == 128) {
        tmem_ld64_async(lane_addr + Cfg::S_COL, x);
        tmem_ld64_async(lane_addr + Cfg::S_COL + 64, x + 64);
        tmem_wait_ld64(x);
        tmem_wait_ld64(x + 64);
      } else {
        tmem_ld32(lane_addr + Cfg::S_COL, x);
      }
      if (Cfg::AHEAD) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_free);
      }
      if (edge) {
        const int first = blk.sink(j) ? blk.nse : lo, upto = blk.sink(j) ? blk.nse : a.sinks;
#pragma unroll
        for (int w = 0; w < NCOL / 32; ++w) {
          const int k0 = key + w * 32;
          uint32_t see = bits_below(hi - k0) & (~bits_below(first - k0) | bits_below(upto - k0));
          if (blk.sink(j)) see &= bits_below(blk.nse - k0);
          if (MASK) see &= kept[w];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see >> i & 1)) x[w * 32 + i] = 0xff800000u;  // -inf
        }
      }
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = __uint_as_float(x[i]);
#pragma unroll
      for (int i = 8; i < NCOL; ++i) t[i & 7] = fmaxf(t[i & 7], __uint_as_float(x[i]));
      const float mx = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
      const bool need = m == -INFINITY ? mx > -INFINITY : mx > m + grow;
      if (__any_sync(0xffffffffu, need)) {
        const float mn = need ? mx : m;
        if (j > 0) {
          // O is stable once P v of the block before is done
          if (!mbar_wait(&sm.pv_done, (j - 1) & 1, abort, 508)) return false;
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
      } else if (Cfg::AHEAD && j > 0) {
        // P of the block before has been read
        if (!mbar_wait(&sm.pv_done, (j - 1) & 1, abort, 509)) return false;
        tc_fence_after();
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      const unsigned long long c2 = f2_pack(c, c), d2 = f2_pack(-mc, -mc);
      unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c0 = 0; c0 < NCOL; c0 += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const unsigned long long e =
              f2_fma(f2_pack(__uint_as_float(x[c0 + 2 * i]), __uint_as_float(x[c0 + 2 * i + 1])), c2, d2);
          float e0, e1;
          f2_unpack(e, e0, e1);
          e0 = ex2_approx(e0);
          e1 = ex2_approx(e1);
          sum[i & 1] = f2_add(sum[i & 1], f2_pack(e0, e1));
          pk[i] = E::pack2(e0, e1);
        }
        tmem_st16(lane_addr + Cfg::P_COL + c0 / 2, pk);
      }
      float s0, s1;
      f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_wait_st();
      return true;
    };

    for (int j = 0; j < blk.n; ++j) {
      const int key = blk.key(j);
      const bool nar = blk.narrow(j);
      uint32_t kept[4];
      bool whole = true;
      if constexpr (MASK) {
        const uint8_t* mk = a.mask + static_cast<int64_t>(b) * a.Nk;
        uint8_t byte[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int k = key + w * 32 + lane;
          byte[w] = k < a.Nk ? mk[k] : 0;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          kept[w] = __ballot_sync(0xffffffffu, byte[w] != 0);
          whole = whole && kept[w] == 0xffffffffu;
        }
      }
      if (!mbar_wait(&sm.s_full, j & 1, abort, 510)) { ok = false; break; }
      tc_fence_after();
      // whole tile inside every row's window: the first row's end and the last row's start
      const bool inside = key + 128 <= min(blk.p0 + a.right + 1, a.Nk) && !blk.sink(j) &&
                          (key >= blk.p0 + blk.rows - 1 - a.left || key + 128 <= a.sinks);
      const bool edge = !inside || !whole;
      const bool done = nar ? work(std::integral_constant<int, 32>(), j, key, true, kept)
                            : work(std::integral_constant<int, 128>(), j, key, edge, kept);
      if (!done) { ok = false; break; }
      if constexpr (MASK) {
        if (!whole) {
          // masked keys' rows of V: zero (the swizzle moves 16-byte chunks within a row only)
          if (!mbar_wait(&sm.v_full[j % NS], (j / NS) & 1, abort, 511)) { ok = false; break; }
          const uint32_t word = wq == 0 ? kept[0] : wq == 1 ? kept[1] : wq == 2 ? kept[2] : kept[3];
          if (!(word >> lane & 1) && (!nar || row < 32)) {
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(sm.v[j % NS] + s * 128 * 128 + row * 128)[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full);
    }
    // ---------------- O / l -> out, lse ----------------
    if (ok && mbar_wait(&sm.pv_done, (blk.n - 1) & 1, abort, 512)) {
      tc_fence_after();
      const int i = q0 + row;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      T* dst = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.Nq + i) * a.Hq + h) * a.D;
#pragma unroll
      for (int c0 = 0; c0 < DT; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(lane_addr + Cfg::O_COL + c0, o);
        if (i < a.Nq) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float o0 = __uint_as_float(o[8 * v + 2 * e]), o1 = __uint_as_float(o[8 * v + 2 * e + 1]);
              pk[e] = l == 0.f ? 0u : E::pack2(o0 * inv, o1 * inv);
            }
            if (c0 + 8 * v < a.D) *reinterpret_cast<uint4*>(dst + c0 + 8 * v) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
        }
      }
      if (a.lse && i < a.Nq)
        a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i] =
            l == 0.f ? -INFINITY : (fmaf(m, c, log2f(l))) * 0.69314718055994531f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tbase, 256);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
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

template <typename T, int DT, bool MASK>
int launch_wattn_forward(int dtype, const WattnArgs& a, void* out, float* lse, cudaStream_t st) {
  CUtensorMap mq, mk, mv, mk32, mv32;
  if (!wattn_map(&mq, dtype, a.q, a.qs, a.B, a.Nq, a.Hq, a.D, 128) ||
      !wattn_map(&mk, dtype, a.k, a.ks, a.B, a.Nk, a.Hkv, a.D, 128) ||
      !wattn_map(&mv, dtype, a.v, a.vs, a.B, a.Nk, a.Hkv, a.D, 128) ||
      !wattn_map(&mk32, dtype, a.k, a.ks, a.B, a.Nk, a.Hkv, a.D, 32) ||
      !wattn_map(&mv32, dtype, a.v, a.vs, a.B, a.Nk, a.Hkv, a.D, 32))
    return TOPS_ERR_TMAP;
  WattnFwdArgs f;
  f.Nq = a.Nq, f.Nk = a.Nk, f.Hq = a.Hq, f.group = a.Hq / a.Hkv, f.D = a.D;
  f.left = a.left, f.right = a.right, f.sinks = a.sinks, f.tiles = (a.Nq + 127) / 128;
  f.mask = a.mask, f.c = a.scale * kLog2e, f.out = out, f.lse = lse;
  const int64_t grid = static_cast<int64_t>(f.tiles) * a.Hq * a.B;
  if (grid >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  const size_t smem = sizeof(WattnFwdSmem<DT>) + 1024;
  auto kern = wattn_forward_kernel<T, DT, MASK>;
  set_smem(kern, smem);
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
