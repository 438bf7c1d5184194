// wattn_generic.cu — windowed attention with sinks on the CUDA cores: any head size up to
// 256, any element strides, fp32 as well as 16-bit IO, fp32 arithmetic throughout. It is the
// path of fp32 IO and of the shapes the tensor-core kernels do not take.
//
// One plan for the forward, dQ and dK with dV: a block keeps 32 rows of one key head in shared
// memory (queries of the heads that share it, or keys), four to a warp, and tiles of 32 rows of the
// other side stream by. For the scores a lane is a streamed row (its 16 bytes against the four
// rows' broadcasts: 16 products for 5 reads), for the sums a lane is every 32nd channel. Forward with
// a running maximum and sum; backward from the saved log-sum-exp, so that P of a pair is one
// exponential. All sums in a fixed order: results repeat bit for bit.
//
// Bound by shared memory's reads and the latency between a tile's steps: fp32, 2 x 4096 queries, 16
// heads of 128, window 512: forward 1.9 ms (18 TFLOP/s), backward 5.4 ms, for 30 and 118 with a warp
// a query that reads rows straight from memory; one token of 8 sequences, 32 heads on 8, window
// 4096: 0.80 ms for 3.7.
#include <cuda_runtime.h>
#include "sm100.cuh"
#include "status.h"
#include "wattn.h"

namespace tops {

template <typename T>
__device__ __forceinline__ float load_f(const T* p) {
  return static_cast<float>(*p);
}
template <typename T>
__device__ __forceinline__ void store_f(T* p, float v) {
  *p = static_cast<T>(v);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kGenWarps = 8, kGenRows = 4, kGenTile = 32;  // rows a warp; rows a block, and of a streamed tile
static_assert(kGenWarps * kGenRows == kGenTile, "");
constexpr int gen_pitch(int nc) { return 32 * nc + 4; }  // of a staged row: a lane's 16 bytes of 8 rows in 8 banks

// rows [0, 32) of `from` to shared memory, times f; zeros where ok(row) says so and past channel D. Loads
// go out eight at a time: one by one, each would wait for memory on its own.
template <typename T, int NC, typename Row, typename Ok>
__device__ __forceinline__ void gen_stage(float* to, int D, float f, Row&& from, Ok&& ok) {
  constexpr int DP = 32 * NC, PASSES = kGenTile * DP / (32 * kGenWarps), BATCH = PASSES < 8 ? PASSES : 8;
  const int d = threadIdx.x % DP, row0 = threadIdx.x / DP;
#pragma unroll 1
  for (int p = 0; p < PASSES; p += BATCH) {
    float v[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int row = row0 + (p + i) * (kGenTile / PASSES);
      v[i] = d < D && ok(row) ? load_f(from(row) + d) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) to[(row0 + (p + i) * (kGenTile / PASSES)) * gen_pitch(NC) + d] = v[i] * f;
  }
}

// x[r] = dot of the lane's streamed row with the warp's row r
template <int NC>
__device__ __forceinline__ void gen_dots(const float* mine, const float* rows, int D, float* x) {
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) x[r] = 0.f;
#pragma unroll 2
  for (int d = 0; d < D; d += 4) {
    const float4 u = *reinterpret_cast<const float4*>(mine + d);
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) {
      const float4 w = *reinterpret_cast<const float4*>(rows + r * gen_pitch(NC) + d);
      x[r] = fmaf(u.x, w.x, fmaf(u.y, w.y, fmaf(u.z, w.z, fmaf(u.w, w.w, x[r]))));
    }
  }
}

// acc[r][c] += sum over the 32 streamed rows of f[row][r] times its channels
template <int NC, int STEP>
__device__ __forceinline__ void gen_sums(const float* f, const float* rows, int lane, float (*acc)[NC]) {
#pragma unroll 4
  for (int u = 0; u < kGenTile; ++u) {
    const float4 w = *reinterpret_cast<const float4*>(f + u * STEP);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float v = rows[u * gen_pitch(NC) + lane + 32 * c];
      acc[0][c] = fmaf(w.x, v, acc[0][c]);
      acc[1][c] = fmaf(w.y, v, acc[1][c]);
      acc[2][c] = fmaf(w.z, v, acc[2][c]);
      acc[3][c] = fmaf(w.w, v, acc[3][c]);
    }
  }
}

// A block's 32 queries: rows (query, head of the group) in that order, of one key head; and the keys
// that any of them sees before the mask: sinks [0, nse), then [start, end).
struct GenQueries {
  int b, hk, g, nk, start, end, nse;
  int64_t row0, rows;
  __device__ explicit GenQueries(const WattnArgs& a) {
    g = a.Hq / a.Hkv;
    rows = static_cast<int64_t>(a.Nq) * g;
    const int64_t tiles = (rows + kGenTile - 1) / kGenTile;
    row0 = blockIdx.x % tiles * kGenTile;
    hk = static_cast<int>(blockIdx.x / tiles % a.Hkv);
    b = static_cast<int>(blockIdx.x / tiles / a.Hkv);
    nk = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
    const int64_t last = min(row0 + kGenTile, rows) - 1;
    start = of(a, row0).lo;
    end = max(start, of(a, last).hi);
    nse = min(a.sinks, start);
  }
  __device__ int query(int64_t row) const { return static_cast<int>(row / g); }
  __device__ int head(int64_t row) const { return hk * g + static_cast<int>(row % g); }
  __device__ Seen of(const WattnArgs& a, int64_t row) const {
    return seen_keys(query(row) + nk - a.Nq, a.left, a.right, a.sinks, nk);
  }
  __device__ int total() const { return nse + end - start; }
  __device__ int key(int t) const { return t < nse ? t : start + t - nse; }
};

// NC: channels per lane (32 NC >= D)
template <typename T, int NC>
__global__ void __launch_bounds__(32 * kGenWarps) wattn_generic_kernel(WattnArgs a, T* __restrict__ out,
                                                                       float* __restrict__ lse) {
  constexpr int P = gen_pitch(NC), TILE = kGenTile * P;
  extern __shared__ __align__(16) float gen_smem[];
  float *qs = gen_smem, *ks = qs + TILE, *vs = ks + TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* ps = vs + TILE + warp * kGenTile * kGenRows;
  const GenQueries w(a);
  const T* k = static_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[2];
  gen_stage<T, NC>(qs, a.D, a.scale, [&](int r) {
    return static_cast<const T*>(a.q) + w.b * a.qs[0] + w.query(w.row0 + r) * a.qs[1] + w.head(w.row0 + r) * a.qs[2];
  }, [&](int r) { return w.row0 + r < w.rows; });
  int lo[kGenRows], hi[kGenRows];
  float m[kGenRows], l[kGenRows], o[kGenRows][NC];
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int64_t row = w.row0 + warp * kGenRows + r;
    const Seen s = row < w.rows ? w.of(a, row) : Seen{0, 0, 0};
    lo[r] = s.lo, hi[r] = s.hi, m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[r][c] = 0.f;
  }
  const int total = w.total();
  for (int t0 = 0; t0 < total; t0 += kGenTile) {
    __syncthreads();
    auto ok = [&](int r) {
      return t0 + r < total && (!a.mask || a.mask[static_cast<int64_t>(w.b) * a.Nk + w.key(t0 + r)]);
    };
    gen_stage<T, NC>(ks, a.D, 1.f, [&](int r) { return k + w.key(t0 + r) * a.ks[1]; }, ok);
    gen_stage<T, NC>(vs, a.D, 1.f, [&](int r) { return v + w.key(t0 + r) * a.vs[1]; }, ok);
    __syncthreads();
    const int j = w.key(t0 + lane);
    const bool there = ok(lane);
    bool see[kGenRows], any = false;
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) any |= see[r] = there && j < hi[r] && (j >= lo[r] || j < a.sinks);
    if (!__any_sync(0xffffffffu, any)) continue;
    float x[kGenRows], f[kGenRows];
    gen_dots<NC>(ks + lane * P, qs + warp * kGenRows * P, a.D, x);
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) {
      if (!see[r]) x[r] = -INFINITY;
      const float top = fmaxf(m[r], warp_max(x[r]));
      f[r] = top == -INFINITY ? 1.f : m[r] == -INFINITY ? 0.f : expf(m[r] - top);
      x[r] = x[r] == -INFINITY || top == -INFINITY ? 0.f : expf(x[r] - top);
      l[r] = l[r] * f[r] + warp_sum(x[r]);
      m[r] = top;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[r][c] *= f[r];
    }
    __syncwarp();
    *reinterpret_cast<float4*>(ps + lane * kGenRows) = make_float4(x[0], x[1], x[2], x[3]);
    __syncwarp();
    gen_sums<NC, kGenRows>(ps, vs, lane, o);
  }
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int64_t row = w.row0 + warp * kGenRows + r;
    if (row >= w.rows) continue;
    const int i = w.query(row), h = w.head(row);
    T* dst = out + ((static_cast<int64_t>(w.b) * a.Nq + i) * a.Hq + h) * a.D;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];  // (a NaN score stays one)
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (lane + 32 * c < a.D) store_f(dst + lane + 32 * c, o[r][c] * inv);
    if (lse && lane == 0)
      lse[(static_cast<int64_t>(w.b) * a.Hq + h) * a.Nq + i] = l[r] == 0.f ? -INFINITY : m[r] + logf(l[r]);
  }
}

// delta[b][h][i] = sum_d dO O
template <typename T>
__global__ void __launch_bounds__(32 * kGenWarps) wattn_delta_kernel(WattnArgs a, const T* __restrict__ dout,
                                                                     int64_t s0, int64_t s1, int64_t s2,
                                                                     const T* __restrict__ out,
                                                                     float* __restrict__ delta) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGenWarps + (threadIdx.x >> 5);  // (b, i, h)
  if (row >= static_cast<int64_t>(a.B) * a.Hq * a.Nq) return;
  const int lane = threadIdx.x & 31;
  const int h = static_cast<int>(row % a.Hq);
  const int i = static_cast<int>(row / a.Hq % a.Nq);
  const int b = static_cast<int>(row / a.Hq / a.Nq);
  const T* d = dout + b * s0 + i * s1 + h * s2;
  const T* o = out + row * a.D;
  float x = 0.f;
  for (int c = lane; c < a.D; c += 32) x = fmaf(load_f(d + c), load_f(o + c), x);
  x = warp_sum(x);
  if (lane == 0) delta[(static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i] = x;
}

template <typename T, int NC>
__global__ void __launch_bounds__(32 * kGenWarps)
    wattn_generic_dq_kernel(WattnArgs a, const T* __restrict__ dout, int64_t s0, int64_t s1, int64_t s2,
                            const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dq) {
  constexpr int P = gen_pitch(NC), TILE = kGenTile * P;
  extern __shared__ __align__(16) float gen_smem[];
  float *qs = gen_smem, *ds = qs + TILE, *ks = ds + TILE, *vs = ks + TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* gs = vs + TILE + warp * kGenTile * kGenRows;
  const GenQueries w(a);
  const T* k = static_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[2];
  auto there = [&](int r) { return w.row0 + r < w.rows; };
  gen_stage<T, NC>(qs, a.D, a.scale, [&](int r) {
    return static_cast<const T*>(a.q) + w.b * a.qs[0] + w.query(w.row0 + r) * a.qs[1] + w.head(w.row0 + r) * a.qs[2];
  }, there);
  gen_stage<T, NC>(ds, a.D, 1.f, [&](int r) {
    return dout + w.b * s0 + w.query(w.row0 + r) * s1 + w.head(w.row0 + r) * s2;
  }, there);
  int lo[kGenRows], hi[kGenRows];
  float ml[kGenRows], dl[kGenRows], acc[kGenRows][NC];
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int64_t row = w.row0 + warp * kGenRows + r;
    Seen s = {0, 0, 0};
    ml[r] = -INFINITY, dl[r] = 0.f;
    if (row < w.rows) {
      const int64_t at = (static_cast<int64_t>(w.b) * a.Hq + w.head(row)) * a.Nq + w.query(row);
      ml[r] = lse[at], dl[r] = delta[at];
      if (ml[r] != -INFINITY) s = w.of(a, row);  // a query that sees nothing passes nothing on
    }
    lo[r] = s.lo, hi[r] = s.hi;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[r][c] = 0.f;
  }
  const int total = w.total();
  for (int t0 = 0; t0 < total; t0 += kGenTile) {
    __syncthreads();
    auto ok = [&](int r) {
      return t0 + r < total && (!a.mask || a.mask[static_cast<int64_t>(w.b) * a.Nk + w.key(t0 + r)]);
    };
    gen_stage<T, NC>(ks, a.D, 1.f, [&](int r) { return k + w.key(t0 + r) * a.ks[1]; }, ok);
    gen_stage<T, NC>(vs, a.D, 1.f, [&](int r) { return v + w.key(t0 + r) * a.vs[1]; }, ok);
    __syncthreads();
    const int j = w.key(t0 + lane);
    const bool key_ok = ok(lane);
    bool see[kGenRows], any = false;
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) any |= see[r] = key_ok && j < hi[r] && (j >= lo[r] || j < a.sinks);
    if (!__any_sync(0xffffffffu, any)) continue;
    float x[kGenRows], y[kGenRows];
    gen_dots<NC>(ks + lane * P, qs + warp * kGenRows * P, a.D, x);
    gen_dots<NC>(vs + lane * P, ds + warp * kGenRows * P, a.D, y);
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) x[r] = see[r] ? expf(x[r] - ml[r]) * (y[r] - dl[r]) * a.scale : 0.f;
    __syncwarp();
    *reinterpret_cast<float4*>(gs + lane * kGenRows) = make_float4(x[0], x[1], x[2], x[3]);
    __syncwarp();
    gen_sums<NC, kGenRows>(gs, ks, lane, acc);
  }
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int64_t row = w.row0 + warp * kGenRows + r;
    if (row >= w.rows) continue;
    T* dst = dq + ((static_cast<int64_t>(w.b) * a.Nq + w.query(row)) * a.Hq + w.head(row)) * a.D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (lane + 32 * c < a.D) store_f(dst + lane + 32 * c, acc[r][c]);
  }
}

// A block: 32 keys of one key head; the queries that any of them meets, one head of the group after
// the other (a key that is a sink meets all later ones).
template <typename T, int NC>
__global__ void __launch_bounds__(32 * kGenWarps)
    wattn_generic_dkv_kernel(WattnArgs a, const T* __restrict__ dout, int64_t s0, int64_t s1, int64_t s2,
                             const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk,
                             T* __restrict__ dv) {
  constexpr int P = gen_pitch(NC), TILE = kGenTile * P;
  extern __shared__ __align__(16) float gen_smem[];
  float *ks = gen_smem, *vs = ks + TILE, *qs = vs + TILE, *ds = qs + TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* fs = ds + TILE + warp * kGenTile * 2 * kGenRows;  // of a query: the four dS, the four P
  const int tiles = (a.Nk + kGenTile - 1) / kGenTile;
  const int j0 = static_cast<int>(blockIdx.x % tiles) * kGenTile, hk = static_cast<int>(blockIdx.x / tiles % a.Hkv);
  const int b = static_cast<int>(blockIdx.x / tiles / a.Hkv);
  const int g = a.Hq / a.Hkv, off = a.Nk - a.Nq;
  auto kept = [&](int r) { return j0 + r < a.Nk && (!a.mask || a.mask[static_cast<int64_t>(b) * a.Nk + j0 + r]); };
  gen_stage<T, NC>(ks, a.D, a.scale, [&](int r) {
    return static_cast<const T*>(a.k) + b * a.ks[0] + (j0 + r) * a.ks[1] + hk * a.ks[2];
  }, kept);
  gen_stage<T, NC>(vs, a.D, 1.f, [&](int r) {
    return static_cast<const T*>(a.v) + b * a.vs[0] + (j0 + r) * a.vs[1] + hk * a.vs[2];
  }, kept);
  int lo[kGenRows], hi[kGenRows], first, end, none;  // as queries
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int key = warp * kGenRows + r;
    lo[r] = hi[r] = 0;
    if (kept(key)) {
      seen_by(j0 + key, a.left, a.right, a.sinks, a.Nk, lo[r], hi[r]);
      lo[r] = max(lo[r] - off, 0), hi[r] -= off;
    }
  }
  seen_by(j0, a.left, a.right, a.sinks, a.Nk, first, end);  // (the first key sinks if any does)
  const int last = min(j0 + kGenTile, a.Nk) - 1;
  int to;
  seen_by(last, a.left, a.right, a.sinks, a.Nk, none, to);
  first = max(first - off, 0), end = max(end, to) - off;
  float ak[kGenRows][NC], av[kGenRows][NC];
#pragma unroll
  for (int r = 0; r < kGenRows; ++r)
#pragma unroll
    for (int c = 0; c < NC; ++c) ak[r][c] = av[r][c] = 0.f;
  for (int h = hk * g; h < hk * g + g; ++h)
    for (int i0 = first; i0 < end; i0 += kGenTile) {
      __syncthreads();
      const int64_t stat = (static_cast<int64_t>(b) * a.Hq + h) * a.Nq;
      auto ok = [&](int r) { return i0 + r < end && lse[stat + i0 + r] != -INFINITY; };
      gen_stage<T, NC>(qs, a.D, 1.f, [&](int r) {
        return static_cast<const T*>(a.q) + b * a.qs[0] + (i0 + r) * a.qs[1] + h * a.qs[2];
      }, ok);
      gen_stage<T, NC>(ds, a.D, 1.f, [&](int r) { return dout + b * s0 + (i0 + r) * s1 + h * s2; }, ok);
      __syncthreads();
      const int i = i0 + lane;
      const bool there = ok(lane);
      bool see[kGenRows], any = false;
#pragma unroll
      for (int r = 0; r < kGenRows; ++r) any |= see[r] = there && i >= lo[r] && i < hi[r];
      if (!__any_sync(0xffffffffu, any)) continue;
      const float ml = there ? lse[stat + i] : 0.f, dl = there ? delta[stat + i] : 0.f;
      float x[kGenRows], y[kGenRows];
      gen_dots<NC>(qs + lane * P, ks + warp * kGenRows * P, a.D, x);
      gen_dots<NC>(ds + lane * P, vs + warp * kGenRows * P, a.D, y);
#pragma unroll
      for (int r = 0; r < kGenRows; ++r) {
        x[r] = see[r] ? expf(x[r] - ml) : 0.f;
        y[r] = see[r] ? x[r] * (y[r] - dl) * a.scale : 0.f;
      }
      __syncwarp();
      *reinterpret_cast<float4*>(fs + lane * 2 * kGenRows) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(fs + lane * 2 * kGenRows + kGenRows) = make_float4(x[0], x[1], x[2], x[3]);
      __syncwarp();
      gen_sums<NC, 2 * kGenRows>(fs, qs, lane, ak);
      gen_sums<NC, 2 * kGenRows>(fs + kGenRows, ds, lane, av);
    }
#pragma unroll
  for (int r = 0; r < kGenRows; ++r) {
    const int j = j0 + warp * kGenRows + r;
    if (j >= a.Nk) continue;
    const int64_t at = ((static_cast<int64_t>(b) * a.Nk + j) * a.Hkv + hk) * a.D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (lane + 32 * c < a.D) {
        store_f(dk + at + lane + 32 * c, ak[r][c]);
        store_f(dv + at + lane + 32 * c, av[r][c]);
      }
  }
}

template <typename F>
int by_channels(int D, F&& f) {
  if (D <= 32) return f(std::integral_constant<int, 1>());
  if (D <= 64) return f(std::integral_constant<int, 2>());
  if (D <= 128) return f(std::integral_constant<int, 4>());
  return f(std::integral_constant<int, 8>());
}

// blocks of 32 of `rows` rows for each key head of each sequence
inline int64_t gen_blocks(const WattnArgs& a, int64_t rows) {
  return (rows + kGenTile - 1) / kGenTile * a.Hkv * a.B;
}
// bytes of `tiles` staged tiles and `per` factors a streamed row and warp
constexpr size_t gen_smem_bytes(int nc, int tiles, int per) {
  return sizeof(float) * kGenTile * (static_cast<size_t>(tiles) * gen_pitch(nc) + kGenWarps * per);
}

template <typename T>
int run_wattn_generic(const WattnArgs& a, void* out, float* lse, cudaStream_t st) {
  const int64_t grid = gen_blocks(a, static_cast<int64_t>(a.Nq) * (a.Hq / a.Hkv));
  if (grid >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  return by_channels(a.D, [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    constexpr size_t smem = gen_smem_bytes(NC, 3, kGenRows);
    if (smem > 48 * 1024) set_smem(wattn_generic_kernel<T, NC>, smem);
    wattn_generic_kernel<T, NC>
        <<<static_cast<unsigned>(grid), 32 * kGenWarps, smem, st>>>(a, static_cast<T*>(out), lse);
    return launch_status();
  });
}

template <typename T>
int run_wattn_delta(const WattnArgs& a, const void* dout, const int64_t* ds, const void* out, float* delta,
                    cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  wattn_delta_kernel<T><<<static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 32 * kGenWarps, 0, st>>>(
      a, static_cast<const T*>(dout), ds[0], ds[1], ds[2], static_cast<const T*>(out), delta);
  return launch_status();
}

template <typename T>
int run_wattn_generic_backward(const WattnArgs& a, const void* dout, const int64_t* ds, const float* lse,
                               const float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
  const int64_t rows = gen_blocks(a, static_cast<int64_t>(a.Nq) * (a.Hq / a.Hkv)), keys = gen_blocks(a, a.Nk);
  if (rows >= (int64_t(1) << 31) || keys >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  const T* d = static_cast<const T*>(dout);
  return by_channels(a.D, [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    constexpr size_t smem_q = gen_smem_bytes(NC, 4, kGenRows), smem_kv = gen_smem_bytes(NC, 4, 2 * kGenRows);
    if (smem_q > 48 * 1024) set_smem(wattn_generic_dq_kernel<T, NC>, smem_q);
    if (smem_kv > 48 * 1024) set_smem(wattn_generic_dkv_kernel<T, NC>, smem_kv);
    wattn_generic_dq_kernel<T, NC><<<static_cast<unsigned>(rows), 32 * kGenWarps, smem_q, st>>>(
        a, d, ds[0], ds[1], ds[2], lse, delta, static_cast<T*>(dq));
    if (const int rc = launch_status()) return rc;
    wattn_generic_dkv_kernel<T, NC><<<static_cast<unsigned>(keys), 32 * kGenWarps, smem_kv, st>>>(
        a, d, ds[0], ds[1], ds[2], lse, delta, static_cast<T*>(dk), static_cast<T*>(dv));
    return launch_status();
  });
}

}  // namespace tops
