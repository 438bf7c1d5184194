// wattn_generic.cu — windowed attention with sinks on the CUDA cores: any head size up to
// 256, any element strides, fp32 as well as 16-bit IO, fp32 arithmetic throughout. It is the
// path of fp32 IO and of the shapes the tensor-core kernels do not take: accurate, not tuned.
//
// Forward, one warp per (sequence, head, query): the seen keys 32 at a time, a lane to a key
// for the scores, then a lane to every 32nd channel for P V, with a running maximum and sum.
// Backward, from the saved log-sum-exp, so that P of a pair is one exponential:
//   dQ: one warp per query, the forward's walk once more;
//   dK, dV: one block per key; its warps share the queries that see the key (all later ones
//   for a sink) and their sums are added in a fixed order, so results repeat bit for bit.
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

constexpr int kGenWarps = 4;

// NC: channels per lane (32 NC >= D)
template <typename T, int NC>
__global__ void __launch_bounds__(32 * kGenWarps) wattn_generic_kernel(WattnArgs a, T* __restrict__ out,
                                                                       float* __restrict__ lse) {
  __shared__ float qs[kGenWarps][32 * NC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGenWarps + warp;  // (b, h, i)
  if (row >= static_cast<int64_t>(a.B) * a.Hq * a.Nq) return;
  const int i = static_cast<int>(row % a.Nq);
  const int h = static_cast<int>(row / a.Nq % a.Hq);
  const int b = static_cast<int>(row / a.Nq / a.Hq);
  const int hk = h / (a.Hq / a.Hkv);
  const int nk = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const Seen s = seen_keys(i + nk - a.Nq, a.left, a.right, a.sinks, nk);
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  for (int d = lane; d < a.D; d += 32) qs[warp][d] = load_f(q + d) * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = 0.f;
  const int total = s.n_sink + s.hi - s.lo;
  for (int t0 = 0; t0 < total; t0 += 32) {
    const int t = t0 + lane;
    const int j = t < s.n_sink ? t : s.lo + t - s.n_sink;
    float x = -INFINITY;
    if (t < total && (!a.mask || a.mask[static_cast<int64_t>(b) * a.Nk + j])) {
      const T* kr = k + j * a.ks[1];
      x = 0.f;
      for (int d = 0; d < a.D; ++d) x = fmaf(qs[warp][d], load_f(kr + d), x);
    }
    const float top = fmaxf(m, warp_max(x));
    if (top == -INFINITY) continue;
    const float p = x == -INFINITY ? 0.f : expf(x - top);
    const float f = m == -INFINITY ? 0.f : expf(m - top);
    l = l * f + warp_sum(p);
    m = top;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] *= f;
    for (int u = 0; u < 32 && t0 + u < total; ++u) {
      const float pu = __shfl_sync(0xffffffffu, p, u);
      const int ju = __shfl_sync(0xffffffffu, j, u);
      if (pu == 0.f) continue;  // an unseen key's values are not read
      const T* vr = v + ju * a.vs[1];
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < a.D) o[c] = fmaf(pu, load_f(vr + lane + 32 * c), o[c]);
    }
  }
  T* dst = out + ((static_cast<int64_t>(b) * a.Nq + i) * a.Hq + h) * a.D;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN score stays one)
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (lane + 32 * c < a.D) store_f(dst + lane + 32 * c, o[c] * inv);
  if (lse && lane == 0) lse[row] = l == 0.f ? -INFINITY : m + logf(l);
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
  __shared__ float qs[kGenWarps][32 * NC], ds[kGenWarps][32 * NC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGenWarps + warp;
  if (row >= static_cast<int64_t>(a.B) * a.Hq * a.Nq) return;
  const int i = static_cast<int>(row % a.Nq);
  const int h = static_cast<int>(row / a.Nq % a.Hq);
  const int b = static_cast<int>(row / a.Nq / a.Hq);
  const int hk = h / (a.Hq / a.Hkv);
  const Seen s = seen_keys(i + a.Nk - a.Nq, a.left, a.right, a.sinks, a.Nk);
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  const T* d0 = dout + b * s0 + i * s1 + h * s2;
  for (int d = lane; d < a.D; d += 32) {
    qs[warp][d] = load_f(q + d) * a.scale;
    ds[warp][d] = load_f(d0 + d);
  }
  __syncwarp();
  const float ml = lse[row], dl = delta[row];
  float acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = 0.f;
  const int total = ml == -INFINITY ? 0 : s.n_sink + s.hi - s.lo;
  for (int t0 = 0; t0 < total; t0 += 32) {
    const int t = t0 + lane;
    const int j = t < s.n_sink ? t : s.lo + t - s.n_sink;
    float g = 0.f;
    const bool seen = t < total && (!a.mask || a.mask[static_cast<int64_t>(b) * a.Nk + j]);
    if (seen) {
      const T* kr = k + j * a.ks[1];
      const T* vr = v + j * a.vs[1];
      float x = 0.f, y = 0.f;
      for (int d = 0; d < a.D; ++d) {
        x = fmaf(qs[warp][d], load_f(kr + d), x);
        y = fmaf(ds[warp][d], load_f(vr + d), y);
      }
      g = expf(x - ml) * (y - dl) * a.scale;
    }
    const unsigned any = __ballot_sync(0xffffffffu, seen);
    for (int u = 0; u < 32; ++u) {
      if (!(any >> u & 1)) continue;
      const float gu = __shfl_sync(0xffffffffu, g, u);
      const T* kr = k + __shfl_sync(0xffffffffu, j, u) * a.ks[1];
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < a.D) acc[c] = fmaf(gu, load_f(kr + lane + 32 * c), acc[c]);
    }
  }
  T* dst = dq + ((static_cast<int64_t>(b) * a.Nq + i) * a.Hq + h) * a.D;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (lane + 32 * c < a.D) store_f(dst + lane + 32 * c, acc[c]);
}

template <typename T, int NC>
__global__ void __launch_bounds__(32 * kGenWarps)
    wattn_generic_dkv_kernel(WattnArgs a, const T* __restrict__ dout, int64_t s0, int64_t s1, int64_t s2,
                             const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk,
                             T* __restrict__ dv) {
  __shared__ float ks[32 * NC], vs[32 * NC], part[kGenWarps][2][32 * NC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;  // (b, j, hk): the layout of dk and dv
  const int hk = static_cast<int>(row % a.Hkv);
  const int j = static_cast<int>(row / a.Hkv % a.Nk);
  const int b = static_cast<int>(row / a.Hkv / a.Nk);
  const int g = a.Hq / a.Hkv, off = a.Nk - a.Nq;
  const bool kept = !a.mask || a.mask[static_cast<int64_t>(b) * a.Nk + j];
  int lo, hi;
  seen_by(j, a.left, a.right, a.sinks, a.Nk, lo, hi);
  lo = max(lo - off, 0);  // as queries
  hi -= off;
  const int per = hi > lo && kept ? hi - lo : 0, total = per * g;
  const T* kr = static_cast<const T*>(a.k) + b * a.ks[0] + j * a.ks[1] + hk * a.ks[2];
  const T* vr = static_cast<const T*>(a.v) + b * a.vs[0] + j * a.vs[1] + hk * a.vs[2];
  if (kept)
    for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
      ks[d] = load_f(kr + d) * a.scale;
      vs[d] = load_f(vr + d);
    }
  __syncthreads();
  float ak[NC], av[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) ak[c] = av[c] = 0.f;
  for (int t0 = warp * 32; t0 < total; t0 += 32 * kGenWarps) {
    const int t = t0 + lane;
    const int h = hk * g + t / max(per, 1), i = lo + t % max(per, 1);
    float p = 0.f, w = 0.f;
    bool seen = t < total;
    if (seen) {
      const int64_t r = (static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i;
      const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
      const T* d0 = dout + b * s0 + i * s1 + h * s2;
      float x = 0.f, y = 0.f;
      for (int d = 0; d < a.D; ++d) {
        x = fmaf(ks[d], load_f(q + d), x);
        y = fmaf(vs[d], load_f(d0 + d), y);
      }
      p = lse[r] == -INFINITY ? 0.f : expf(x - lse[r]);
      w = p * (y - delta[r]) * a.scale;
    }
    const int live = min(32, total - t0);
    for (int u = 0; u < live; ++u) {
      const float pu = __shfl_sync(0xffffffffu, p, u), wu = __shfl_sync(0xffffffffu, w, u);
      const int hu = __shfl_sync(0xffffffffu, h, u), iu = __shfl_sync(0xffffffffu, i, u);
      const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + iu * a.qs[1] + hu * a.qs[2];
      const T* d0 = dout + b * s0 + iu * s1 + hu * s2;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < a.D) {
          ak[c] = fmaf(wu, load_f(q + lane + 32 * c), ak[c]);
          av[c] = fmaf(pu, load_f(d0 + lane + 32 * c), av[c]);
        }
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    part[warp][0][lane + 32 * c] = ak[c];
    part[warp][1][lane + 32 * c] = av[c];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kGenWarps; ++w) {
      x += part[w][0][d];
      y += part[w][1][d];
    }
    store_f(dk + row * a.D + d, x);
    store_f(dv + row * a.D + d, y);
  }
}

template <typename F>
int by_channels(int D, F&& f) {
  if (D <= 32) return f(std::integral_constant<int, 1>());
  if (D <= 64) return f(std::integral_constant<int, 2>());
  if (D <= 128) return f(std::integral_constant<int, 4>());
  return f(std::integral_constant<int, 8>());
}

template <typename T>
int run_wattn_generic(const WattnArgs& a, void* out, float* lse, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  const unsigned grid = static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps);
  return by_channels(a.D, [&](auto nc) {
    wattn_generic_kernel<T, decltype(nc)::value><<<grid, 32 * kGenWarps, 0, st>>>(a, static_cast<T*>(out), lse);
    return launch_status();
  });
}

template <typename T>
int run_wattn_delta(const WattnArgs& a, const void* dout, const int64_t* ds, const void* out, float* delta,
                    cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  if (rows == 0) return TOPS_OK;
  wattn_delta_kernel<T><<<static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 32 * kGenWarps, 0, st>>>(
      a, static_cast<const T*>(dout), ds[0], ds[1], ds[2], static_cast<const T*>(out), delta);
  return launch_status();
}

template <typename T>
int run_wattn_generic_backward(const WattnArgs& a, const void* dout, const int64_t* ds, const float* lse,
                               const float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Nq, keys = static_cast<int64_t>(a.B) * a.Hkv * a.Nk;
  const T* d = static_cast<const T*>(dout);
  return by_channels(a.D, [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    if (rows > 0)
      wattn_generic_dq_kernel<T, NC>
          <<<static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 32 * kGenWarps, 0, st>>>(
            a, d, ds[0], ds[1], ds[2], lse, delta, static_cast<T*>(dq));
    if (const int rc = launch_status()) return rc;
    wattn_generic_dkv_kernel<T, NC><<<static_cast<unsigned>(keys), 32 * kGenWarps, 0, st>>>(
        a, d, ds[0], ds[1], ds[2], lse, delta, static_cast<T*>(dk), static_cast<T*>(dv));
    return launch_status();
  });
}

}  // namespace tops
