// gnorm.cu — what stands between two blocks of a residual stream, in one pass: the norm after
// a block, its gate and residual scale, the residual add, and the norm before the next block.
//
//   u = post(y)                         (or y)
//   r = u * sigmoid(gate)               (or u)
//   h = x + s * r                       (s per channel, or 1)
//   n = pre(h)                          (optional)
//   layer: norm(t) = (t - mean) / sqrt(var + eps) * w + b;  rms: t / sqrt(mean(t^2) + eps) * w
//
// Backward, with t^ the normalised t and rstd its factor: for d the gradient of norm(t),
//   dt = rstd (d w - t^ mean(d w t^) - mean(d w)),  dw = sum d t^,  db = sum d
//   (rms without the last mean),
// through pre into h, then ds = sum dh r, dr = dh s, dgate = dr u sg (1 - sg), du = dr sg, and
// through post into y; dx = dh.
//
// Bound by memory: forward reads x, y and the gate and writes h and n, backward reads x, y, the
// gate, dh and dn and writes dx, dy and dgate, each once; h is computed again from x and y (not
// read back rounded). Everything between is fp32 in registers; the variance is the mean of
// squared distances from the mean (two passes over registers). A thread owns the same 8 channels
// of every row it works on, so the weights stay in its registers, and so do the weights'
// gradients, which leave as one partial row per block and are added up in a fixed order.
// 1024 x 1024 rows of 128 channels in 16 bits, a gate a row: forward 0.23 ms (5.8 TB/s), backward 0.43 ms
// (4.9 TB/s, the issue slots 66 % busy).
#include <cuda_runtime.h>
#include "sm100.cuh"
#include "status.h"

namespace tops {

struct GnormArgs {
  int64_t rows;            // tokens
  int64_t group_rows;      // consecutive tokens that share a row of the gate (a gate of their own: all)
  int64_t groups;          // such groups
  int shared;              // tokens share the gate
  int C;
  int layer, has_post, has_pre;
  int w_io;                // weights and their gradients in the IO dtype (else fp32)
  float eps;
  int xs, ys, gs, dhs, dns;      // row strides in elements
  const void *x, *y, *gate, *dh, *dn;
  const void *post_w, *post_b, *res_s, *pre_w, *pre_b;  // null: 1, 0, 1, 1, 0
  void *h, *n;
  float* stats;            // [rows][4]: mean and 1/std of y, mean and 1/std of h
  void *dx, *dy, *dgate;
  float* part;             // [blocks][5][C]: gradients of post_w, post_b, res_s, pre_w, pre_b
  float* gpart;            // [groups][splits][C], or null where a group has one block
  int splits;              // blocks that share a group
  int summed;              // a kernel that adds up the parts follows
  int tpr;                 // threads to a row
};

// A thread holds V channels of a row as V / 2 pairs (packed fp32 arithmetic): 8 in the forward, 4 in
// the backward, whose 5 sums a channel would not leave it registers for enough threads otherwise
// (1024 x 1024 x 128 in 16 bits: 0.60 ms with 8 channels a thread, 0.44 with 4).
// Channel of value i of the thread at `t` of a row of tpr threads:
template <int VEC>
__device__ __forceinline__ int gn_channel(int t, int tpr, int i) {
  return (t + (i / VEC) * tpr) * VEC + i % VEC;
}

template <typename T>
__device__ __forceinline__ const T* gn_row(const void* p, int row, int stride) {
  return static_cast<const T*>(p) + static_cast<int64_t>(row) * stride;
}
template <typename T>
__device__ __forceinline__ T* gn_row(void* p, int row, int stride) {
  return static_cast<T*>(p) + static_cast<int64_t>(row) * stride;
}

// A thread's channels as they lie in memory: 8- or 16-byte pieces of VEC values, or (VEC 1) one by
// one. Channels past C are zero.
template <typename T, int VEC, int V>
struct GnRaw {
  static constexpr int WORDS = VEC * sizeof(T) / 4;  // of a piece
  uint32_t w[V / VEC * WORDS];
  __device__ __forceinline__ void load(const T* p, int t, int tpr, int C) {
#pragma unroll
    for (int k = 0; k < V / VEC; ++k) {
      const int c = (t + k * tpr) * VEC;
      uint32_t* d = w + k * WORDS;
      if constexpr (WORDS == 4) {
        const uint4 u = c < C ? *reinterpret_cast<const uint4*>(p + c) : make_uint4(0, 0, 0, 0);
        d[0] = u.x, d[1] = u.y, d[2] = u.z, d[3] = u.w;
      } else {
        const uint2 u = c < C ? *reinterpret_cast<const uint2*>(p + c) : make_uint2(0, 0);
        d[0] = u.x, d[1] = u.y;
      }
    }
  }
  __device__ __forceinline__ void get(f2* f) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      if constexpr (sizeof(T) == 4)
        f[i] = f2_pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else
        f[i] = f2_pack(Elem<T>::lo(w[i]), Elem<T>::hi(w[i]));
  }
};
template <typename T, int V>
struct GnRaw<T, 1, V> {
  T v[V];
  __device__ __forceinline__ void load(const T* p, int t, int tpr, int C) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = t + i * tpr < C ? p[t + i * tpr] : T(0.f);
  }
  __device__ __forceinline__ void get(f2* f) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) f[i] = f2_pack(static_cast<float>(v[2 * i]), static_cast<float>(v[2 * i + 1]));
  }
};

template <typename T, int VEC, int V>
__device__ __forceinline__ void gn_store(T* p, int t, int tpr, int C, const f2* v) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) f2_unpack(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int k = 0; k < V / VEC; ++k) {
    const int c = (t + k * tpr) * VEC;
    if (c >= C) continue;
    const float* g = f + k * VEC;
    if constexpr (VEC == 1)
      p[c] = static_cast<T>(g[0]);
    else if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(p + c) = make_float4(g[0], g[1], g[2], g[3]);
    else if constexpr (VEC == 4)
      *reinterpret_cast<uint2*>(p + c) = make_uint2(Elem<T>::pack2(g[0], g[1]), Elem<T>::pack2(g[2], g[3]));
    else
      *reinterpret_cast<uint4*>(p + c) = make_uint4(Elem<T>::pack2(g[0], g[1]), Elem<T>::pack2(g[2], g[3]),
                                                    Elem<T>::pack2(g[4], g[5]), Elem<T>::pack2(g[6], g[7]));
  }
}

// A weight row of either dtype, read once a block. Channels past C get 0, whatever the default:
// then nothing of theirs enters a sum.
template <typename T, int VEC, int V>
__device__ __forceinline__ void gn_weight(const void* w, int io, int t, int tpr, int C, float none, f2* f) {
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = gn_channel<VEC>(t, tpr, i);
    v[i] = c < C ? none : 0.f;
    if (w != nullptr && c < C)
      v[i] = io ? static_cast<float>(static_cast<const T*>(w)[c]) : static_cast<const float*>(w)[c];
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) f[i] = f2_pack(v[2 * i], v[2 * i + 1]);
}

// Sums of N values over the threads of a row. TPR: threads to a row, side by side in a warp (0: a
// number that only the launch knows); above 32 the row takes the whole block, and `red` is two
// buffers of N x 32 floats used in turn, so that one barrier a sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float* v, int tpr, float* red, int& turn) {
  if constexpr (TPR == 0) {
    for (int o = tpr >> 1; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  } else {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) >> 1; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (TPR > 32) {
    float* r = red + (turn ^= 1) * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) r[32 * i + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = lane < nw ? r[32 * i + lane] : 0.f;
#pragma unroll
      for (int o = TPR / 64; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      v[i] = __shfl_sync(0xffffffffu, v[i], 0);
    }
  }
}

// 16-bit IO: the hardware's exponential and reciprocal are some ulps of fp32 off, far below its
// rounding; 2^x of a far negative gate is infinite and its reciprocal 0
template <typename T>
__device__ __forceinline__ f2 gn_sigmoid2(f2 x) {
  float a, b;
  if constexpr (sizeof(T) == 4) {
    f2_unpack(x, a, b);
    return f2_pack(1.f / (1.f + expf(-a)), 1.f / (1.f + expf(-b)));
  } else {
    f2_unpack(f2_mul(x, f2_both(-1.4426950408889634f)), a, b);
    f2_unpack(f2_add(f2_pack(ex2_approx(a), ex2_approx(b)), f2_both(1.f)), a, b);
    return f2_pack(rcp_approx(a), rcp_approx(b));
  }
}

// mean and 1/std of a row's values (rms: mean 0)
template <typename T, int VEC, int V, int TPR>
__device__ __forceinline__ float2 gn_stats(const f2* f, int t, int tpr, const GnormArgs& a, float* red, int& turn) {
  const float inv = 1.f / a.C;
  float mean = 0.f, s;
  if (a.layer) {
    f2 sum = f[0];  // channels past C hold 0
#pragma unroll
    for (int i = 1; i < V / 2; ++i) sum = f2_add(sum, f[i]);
    s = f2_sum(sum);
    row_sum<TPR, 1>(&s, tpr, red, turn);
    mean = s * inv;
  }
  f2 acc = 0;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float m0 = gn_channel<VEC>(t, tpr, 2 * i) < a.C ? mean : 0.f;
    const float m1 = VEC > 1 ? m0 : gn_channel<VEC>(t, tpr, 2 * i + 1) < a.C ? mean : 0.f;
    const f2 d = f2_add(f[i], f2_pack(-m0, -m1));
    acc = f2_fma(d, d, acc);
  }
  s = f2_sum(acc);
  row_sum<TPR, 1>(&s, tpr, red, turn);
  s = fmaf(s, inv, a.eps);
  return make_float2(mean, sizeof(T) == 4 ? 1.f / sqrtf(s) : rsqrtf(s));
}

// Rows side by side in blocks of 128 threads (TPR up to 32; 0: a number that only the launch knows),
// or one row a block. Block b takes rows b * slots + slot, then on by the grid; the next row's values
// are on their way while the present one's are worked on. ALL: both norms and a gate (the launch's
// flags are then not asked, which some 40 branches a row would).
template <typename T, int VEC, int TPR, bool ALL>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 128, TPR > 256 ? 1 : TPR == 256 ? 2 : VEC > 1 ? 5 : 4)
    gnorm_forward_kernel(const GnormArgs a) {
  constexpr int V = 8, NP = V / 2;
  __shared__ float red[TPR > 32 ? 128 : 1];
  const bool has_post = ALL || a.has_post, has_pre = ALL || a.has_pre, gated = ALL || a.gate != nullptr;
  int turn = 0;
  const int tpr = TPR > 0 ? TPR : a.tpr;
  const int t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = TPR > 32 ? 1 : blockDim.x / tpr, C = a.C;
  f2 pw[NP], pb[NP], sc[NP], nw[NP], nb[NP];
  gn_weight<T, VEC, V>(a.post_w, a.w_io, t, tpr, C, 1.f, pw);
  gn_weight<T, VEC, V>(a.post_b, a.w_io, t, tpr, C, 0.f, pb);
  gn_weight<T, VEC, V>(a.res_s, a.w_io, t, tpr, C, 1.f, sc);
  gn_weight<T, VEC, V>(a.pre_w, a.w_io, t, tpr, C, 1.f, nw);
  gn_weight<T, VEC, V>(a.pre_b, a.w_io, t, tpr, C, 0.f, nb);
  const int rows = static_cast<int>(a.rows), step = gridDim.x * slots;
  int r = blockIdx.x * slots + slot;
  GnRaw<T, VEC, V> rx = {}, ry = {}, rg = {};
  int group = -1;  // whose gate rg holds, where tokens share one
  auto load = [&](int row) {  // (a thread without a row works on zeros and keeps up with the others)
    if (row >= rows) return;
    rx.load(gn_row<T>(a.x, row, a.xs), t, tpr, C);
    ry.load(gn_row<T>(a.y, row, a.ys), t, tpr, C);
    if (gated && !a.shared) rg.load(gn_row<T>(a.gate, row, a.gs), t, tpr, C);
    if (gated && a.shared) {
      const int of = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.group_rows);
      if (of != group) rg.load(gn_row<T>(a.gate, of, a.gs), t, tpr, C);
      group = of;
    }
  };
  load(r);
  for (int r0 = blockIdx.x * slots; r0 < rows; r0 += step, r += step) {
    f2 x[NP], y[NP], g[NP];
    rx.get(x);
    ry.get(y);
    if (gated) rg.get(g);
    load(r + step);
    float2 sy = make_float2(0.f, 1.f), sh = sy;
    if (has_post) {
      sy = gn_stats<T, VEC, V, TPR>(y, t, tpr, a, red, turn);
      const f2 m = f2_both(-sy.x), q = f2_both(sy.y);
#pragma unroll
      for (int i = 0; i < NP; ++i) y[i] = f2_fma(f2_mul(f2_add(y[i], m), q), pw[i], pb[i]);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (gated) y[i] = f2_mul(y[i], gn_sigmoid2<T>(g[i]));
      x[i] = f2_fma(sc[i], y[i], x[i]);  // h
    }
    const bool live = r < rows;
    if (live) gn_store<T, VEC, V>(gn_row<T>(a.h, r, C), t, tpr, C, x);
    if (has_pre) {
      sh = gn_stats<T, VEC, V, TPR>(x, t, tpr, a, red, turn);
      const f2 m = f2_both(-sh.x), q = f2_both(sh.y);
#pragma unroll
      for (int i = 0; i < NP; ++i) x[i] = f2_fma(f2_mul(f2_add(x[i], m), q), nw[i], nb[i]);
      if (live) gn_store<T, VEC, V>(gn_row<T>(a.n, r, C), t, tpr, C, x);
    }
    if (live && a.stats && t == 0) reinterpret_cast<float4*>(a.stats)[r] = make_float4(sy.x, sy.y, sh.x, sh.y);
  }
}

// Adds each thread's sums over the block's row slots, in order; slot 0 is left with the total.
template <int NP>
__device__ __forceinline__ void slot_sum(f2* f, float* buf, int t, int slot, int slots, int tpr) {
  if (slots == 1) return;
  f2* at = reinterpret_cast<f2*>(buf);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NP; ++i) at[(slot * NP + i) * tpr + t] = f[i];
  __syncthreads();
  if (slot == 0)
    for (int s = 1; s < slots; ++s)
#pragma unroll
      for (int i = 0; i < NP; ++i) f[i] = f2_add(f[i], at[(s * NP + i) * tpr + t]);
}

template <int VEC, int NP>
__device__ __forceinline__ void gn_part(float* p, const f2* v, int t, int tpr, int C) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    float f[2];
    f2_unpack(v[i], f[0], f[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = gn_channel<VEC>(t, tpr, 2 * i + j);
      if (c < C) p[c] = f[j];
    }
  }
}

// Block b takes group b / splits, share b % splits of its rows, then on by the grid. The weights
// wait in shared memory (a thread's sums take the registers).
template <typename T, int VEC, int V, int TPR, bool ALL>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 128, TPR > 512 ? 1 : TPR > 256 ? 2 : TPR > 128 ? 3 : TPR == 64 ? 10 : 5)
    gnorm_backward_kernel(const GnormArgs a) {
  constexpr int NP = V / 2;
  if (a.summed) pdl_trigger();
  __shared__ float red[TPR > 32 ? 128 : 1];
  extern __shared__ __align__(16) float buf[];  // weights [4][NP / 2][tpr] of two pairs, then the row slots' sums
  const bool has_post = ALL || a.has_post, has_pre = ALL || a.has_pre, gated = ALL || a.gate != nullptr;
  const bool has_dh = ALL || a.dh != nullptr, has_dn = ALL || a.dn != nullptr;
  int turn = 0;
  const int tpr = TPR > 0 ? TPR : a.tpr;
  const int t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = TPR > 32 ? 1 : blockDim.x / tpr, C = a.C;
  const float inv = 1.f / C;
  ulonglong2* wts = reinterpret_cast<ulonglong2*>(buf);
  if (slot == 0) {
    f2 w[NP];
    const void* const from[4] = {a.post_w, a.post_b, a.res_s, a.pre_w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      gn_weight<T, VEC, V>(from[k], a.w_io, t, tpr, C, k == 1 ? 0.f : 1.f, w);
#pragma unroll
      for (int i = 0; i < NP / 2; ++i) wts[(k * (NP / 2) + i) * tpr + t] = make_ulonglong2(w[2 * i], w[2 * i + 1]);
    }
  }
  __syncthreads();
  auto weights = [&](int k, f2* w) {
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) {
      const ulonglong2 u = wts[(k * (NP / 2) + i) * tpr + t];
      w[2 * i] = u.x, w[2 * i + 1] = u.y;
    }
  };
  float* sums = buf + 4 * V * tpr;
  f2 apw[NP] = {}, apb[NP] = {}, asc[NP] = {}, anw[NP] = {}, anb[NP] = {};
  const int share = blockIdx.x % a.splits, step = a.splits * slots;
  const int per = static_cast<int>(a.group_rows);
  for (int grp = blockIdx.x / a.splits; grp < a.groups; grp += gridDim.x / a.splits) {
    f2 ag[NP] = {};
    const int r_group = grp * per;
    int i0 = share * slots + slot;  // row of the group
    GnRaw<T, VEC, V> rx = {}, ry = {}, rg = {}, rh = {}, rn = {};
    float4 st_next = make_float4(0.f, 1.f, 0.f, 1.f);
    auto load = [&](int i) {
      if (i >= per) {  // without a row: zero gradients, which add nothing to a sum
        rh = GnRaw<T, VEC, V>{};
        rn = GnRaw<T, VEC, V>{};
        return;
      }
      const int r = r_group + i;
      rx.load(gn_row<T>(a.x, r, a.xs), t, tpr, C);
      ry.load(gn_row<T>(a.y, r, a.ys), t, tpr, C);
      if (gated && !a.shared) rg.load(gn_row<T>(a.gate, r, a.gs), t, tpr, C);
      if (has_dh) rh.load(gn_row<T>(a.dh, r, a.dhs), t, tpr, C);
      if (has_dn) rn.load(gn_row<T>(a.dn, r, a.dns), t, tpr, C);
      st_next = reinterpret_cast<const float4*>(a.stats)[r];
    };
    if (gated && a.shared) rg.load(gn_row<T>(a.gate, grp, a.gs), t, tpr, C);
    load(i0);
    for (int base = share * slots; base < per; base += step, i0 += step) {
      const bool live = i0 < per;
      const int r = r_group + i0;
      f2 x[NP], y[NP], g[NP], dh[NP], dn[NP], w0[NP], w1[NP], w2[NP], w3[NP];
      rx.get(x);
      ry.get(y);
      if (gated) rg.get(g);
      rh.get(dh);
      rn.get(dn);
      const float4 st = st_next;
      load(i0 + step);
      weights(0, w0);
      weights(1, w1);
      weights(2, w2);
      float s[2];
      f2 s1 = 0, s2 = 0;
      // y: normalised y; g: the gate's sigmoid; x: normalised h; dn: d n * pre weight
      weights(3, w3);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (has_post) y[i] = f2_mul(f2_add(y[i], f2_both(-st.x)), f2_both(st.y));
        if (gated) g[i] = gn_sigmoid2<T>(g[i]);
        if (has_pre) {
          f2 u = has_post ? f2_fma(y[i], w0[i], w1[i]) : y[i];
          if (gated) u = f2_mul(u, g[i]);
          x[i] = f2_mul(f2_add(f2_fma(w2[i], u, x[i]), f2_both(-st.z)), f2_both(st.w));
          anw[i] = f2_fma(dn[i], x[i], anw[i]);
          anb[i] = f2_add(dn[i], anb[i]);
          dn[i] = f2_mul(dn[i], w3[i]);
          s1 = f2_fma(dn[i], x[i], s1);
          s2 = f2_add(dn[i], s2);
        }
      }
      if (has_pre) {
        s[0] = f2_sum(s1), s[1] = f2_sum(s2);
        row_sum<TPR, 2>(s, tpr, red, turn);
        const f2 m1 = f2_both(-s[0] * inv), m2 = f2_both(a.layer ? -s[1] * inv : 0.f), q = f2_both(st.w);
#pragma unroll
        for (int i = 0; i < NP; ++i) dh[i] = f2_fma(q, f2_add(f2_fma(x[i], m1, dn[i]), m2), dh[i]);
      }
      if (live) gn_store<T, VEC, V>(gn_row<T>(a.dx, r, C), t, tpr, C, dh);
      s1 = s2 = 0;
      asm volatile("" ::: "memory");  // read the weights again rather than keep them in registers
      weights(0, w0);
      weights(1, w1);
      weights(2, w2);
      // dh: d y^; dn: d gate
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const f2 u = has_post ? f2_fma(y[i], w0[i], w1[i]) : y[i];
        f2 dr = dh[i];
        if (gated) {
          const f2 ug = f2_mul(u, g[i]);
          asc[i] = f2_fma(dr, ug, asc[i]);
          dr = f2_mul(dr, w2[i]);
          // u sg (1 - sg)
          dn[i] = f2_mul(dr, f2_fma(f2_mul(ug, g[i]), f2_both(-1.f), ug));
          ag[i] = f2_add(dn[i], ag[i]);
          dr = f2_mul(dr, g[i]);
        } else {
          asc[i] = f2_fma(dr, u, asc[i]);
          dr = f2_mul(dr, w2[i]);
        }
        if (has_post) {
          apw[i] = f2_fma(dr, y[i], apw[i]);
          apb[i] = f2_add(dr, apb[i]);
          dr = f2_mul(dr, w0[i]);
          s1 = f2_fma(dr, y[i], s1);
          s2 = f2_add(dr, s2);
        }
        dh[i] = dr;
      }
      if (live && gated && !a.shared) gn_store<T, VEC, V>(gn_row<T>(a.dgate, r, C), t, tpr, C, dn);
      if (has_post) {
        s[0] = f2_sum(s1), s[1] = f2_sum(s2);
        row_sum<TPR, 2>(s, tpr, red, turn);
        const f2 m1 = f2_both(-s[0] * inv), m2 = f2_both(a.layer ? -s[1] * inv : 0.f), q = f2_both(st.y);
#pragma unroll
        for (int i = 0; i < NP; ++i) dh[i] = f2_mul(q, f2_add(f2_fma(y[i], m1, dh[i]), m2));
      }
      if (live) gn_store<T, VEC, V>(gn_row<T>(a.dy, r, C), t, tpr, C, dh);
    }
    if (a.shared) {
      slot_sum<NP>(ag, sums, t, slot, slots, tpr);
      if (slot == 0) {
        if (a.gpart)
          gn_part<VEC, NP>(a.gpart + (static_cast<int64_t>(grp) * a.splits + share) * C, ag, t, tpr, C);
        else
          gn_store<T, VEC, V>(gn_row<T>(a.dgate, grp, C), t, tpr, C, ag);
      }
    }
  }
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 5 * C;
  auto leave = [&](f2* v, int k) {
    slot_sum<NP>(v, sums, t, slot, slots, tpr);
    if (slot == 0) gn_part<VEC, NP>(part + k * C, v, t, tpr, C);
  };
  leave(apw, 0);
  leave(apb, 1);
  leave(asc, 2);
  leave(anw, 3);
  leave(anb, 4);
}

// out[set][c] = sum over n of in[set * set_step + n * row_step + c]: the blocks' partial rows, added
// in a fixed order, for the 5 weights and then for the groups of a gate shared by several blocks, in one
// launch (backward of 3 groups of 1367 rows of 771 channels: 43 us with two, 39 with one).
// One block takes 32 channels of one set; its 32 warps share the rows, four loads of a thread at a time.
struct GnReduceArgs {
  const float *part, *gpart;
  int64_t n, splits;  // rows to add of a weight and of a group
  int C, io, first;   // weights in the IO dtype; first set to add: 0, or 5 (no weight's gradient is wanted)
  void* out[5];       // a weight's gradient (null: not wanted)
  void* dgate;
};
template <typename T>
__global__ void __launch_bounds__(1024) gnorm_reduce_kernel(const GnReduceArgs a) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, C = a.C;
  const int set = blockIdx.y + a.first;
  const bool weight = set < 5;
  void* out = weight ? a.out[set] : a.dgate;
  if (out == nullptr) return;
  const int64_t grp = set - 5, step = weight ? 5 * C : C, n = weight ? a.n : a.splits;
  float v = 0.f;
  pdl_wait();
  if (c < C) {
    const float* p = (weight ? a.part + set * C : a.gpart + grp * a.splits * C) + c;
    int i = warp;
    for (; i + 96 < n; i += 128) {
      float u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = p[(i + 32 * k) * step];
#pragma unroll
      for (int k = 0; k < 4; ++k) v += u[k];
    }
    for (; i < n; i += 32) v += p[i * step];
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || c >= C) return;
  v = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) v += s[w][lane];
  const int64_t at = weight ? c : grp * C + c;
  if (a.io || !weight)
    static_cast<T*>(out)[at] = static_cast<T>(v);
  else
    static_cast<float*>(out)[at] = v;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Threads to a row of C channels, V a thread: up to 32 side by side in blocks of 128, else a block.
struct GnormShape {
  int tpr, threads, slots;
  GnormShape(int64_t C, int V) {
    tpr = 8;
    while (static_cast<int64_t>(tpr) * V < C) tpr *= 2;
    threads = tpr <= 32 ? 128 : tpr;
    slots = threads / tpr;
  }
};

struct GnormPlan {
  GnormShape fwd, bwd;
  int v;              // channels a thread in the backward
  int64_t blocks, bblocks;
  int splits;
  bool shared, gpart;
  int64_t groups;
};

inline GnormPlan gnorm_plan(int64_t rows, int64_t gate_rows, int64_t C) {
  const int v = C <= 4096 ? 4 : 8;
  GnormPlan p = {GnormShape(C, 8), GnormShape(C, v), v, 0, 0, 0, false, false, 0};
  p.shared = gate_rows < rows;
  const int64_t groups = p.groups = p.shared ? gate_rows : 1;
  const int64_t sms = sm_count();
  // as many blocks as the kernels' launch bounds let the SMs hold
  auto resident = [&](int threads) -> int64_t {
    if (threads > 512) return sms;
    if (threads > 256) return sms * 2;
    if (threads > 128) return sms * 3;
    return sms * (threads == 64 ? 10 : 5);
  };
  const int64_t need = (rows + p.fwd.slots - 1) / p.fwd.slots, most = resident(p.fwd.threads);
  p.blocks = need < most ? need : most;
  const int64_t per = rows / groups, bmost = resident(p.bwd.threads);
  const int64_t gneed = (per + p.bwd.slots - 1) / p.bwd.slots;
  int64_t splits = bmost / groups;
  if (splits < 1) splits = 1;
  if (splits > gneed) splits = gneed;
  p.splits = static_cast<int>(splits);
  const int64_t gb = groups < bmost ? groups : bmost;
  p.bblocks = gb * splits;
  p.gpart = p.shared && splits > 1;
  return p;
}

// f(type, vector length, threads to a row): the instance of a call with V channels a thread. vec:
// whole pieces (16 bytes, or the 8 of 4 channels in 16 bits), else channel by channel.
template <int V, typename F>
int gnorm_dispatch(int dtype, bool vec, int tpr, F&& f) {
  using std::integral_constant;
  auto with = [&](auto t, auto w) {
    if (tpr > 512) return f(t, w, integral_constant<int, 1024>());
    if (tpr > 256) return f(t, w, integral_constant<int, 512>());
    if (tpr > 128) return f(t, w, integral_constant<int, 256>());
    if (tpr > 64) return f(t, w, integral_constant<int, 128>());
    if (tpr > 32) return f(t, w, integral_constant<int, 64>());
    if constexpr (decltype(w)::value > 1) {
      if (tpr == 8) return f(t, w, integral_constant<int, 8>());
      if (tpr == 16) return f(t, w, integral_constant<int, 16>());
      return f(t, w, integral_constant<int, 32>());
    } else {
      return f(t, w, integral_constant<int, 0>());
    }
  };
  return by_io_type(dtype, [&](auto t) {
    constexpr int VEC = sizeof(t) == 2 ? V : 4;
    return vec ? with(t, integral_constant<int, VEC>()) : with(t, integral_constant<int, 1>());
  });
}

// whether rows of C channels, `stride` apart, can be read in pieces of `vec` channels
inline bool gn_pieces(const void* p, int64_t stride, int vec, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (vec * bytes) == 0 && stride % vec == 0);
}

constexpr int kGnMostC = 8192;
inline bool gn_stride(int64_t s) { return s > -(int64_t(1) << 31) && s < (int64_t(1) << 31); }

}  // namespace tops

using namespace tops;

extern "C" int tops_gated_norm_forward(int dtype, int w_dtype, int64_t rows, int64_t groups, int64_t C, int layer,
                                       int has_post, int has_pre, float eps, const void* x, int64_t xs, const void* y,
                                       int64_t ys, const void* gate, int64_t gs, const void* post_w,
                                       const void* post_b, const void* res_s, const void* pre_w, const void* pre_b,
                                       void* h, void* n, float* stats, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (w_dtype != dtype && w_dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (rows < 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0 || rows >= (int64_t(1) << 30))
    return TOPS_ERR_SHAPE;
  if (rows == 0) return TOPS_OK;
  if (x == nullptr || y == nullptr || h == nullptr || (has_pre && n == nullptr)) return TOPS_ERR_ARG;
  if (stats != nullptr && !aligned16(stats)) return TOPS_ERR_ALIGN;
  if (!gn_stride(xs) || !gn_stride(ys) || !gn_stride(gs)) return TOPS_ERR_SHAPE;
  const GnormPlan p = gnorm_plan(rows, groups, C);
  GnormArgs a = {};
  a.rows = rows, a.groups = p.groups, a.group_rows = rows / p.groups, a.C = static_cast<int>(C);
  a.shared = gate != nullptr && p.shared;
  a.layer = layer, a.has_post = has_post, a.has_pre = has_pre, a.w_io = w_dtype == dtype, a.eps = eps;
  a.x = x, a.xs = static_cast<int>(xs), a.y = y, a.ys = static_cast<int>(ys), a.gate = gate, a.gs = static_cast<int>(gs);
  a.post_w = post_w, a.post_b = post_b, a.res_s = res_s, a.pre_w = pre_w, a.pre_b = pre_b;
  a.h = h, a.n = n, a.stats = stats, a.tpr = p.fwd.tpr;
  const int vec = dtype == TOPS_F32 ? 4 : 8, bytes = dtype == TOPS_F32 ? 4 : 2;
  auto fits = [&](const void* q, int64_t stride) { return gn_pieces(q, stride, vec, bytes); };
  const bool whole = fits(x, xs) && fits(y, ys) && fits(gate, gs) && fits(h, C) && fits(n, C);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return gnorm_dispatch<8>(dtype, whole, p.fwd.tpr, [&](auto t, auto w, auto tpr) {
    constexpr int VEC = decltype(w)::value, TPR = decltype(tpr)::value;
    const int64_t fit = VEC == 1 && p.fwd.threads == 128 ? int64_t(4) * sm_count() : p.blocks;
    const unsigned grid = static_cast<unsigned>(p.blocks < fit ? p.blocks : fit);
    if (has_post && has_pre && gate != nullptr)
      gnorm_forward_kernel<decltype(t), VEC, TPR, true><<<grid, p.fwd.threads, 0, st>>>(a);
    else
      gnorm_forward_kernel<decltype(t), VEC, TPR, false><<<grid, p.fwd.threads, 0, st>>>(a);
    return launch_status();
  });
}

extern "C" int tops_gated_norm_backward_workspace_bytes(int64_t rows, int64_t groups, int64_t C, int64_t* bytes) {
  if (bytes == nullptr) return TOPS_ERR_ARG;
  if (rows < 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0 || rows >= (int64_t(1) << 30))
    return TOPS_ERR_SHAPE;
  const GnormPlan p = gnorm_plan(rows, groups, C);
  *bytes = (p.bblocks * 5 + (p.gpart ? groups * p.splits : 0)) * C * 4;
  return TOPS_OK;
}

extern "C" int tops_gated_norm_backward(int dtype, int w_dtype, int64_t rows, int64_t groups, int64_t C, int layer,
                                        int has_post, int has_pre, const void* dh, int64_t dhs, const void* dn,
                                        int64_t dns, const void* x, int64_t xs, const void* y, int64_t ys,
                                        const void* gate, int64_t gs, const float* stats, const void* post_w,
                                        const void* post_b, const void* res_s, const void* pre_w, void* dx, void* dy,
                                        void* dgate, void* dpost_w, void* dpost_b, void* dres_s, void* dpre_w,
                                        void* dpre_b, void* workspace, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (w_dtype != dtype && w_dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (rows < 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0 || rows >= (int64_t(1) << 30))
    return TOPS_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // sums of nothing
    const size_t w_bytes = C * (w_dtype == TOPS_F32 ? 4 : 2), g_bytes = groups * C * (dtype == TOPS_F32 ? 4 : 2);
    bool ok = dgate == nullptr || cudaMemsetAsync(dgate, 0, g_bytes, st) == cudaSuccess;
    for (void* w : {dpost_w, dpost_b, dres_s, dpre_w, dpre_b})
      ok = ok && (w == nullptr || cudaMemsetAsync(w, 0, w_bytes, st) == cudaSuccess);
    return ok ? TOPS_OK : TOPS_ERR_CUDA;
  }
  if (x == nullptr || y == nullptr || stats == nullptr || dx == nullptr || dy == nullptr || workspace == nullptr ||
      (gate != nullptr && dgate == nullptr))
    return TOPS_ERR_ARG;
  if (!aligned16(stats) || !aligned16(workspace)) return TOPS_ERR_ALIGN;
  if (!gn_stride(xs) || !gn_stride(ys) || !gn_stride(gs) || !gn_stride(dhs) || !gn_stride(dns)) return TOPS_ERR_SHAPE;
  const GnormPlan p = gnorm_plan(rows, groups, C);
  GnormArgs a = {};
  a.rows = rows, a.groups = p.groups, a.group_rows = rows / p.groups, a.C = static_cast<int>(C);
  a.shared = gate != nullptr && p.shared;
  a.layer = layer, a.has_post = has_post, a.has_pre = has_pre, a.w_io = w_dtype == dtype;
  a.x = x, a.xs = static_cast<int>(xs), a.y = y, a.ys = static_cast<int>(ys), a.gate = gate, a.gs = static_cast<int>(gs);
  a.dh = dh, a.dhs = static_cast<int>(dhs), a.dn = has_pre ? dn : nullptr, a.dns = static_cast<int>(dns);
  a.post_w = post_w, a.post_b = post_b, a.res_s = res_s, a.pre_w = pre_w;
  a.stats = const_cast<float*>(stats);
  a.dx = dx, a.dy = dy, a.dgate = dgate;
  a.part = static_cast<float*>(workspace);
  a.gpart = p.gpart ? a.part + p.bblocks * 5 * C : nullptr;
  a.splits = p.splits, a.tpr = p.bwd.tpr;
  const int weights = dpost_w || dpost_b || dres_s || dpre_w || dpre_b ? 5 : 0;
  const int64_t sets = weights + (a.gpart != nullptr && gate != nullptr ? groups : 0);
  a.summed = sets > 0;
  const int vec = dtype == TOPS_F32 ? 4 : p.v, bytes = dtype == TOPS_F32 ? 4 : 2;
  auto fits = [&](const void* q, int64_t stride) { return gn_pieces(q, stride, vec, bytes); };
  const bool whole = fits(x, xs) && fits(y, ys) && fits(gate, gs) && fits(dh, dhs) && fits(dn, dns) && fits(dx, C) &&
                     fits(dy, C) && fits(dgate, C);
  const GnormShape& g = p.bwd;
  const size_t smem = (static_cast<size_t>(4 * g.tpr) + (g.slots > 1 ? g.threads : 0)) * p.v * 4;
  auto run = [&](auto t, auto w, auto v, auto tpr) {
    constexpr int VEC = decltype(w)::value, V = decltype(v)::value, TPR = decltype(tpr)::value;
    auto kern = gnorm_backward_kernel<decltype(t), VEC, V, TPR, false>;
    if (has_post && has_pre && gate != nullptr && dh != nullptr && dn != nullptr)
      kern = gnorm_backward_kernel<decltype(t), VEC, V, TPR, true>;
    if (smem > 48 * 1024) set_smem(kern, smem);
    kern<<<static_cast<unsigned>(p.bblocks), g.threads, smem, st>>>(a);
    return launch_status();
  };
  using std::integral_constant;
  int rc = p.v == 4 ? gnorm_dispatch<4>(dtype, whole, g.tpr,
                                        [&](auto t, auto w, auto tpr) { return run(t, w, integral_constant<int, 4>(), tpr); })
                    : by_io_type(dtype, [&](auto t) {  // C > 4096: 1024 threads a row
                        constexpr int VEC = 16 / sizeof(t);
                        constexpr integral_constant<int, 1024> tpr;
                        constexpr integral_constant<int, 8> v;
                        return whole ? run(t, integral_constant<int, VEC>(), v, tpr) : run(t, integral_constant<int, 1>(), v, tpr);
                      });
  if (rc != TOPS_OK) return rc;
  if (sets == 0) return TOPS_OK;
  const GnReduceArgs r = {a.part, a.gpart, p.bblocks, p.splits, a.C, a.w_io, 5 - weights,
                          {dpost_w, dpost_b, dres_s, dpre_w, dpre_b}, dgate};
  return by_io_type(dtype, [&](auto t) {
    launch_pdl(gnorm_reduce_kernel<decltype(t)>,
               dim3(static_cast<unsigned>((C + 31) / 32), static_cast<unsigned>(sets)), 1024, 0, st, r);
    return launch_status();
  });
}
