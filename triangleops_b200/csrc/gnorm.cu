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
  int64_t xs, ys, gs, dhs, dns;  // row strides in elements
  const void *x, *y, *gate, *dh, *dn;
  const void *post_w, *post_b, *res_s, *pre_w, *pre_b;  // null: 1, 0, 1, 1, 0
  void *h, *n;
  float* stats;            // [rows][4]: mean and 1/std of y, mean and 1/std of h
  void *dx, *dy, *dgate;
  float* part;             // [blocks][5][C]: gradients of post_w, post_b, res_s, pre_w, pre_b
  float* gpart;            // [groups][splits][C], or null where a group has one block
  int splits;              // blocks that share a group
  int tpr;                 // threads to a row
};

constexpr int kGnVals = 8;  // channels per thread, held as 4 pairs (packed fp32 arithmetic)

// channel of value i (0..7) of the thread at `t` of a row of tpr threads
template <int VEC>
__device__ __forceinline__ int gn_channel(int t, int tpr, int i) {
  return (t + (i / VEC) * tpr) * VEC + i % VEC;
}

// A thread's 8 channels as they lie in memory: 16-byte pieces of VEC values, or (VEC 1) one by
// one. Channels past C are zero.
template <typename T, int VEC>
struct GnRaw {
  uint4 w[8 / VEC];
  __device__ __forceinline__ void load(const T* p, int t, int tpr, int C) {
#pragma unroll
    for (int k = 0; k < 8 / VEC; ++k) {
      const int c = (t + k * tpr) * VEC;
      w[k] = c < C ? *reinterpret_cast<const uint4*>(p + c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void get(f2* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[2 * k] = f2_pack(__uint_as_float(w[k].x), __uint_as_float(w[k].y));
        f[2 * k + 1] = f2_pack(__uint_as_float(w[k].z), __uint_as_float(w[k].w));
      }
    } else {
      using E = Elem<T>;
      f[0] = f2_pack(E::lo(w[0].x), E::hi(w[0].x));
      f[1] = f2_pack(E::lo(w[0].y), E::hi(w[0].y));
      f[2] = f2_pack(E::lo(w[0].z), E::hi(w[0].z));
      f[3] = f2_pack(E::lo(w[0].w), E::hi(w[0].w));
    }
  }
};
template <typename T>
struct GnRaw<T, 1> {
  T v[8];
  __device__ __forceinline__ void load(const T* p, int t, int tpr, int C) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t + i * tpr < C ? p[t + i * tpr] : T(0.f);
  }
  __device__ __forceinline__ void get(f2* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = f2_pack(static_cast<float>(v[2 * i]), static_cast<float>(v[2 * i + 1]));
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, int t, int tpr, int C, const f2* v) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int k = 0; k < kGnVals / VEC; ++k) {
    const int c = (t + k * tpr) * VEC;
    if (c >= C) continue;
    if constexpr (VEC == 1) {
      p[c] = static_cast<T>(f[k]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + c) = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
    } else {
      using E = Elem<T>;
      *reinterpret_cast<uint4*>(p + c) = make_uint4(E::pack2(f[0], f[1]), E::pack2(f[2], f[3]), E::pack2(f[4], f[5]),
                                                    E::pack2(f[6], f[7]));
    }
  }
}

// A weight row of either dtype, read once a block. Channels past C get 0, whatever the default:
// then nothing of theirs enters a sum.
template <typename T, int VEC>
__device__ __forceinline__ void gn_weight(const void* w, int io, int t, int tpr, int C, float none, f2* f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < kGnVals; ++i) {
    const int c = gn_channel<VEC>(t, tpr, i);
    v[i] = c < C ? none : 0.f;
    if (w != nullptr && c < C)
      v[i] = io ? static_cast<float>(static_cast<const T*>(w)[c]) : static_cast<const float*>(w)[c];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_pack(v[2 * i], v[2 * i + 1]);
}

__device__ __forceinline__ float f2_sum(f2 v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// Sums of N values over the threads of a row. MULTI: the row takes the whole block; `red` is then
// two buffers of N x 32 floats used in turn, so that one barrier a sum is enough.
template <bool MULTI, int N>
__device__ __forceinline__ void row_sum(float* v, int tpr, float* red, int& turn) {
  const int width = MULTI ? 32 : tpr;
  for (int o = width >> 1; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (MULTI) {
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
      for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
}

// 16-bit IO: two ulps of the hardware's exponential and quotient are far below its rounding
template <typename T>
__device__ __forceinline__ float gn_sigmoid(float x) {
  if constexpr (sizeof(T) == 4)
    return 1.f / (1.f + expf(-x));
  else
    return __fdividef(1.f, 1.f + __expf(-x));  // 0 once the divisor passes 2^126
}
template <typename T>
__device__ __forceinline__ f2 gn_sigmoid2(f2 x) {
  float a, b;
  f2_unpack(x, a, b);
  return f2_pack(gn_sigmoid<T>(a), gn_sigmoid<T>(b));
}

// mean and 1/std of a row's values (rms: mean 0)
template <typename T, int VEC, bool MULTI>
__device__ __forceinline__ float2 gn_stats(const f2* f, int t, const GnormArgs& a, float* red, int& turn) {
  const float inv = 1.f / a.C;
  float mean = 0.f, s;
  if (a.layer) {
    s = f2_sum(f2_add(f2_add(f[0], f[1]), f2_add(f[2], f[3])));  // channels past C hold 0
    row_sum<MULTI, 1>(&s, a.tpr, red, turn);
    mean = s * inv;
  }
  f2 acc = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m0 = gn_channel<VEC>(t, a.tpr, 2 * i) < a.C ? mean : 0.f;
    const float m1 = VEC > 1 ? m0 : gn_channel<VEC>(t, a.tpr, 2 * i + 1) < a.C ? mean : 0.f;
    const f2 d = f2_add(f[i], f2_pack(-m0, -m1));
    acc = f2_fma(d, d, acc);
  }
  s = f2_sum(acc);
  row_sum<MULTI, 1>(&s, a.tpr, red, turn);
  s = fmaf(s, inv, a.eps);
  return make_float2(mean, sizeof(T) == 4 ? 1.f / sqrtf(s) : rsqrtf(s));
}

// Threads of a block, at most THREADS: rows side by side, a.tpr threads each, or (more than 128)
// one row. Block b takes rows b * slots + slot, then on by the grid; the next row's values are on
// their way while the present one's are worked on.
template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 128 && VEC > 1 ? 5 : 1) gnorm_forward_kernel(GnormArgs a) {
  constexpr bool MULTI = THREADS > 128;
  __shared__ float red[MULTI ? 128 : 1];
  int turn = 0;
  const int tpr = a.tpr, t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = blockDim.x / tpr, C = a.C;
  f2 pw[4], pb[4], sc[4], nw[4], nb[4];
  gn_weight<T, VEC>(a.post_w, a.w_io, t, tpr, C, 1.f, pw);
  gn_weight<T, VEC>(a.post_b, a.w_io, t, tpr, C, 0.f, pb);
  gn_weight<T, VEC>(a.res_s, a.w_io, t, tpr, C, 1.f, sc);
  gn_weight<T, VEC>(a.pre_w, a.w_io, t, tpr, C, 1.f, nw);
  gn_weight<T, VEC>(a.pre_b, a.w_io, t, tpr, C, 0.f, nb);
  const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
  GnRaw<T, VEC> rx, ry, rg;
  auto load = [&](int64_t r) {
    r = r < a.rows ? r : a.rows - 1;  // a thread without a row keeps up with its warp's shuffles
    rx.load(static_cast<const T*>(a.x) + r * a.xs, t, tpr, C);
    ry.load(static_cast<const T*>(a.y) + r * a.ys, t, tpr, C);
    if (a.gate) rg.load(static_cast<const T*>(a.gate) + (a.shared ? r / a.group_rows : r) * a.gs, t, tpr, C);
  };
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * slots;
  if (r0 < a.rows) load(r0 + slot);
  for (; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + slot;
    const bool live = r < a.rows;
    f2 x[4], y[4], g[4];
    rx.get(x);
    ry.get(y);
    if (a.gate) rg.get(g);
    if (r0 + step < a.rows) load(r + step);
    float2 sy = make_float2(0.f, 1.f), sh = sy;
    if (a.has_post) {
      sy = gn_stats<T, VEC, MULTI>(y, t, a, red, turn);
      const f2 m = f2_both(-sy.x), q = f2_both(sy.y);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = f2_fma(f2_mul(f2_add(y[i], m), q), pw[i], pb[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (a.gate) y[i] = f2_mul(y[i], gn_sigmoid2<T>(g[i]));
      x[i] = f2_fma(sc[i], y[i], x[i]);  // h
    }
    if (live) gn_store<T, VEC>(static_cast<T*>(a.h) + r * C, t, tpr, C, x);
    if (a.has_pre) {
      sh = gn_stats<T, VEC, MULTI>(x, t, a, red, turn);
      const f2 m = f2_both(-sh.x), q = f2_both(sh.y);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = f2_fma(f2_mul(f2_add(x[i], m), q), nw[i], nb[i]);
      if (live) gn_store<T, VEC>(static_cast<T*>(a.n) + r * C, t, tpr, C, x);
    }
    if (live && a.stats && t == 0) reinterpret_cast<float4*>(a.stats)[r] = make_float4(sy.x, sy.y, sh.x, sh.y);
  }
}

// Adds each thread's 8 sums over the block's row slots, in order; slot 0 is left with the total.
__device__ __forceinline__ void slot_sum(f2* f, float* buf, int t, int slot, int slots, int tpr) {
  if (slots == 1) return;
  f2* at = reinterpret_cast<f2*>(buf);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) at[(slot * 4 + i) * tpr + t] = f[i];
  __syncthreads();
  if (slot == 0)
    for (int s = 1; s < slots; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = f2_add(f[i], at[(s * 4 + i) * tpr + t]);
}

template <int VEC>
__device__ __forceinline__ void gn_part(float* p, const f2* v, int t, int tpr, int C) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
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
// wait in shared memory (a thread's 20 pairs of sums take the registers).
template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 128 && VEC > 1 ? 4 : 1) gnorm_backward_kernel(GnormArgs a) {
  constexpr bool MULTI = THREADS > 128;
  __shared__ float red[MULTI ? 128 : 1];
  extern __shared__ float buf[];  // weights [4][4][tpr] pairs, then the row slots' sums
  int turn = 0;
  const int tpr = a.tpr, t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = blockDim.x / tpr, C = a.C;
  const float inv = 1.f / C;
  f2* wts = reinterpret_cast<f2*>(buf);
  if (slot == 0) {
    f2 w[4];
    const void* const from[4] = {a.post_w, a.post_b, a.res_s, a.pre_w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      gn_weight<T, VEC>(from[k], a.w_io, t, tpr, C, k == 1 ? 0.f : 1.f, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) wts[(k * 4 + i) * tpr + t] = w[i];
    }
  }
  __syncthreads();
  auto weight = [&](int k, int i) { return wts[(k * 4 + i) * tpr + t]; };
  float* sums = buf + 32 * tpr;
  f2 apw[4] = {}, apb[4] = {}, asc[4] = {}, anw[4] = {}, anb[4] = {};
  const int share = blockIdx.x % a.splits;
  const int64_t step = static_cast<int64_t>(a.splits) * slots;
  for (int64_t grp = blockIdx.x / a.splits; grp < a.groups; grp += gridDim.x / a.splits) {
    f2 ag[4] = {};
    const int64_t end = (grp + 1) * a.group_rows;
    GnRaw<T, VEC> rx, ry, rg, rh, rn;
    float4 st_next;
    auto load = [&](int64_t r) {
      r = r < end ? r : end - 1;
      rx.load(static_cast<const T*>(a.x) + r * a.xs, t, tpr, C);
      ry.load(static_cast<const T*>(a.y) + r * a.ys, t, tpr, C);
      if (a.gate) rg.load(static_cast<const T*>(a.gate) + (a.shared ? grp : r) * a.gs, t, tpr, C);
      if (a.dh) rh.load(static_cast<const T*>(a.dh) + r * a.dhs, t, tpr, C);
      if (a.dn) rn.load(static_cast<const T*>(a.dn) + r * a.dns, t, tpr, C);
      st_next = reinterpret_cast<const float4*>(a.stats)[r];
    };
    int64_t r0 = grp * a.group_rows + share * slots;
    if (r0 < end) load(r0 + slot);
    for (; r0 < end; r0 += step) {
      const int64_t r = r0 + slot;
      const bool live = r < end;  // without a row: zero gradients, which add nothing to a sum
      f2 x[4], y[4], g[4], dh[4] = {}, dn[4] = {};
      rx.get(x);
      ry.get(y);
      if (a.gate) rg.get(g);
      if (a.dh && live) rh.get(dh);
      if (a.dn && live) rn.get(dn);
      const float4 st = st_next;
      if (r0 + step < end) load(r + step);
      float s[2];
      f2 s1 = 0, s2 = 0;
      // y: normalised y; g: its sigmoid; x: normalised h; dn: d n * pre weight
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (a.has_post) y[i] = f2_mul(f2_add(y[i], f2_both(-st.x)), f2_both(st.y));
        if (a.gate) g[i] = gn_sigmoid2<T>(g[i]);
        if (a.has_pre) {
          f2 u = a.has_post ? f2_fma(y[i], weight(0, i), weight(1, i)) : y[i];
          if (a.gate) u = f2_mul(u, g[i]);
          x[i] = f2_mul(f2_add(f2_fma(weight(2, i), u, x[i]), f2_both(-st.z)), f2_both(st.w));
          anw[i] = f2_fma(dn[i], x[i], anw[i]);
          anb[i] = f2_add(dn[i], anb[i]);
          dn[i] = f2_mul(dn[i], weight(3, i));
          s1 = f2_fma(dn[i], x[i], s1);
          s2 = f2_add(dn[i], s2);
        }
      }
      if (a.has_pre) {
        s[0] = f2_sum(s1), s[1] = f2_sum(s2);
        row_sum<MULTI, 2>(s, tpr, red, turn);
        const f2 m1 = f2_both(-s[0] * inv), m2 = f2_both(a.layer ? -s[1] * inv : 0.f), q = f2_both(st.w);
#pragma unroll
        for (int i = 0; i < 4; ++i) dh[i] = f2_fma(q, f2_add(f2_fma(x[i], m1, dn[i]), m2), dh[i]);
      }
      if (live) gn_store<T, VEC>(static_cast<T*>(a.dx) + r * C, t, tpr, C, dh);
      s1 = s2 = 0;
      // dh: d y^; dn: d gate
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f2 u = a.has_post ? f2_fma(y[i], weight(0, i), weight(1, i)) : y[i];
        f2 dr = dh[i];
        if (a.gate) {
          const f2 ug = f2_mul(u, g[i]);
          asc[i] = f2_fma(dr, ug, asc[i]);
          dr = f2_mul(dr, weight(2, i));
          // u sg (1 - sg)
          dn[i] = f2_mul(dr, f2_fma(f2_mul(ug, g[i]), f2_both(-1.f), ug));
          ag[i] = f2_add(dn[i], ag[i]);
          dr = f2_mul(dr, g[i]);
        } else {
          asc[i] = f2_fma(dr, u, asc[i]);
          dr = f2_mul(dr, weight(2, i));
        }
        if (a.has_post) {
          apw[i] = f2_fma(dr, y[i], apw[i]);
          apb[i] = f2_add(dr, apb[i]);
          dr = f2_mul(dr, weight(0, i));
          s1 = f2_fma(dr, y[i], s1);
          s2 = f2_add(dr, s2);
        }
        dh[i] = dr;
      }
      if (live && a.gate && !a.shared) gn_store<T, VEC>(static_cast<T*>(a.dgate) + r * C, t, tpr, C, dn);
      if (a.has_post) {
        s[0] = f2_sum(s1), s[1] = f2_sum(s2);
        row_sum<MULTI, 2>(s, tpr, red, turn);
        const f2 m1 = f2_both(-s[0] * inv), m2 = f2_both(a.layer ? -s[1] * inv : 0.f), q = f2_both(st.y);
#pragma unroll
        for (int i = 0; i < 4; ++i) dh[i] = f2_mul(q, f2_add(f2_fma(y[i], m1, dh[i]), m2));
      }
      if (live) gn_store<T, VEC>(static_cast<T*>(a.dy) + r * C, t, tpr, C, dh);
    }
    if (a.shared) {
      slot_sum(ag, sums, t, slot, slots, tpr);
      if (slot == 0) {
        if (a.gpart)
          gn_part<VEC>(a.gpart + (grp * a.splits + share) * C, ag, t, tpr, C);
        else
          gn_store<T, VEC>(static_cast<T*>(a.dgate) + grp * C, t, tpr, C, ag);
      }
    }
  }
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 5 * C;
  auto leave = [&](f2* v, int k) {
    slot_sum(v, sums, t, slot, slots, tpr);
    if (slot == 0) gn_part<VEC>(part + k * C, v, t, tpr, C);
  };
  leave(apw, 0);
  leave(apb, 1);
  leave(asc, 2);
  leave(anw, 3);
  leave(anb, 4);
}

// out[set][c] = sum over n of in[(set_base + n * set_step) ...]: the blocks' partial rows, added
// in a fixed order. One block takes 32 channels of one set; its 8 warps share the rows.
struct GnReduceArgs {
  const float* in;
  int64_t n, row_step, set_step;  // rows to add, distance between them and between sets, in elements
  int C;
  void* out[5];                   // a row per set (null: not wanted), or
  void* rows;                     // all sets' rows one after the other
  int sets, io;
};
template <typename T>
__global__ void __launch_bounds__(256) gnorm_reduce_kernel(GnReduceArgs a) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t set = blockIdx.y;
  void* out = a.rows ? a.rows : a.out[set];
  if (out == nullptr) return;
  float v = 0.f;
  if (c < a.C)
    for (int64_t i = warp; i < a.n; i += 8) v += a.in[set * a.set_step + i * a.row_step + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || c >= a.C) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) v += s[w][lane];
  const int64_t at = a.rows ? set * a.C + c : c;
  if (a.io)
    static_cast<T*>(out)[at] = static_cast<T>(v);
  else
    static_cast<float*>(out)[at] = v;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct GnormPlan {
  int tpr, threads, slots;
  int64_t blocks;     // forward
  int64_t bblocks;    // backward
  int splits;
  bool shared, gpart;
  int64_t groups;
};

inline GnormPlan gnorm_plan(int64_t rows, int64_t gate_rows, int64_t C) {
  GnormPlan p;
  p.shared = gate_rows < rows;
  const int64_t groups = p.groups = p.shared ? gate_rows : 1;
  p.tpr = 8;
  while (p.tpr * kGnVals < C) p.tpr *= 2;
  p.threads = p.tpr <= 32 ? 128 : p.tpr;
  p.slots = p.threads / p.tpr;
  const int64_t sms = sm_count();
  const int64_t most = sms * (p.threads <= 128 ? 5 : p.threads <= 256 ? 3 : 2);
  const int64_t need = (rows + p.slots - 1) / p.slots;
  p.blocks = need < most ? need : most;
  const int64_t bmost = sms * (p.threads <= 128 ? 4 : p.threads <= 256 ? 2 : 1);
  const int64_t per = rows / groups;
  const int64_t gneed = (per + p.slots - 1) / p.slots;
  int64_t splits = bmost / groups;
  if (splits < 1) splits = 1;
  if (splits > gneed) splits = gneed;
  p.splits = static_cast<int>(splits);
  const int64_t gb = groups < bmost ? groups : bmost;
  p.bblocks = gb * splits;
  p.gpart = p.shared && splits > 1;
  return p;
}

template <typename F>
int gnorm_dispatch(int dtype, bool vec, int tpr, F&& f) {
  auto with = [&](auto t, auto v) {
    if (tpr <= 32) return f(t, v, std::integral_constant<int, 128>());
    if (tpr <= 512) return f(t, v, std::integral_constant<int, 512>());
    return f(t, v, std::integral_constant<int, 1024>());
  };
  auto typed = [&](auto t) {
    constexpr int VEC = 16 / sizeof(t);
    return vec ? with(t, std::integral_constant<int, VEC>()) : with(t, std::integral_constant<int, 1>());
  };
  if (dtype == TOPS_BF16) return typed(__nv_bfloat16());
  if (dtype == TOPS_F16) return typed(__half());
  return typed(float());
}

constexpr int kGnMostC = 8192;

}  // namespace tops

using namespace tops;

extern "C" int tops_gated_norm_forward(int dtype, int w_dtype, int64_t rows, int64_t groups, int64_t C, int layer,
                                       int has_post, int has_pre, float eps, const void* x, int64_t xs, const void* y,
                                       int64_t ys, const void* gate, int64_t gs, const void* post_w,
                                       const void* post_b, const void* res_s, const void* pre_w, const void* pre_b,
                                       void* h, void* n, float* stats, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (w_dtype != dtype && w_dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (rows < 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0) return TOPS_ERR_SHAPE;
  if (rows == 0) return TOPS_OK;
  if (x == nullptr || y == nullptr || h == nullptr || (has_pre && n == nullptr)) return TOPS_ERR_ARG;
  if (stats != nullptr && !aligned16(stats)) return TOPS_ERR_ALIGN;
  const GnormPlan p = gnorm_plan(rows, groups, C);
  GnormArgs a = {};
  a.rows = rows, a.groups = p.groups, a.group_rows = rows / p.groups, a.C = static_cast<int>(C);
  a.shared = gate != nullptr && p.shared;
  a.layer = layer, a.has_post = has_post, a.has_pre = has_pre, a.w_io = w_dtype == dtype, a.eps = eps;
  a.x = x, a.xs = xs, a.y = y, a.ys = ys, a.gate = gate, a.gs = gs;
  a.post_w = post_w, a.post_b = post_b, a.res_s = res_s, a.pre_w = pre_w, a.pre_b = pre_b;
  a.h = h, a.n = n, a.stats = stats, a.tpr = p.tpr;
  const int vec = dtype == TOPS_F32 ? 4 : 8;
  const bool fits = C % vec == 0 && xs % vec == 0 && ys % vec == 0 && (gate == nullptr || gs % vec == 0) &&
                    aligned16(x) && aligned16(y) && aligned16(gate) && aligned16(h) && aligned16(n);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return gnorm_dispatch(dtype, fits, p.tpr, [&](auto t, auto v, auto m) {
    gnorm_forward_kernel<decltype(t), decltype(v)::value, decltype(m)::value>
        <<<static_cast<unsigned>(p.blocks), p.threads, 0, st>>>(a);
    return launch_status();
  });
}

extern "C" int tops_gated_norm_backward_workspace_bytes(int64_t rows, int64_t groups, int64_t C, int64_t* bytes) {
  if (bytes == nullptr) return TOPS_ERR_ARG;
  if (rows < 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0) return TOPS_ERR_SHAPE;
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
  if (rows <= 0 || C <= 0 || C > kGnMostC || groups <= 0 || rows % groups != 0) return TOPS_ERR_SHAPE;
  if (x == nullptr || y == nullptr || stats == nullptr || dx == nullptr || dy == nullptr || workspace == nullptr ||
      (gate != nullptr && dgate == nullptr))
    return TOPS_ERR_ARG;
  if (!aligned16(stats) || !aligned16(workspace)) return TOPS_ERR_ALIGN;
  const GnormPlan p = gnorm_plan(rows, groups, C);
  GnormArgs a = {};
  a.rows = rows, a.groups = p.groups, a.group_rows = rows / p.groups, a.C = static_cast<int>(C);
  a.shared = gate != nullptr && p.shared;
  a.layer = layer, a.has_post = has_post, a.has_pre = has_pre, a.w_io = w_dtype == dtype;
  a.x = x, a.xs = xs, a.y = y, a.ys = ys, a.gate = gate, a.gs = gs;
  a.dh = dh, a.dhs = dhs, a.dn = has_pre ? dn : nullptr, a.dns = dns;
  a.post_w = post_w, a.post_b = post_b, a.res_s = res_s, a.pre_w = pre_w;
  a.stats = const_cast<float*>(stats);
  a.dx = dx, a.dy = dy, a.dgate = dgate;
  a.part = static_cast<float*>(workspace);
  a.gpart = p.gpart ? a.part + p.bblocks * 5 * C : nullptr;
  a.splits = p.splits, a.tpr = p.tpr;
  const int vec = dtype == TOPS_F32 ? 4 : 8;
  const bool fits = C % vec == 0 && xs % vec == 0 && ys % vec == 0 && (gate == nullptr || gs % vec == 0) &&
                    (dh == nullptr || dhs % vec == 0) && (dn == nullptr || dns % vec == 0) && aligned16(x) &&
                    aligned16(y) && aligned16(gate) && aligned16(dh) && aligned16(dn) && aligned16(dx) &&
                    aligned16(dy) && aligned16(dgate);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = static_cast<size_t>(p.tpr) * 128 + (p.slots > 1 ? static_cast<size_t>(p.threads) * kGnVals * 4 : 0);
  int rc = gnorm_dispatch(dtype, fits, p.tpr, [&](auto t, auto v, auto m) {
    auto kern = gnorm_backward_kernel<decltype(t), decltype(v)::value, decltype(m)::value>;
    if (smem > 48 * 1024) set_smem(kern, smem);
    kern<<<static_cast<unsigned>(p.bblocks), p.threads, smem, st>>>(a);
    return launch_status();
  });
  if (rc != TOPS_OK) return rc;
  auto reduce = [&](const GnReduceArgs& r) {
    return gnorm_dispatch(dtype, false, 8, [&](auto t, auto, auto) {
      gnorm_reduce_kernel<decltype(t)>
          <<<dim3(static_cast<unsigned>((C + 31) / 32), static_cast<unsigned>(r.sets)), 256, 0, st>>>(r);
      return launch_status();
    });
  };
  if (dpost_w || dpost_b || dres_s || dpre_w || dpre_b) {
    const GnReduceArgs r = {a.part, p.bblocks, 5 * C, C, a.C, {dpost_w, dpost_b, dres_s, dpre_w, dpre_b}, nullptr, 5,
                            a.w_io};
    if ((rc = reduce(r)) != TOPS_OK) return rc;
  }
  if (p.gpart && gate != nullptr) {
    const GnReduceArgs r = {a.gpart, p.splits, C, p.splits * C, a.C, {}, dgate, static_cast<int>(groups), 1};
    return reduce(r);
  }
  return TOPS_OK;
}
