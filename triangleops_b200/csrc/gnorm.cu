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

constexpr int kGnVals = 8;  // channels per thread

template <typename T, int VEC>
struct Pack;  // VEC values of T as they lie in memory
template <typename T>
struct Pack<T, 8> {
  using type = uint4;
};
template <>
struct Pack<float, 4> {
  using type = float4;
};

// channel of value i (0..7) of the thread at `t` of a row of tpr threads
template <int VEC>
__device__ __forceinline__ int gn_channel(int t, int tpr, int i) {
  return (t + (i / VEC) * tpr) * VEC + i % VEC;
}

template <typename T, int VEC>
__device__ __forceinline__ void gn_load(const T* p, int t, int tpr, int C, float* f) {
#pragma unroll
  for (int k = 0; k < kGnVals / VEC; ++k) {
    const int c = (t + k * tpr) * VEC;
    if constexpr (VEC == 1) {
      f[k] = c < C ? static_cast<float>(p[c]) : 0.f;
    } else {
      typename Pack<T, VEC>::type w{};
      if (c < C) w = *reinterpret_cast<const typename Pack<T, VEC>::type*>(p + c);
      if constexpr (sizeof(T) == 4) {
        f[4 * k] = w.x, f[4 * k + 1] = w.y, f[4 * k + 2] = w.z, f[4 * k + 3] = w.w;
      } else {
        using E = Elem<T>;
        f[0] = E::lo(w.x), f[1] = E::hi(w.x), f[2] = E::lo(w.y), f[3] = E::hi(w.y);
        f[4] = E::lo(w.z), f[5] = E::hi(w.z), f[6] = E::lo(w.w), f[7] = E::hi(w.w);
      }
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, int t, int tpr, int C, const float* f) {
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

// a weight row of either dtype (read once a block)
template <typename T, int VEC>
__device__ __forceinline__ void gn_weight(const void* w, int io, int t, int tpr, int C, float none, float* f) {
#pragma unroll
  for (int i = 0; i < kGnVals; ++i) {
    const int c = gn_channel<VEC>(t, tpr, i);
    f[i] = none;
    if (w != nullptr && c < C)
      f[i] = io ? static_cast<float>(static_cast<const T*>(w)[c]) : static_cast<const float*>(w)[c];
  }
}

// Sums of two values over the threads of a row. MULTI: the row takes the whole block; `red` is
// then two buffers of 2 x 32 floats used in turn, so that one barrier a sum is enough.
template <bool MULTI>
__device__ __forceinline__ float2 row_sum(float a, float b, int tpr, float* red, int& turn) {
  const int width = MULTI ? 32 : tpr;
  for (int o = width >> 1; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (MULTI) {
    float* r = red + (turn ^= 1) * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0) {
      r[warp] = a;
      r[32 + warp] = b;
    }
    __syncthreads();
    a = lane < nw ? r[lane] : 0.f;
    b = lane < nw ? r[32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
  return make_float2(a, b);
}

// 16-bit IO: two ulps of the hardware's exponential and quotient are far below its rounding
template <typename T>
__device__ __forceinline__ float gn_sigmoid(float x) {
  if constexpr (sizeof(T) == 4)
    return 1.f / (1.f + expf(-x));
  else
    return __fdividef(1.f, 1.f + __expf(-x));  // 0 once the divisor passes 2^126
}
// 1/sqrt, to the last bit but one where the IO shows it
template <typename T>
__device__ __forceinline__ float gn_rsqrt(float x) {
  return sizeof(T) == 4 ? 1.f / sqrtf(x) : rsqrtf(x);
}

// mean and 1/std of a row's values (rms: mean 0)
template <typename T, int VEC, bool MULTI>
__device__ __forceinline__ float2 gn_stats(const float* f, int t, const GnormArgs& a, float* red, int& turn) {
  const float inv = 1.f / a.C;
  float mean = 0.f, s = 0.f;
  if (a.layer) {
#pragma unroll
    for (int i = 0; i < kGnVals; ++i) s += f[i];  // channels past C hold 0
    mean = row_sum<MULTI>(s, 0.f, a.tpr, red, turn).x * inv;
  }
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kGnVals; ++i) {
    const float d = gn_channel<VEC>(t, a.tpr, i) < a.C ? f[i] - mean : 0.f;
    s = fmaf(d, d, s);
  }
  return make_float2(mean, gn_rsqrt<T>(row_sum<MULTI>(s, 0.f, a.tpr, red, turn).x * inv + a.eps));
}

// Threads of a block, at most THREADS: rows side by side, a.tpr threads each, or (more than 128)
// one row. Block b takes rows
// b * slots + slot, then on by the grid.
template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) gnorm_forward_kernel(GnormArgs a) {
  constexpr bool MULTI = THREADS > 128;
  __shared__ float red[MULTI ? 128 : 1];
  int turn = 0;
  const int tpr = a.tpr, t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = blockDim.x / tpr, C = a.C;
  float pw[kGnVals], pb[kGnVals], sc[kGnVals], nw[kGnVals], nb[kGnVals];
  gn_weight<T, VEC>(a.post_w, a.w_io, t, tpr, C, 1.f, pw);
  gn_weight<T, VEC>(a.post_b, a.w_io, t, tpr, C, 0.f, pb);
  gn_weight<T, VEC>(a.res_s, a.w_io, t, tpr, C, 1.f, sc);
  gn_weight<T, VEC>(a.pre_w, a.w_io, t, tpr, C, 1.f, nw);
  gn_weight<T, VEC>(a.pre_b, a.w_io, t, tpr, C, 0.f, nb);
  const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * slots; r0 < a.rows; r0 += step) {
    const bool live = r0 + slot < a.rows;  // the others keep up with the warp's shuffles
    const int64_t r = live ? r0 + slot : a.rows - 1;
    float x[kGnVals], y[kGnVals], g[kGnVals];
    gn_load<T, VEC>(static_cast<const T*>(a.x) + r * a.xs, t, tpr, C, x);
    gn_load<T, VEC>(static_cast<const T*>(a.y) + r * a.ys, t, tpr, C, y);
    if (a.gate) gn_load<T, VEC>(static_cast<const T*>(a.gate) + (a.shared ? r / a.group_rows : r) * a.gs, t, tpr, C, g);
    float2 sy = make_float2(0.f, 1.f), sh = sy;
    if (a.has_post) sy = gn_stats<T, VEC, MULTI>(y, t, a, red, turn);
#pragma unroll
    for (int i = 0; i < kGnVals; ++i) {
      float u = a.has_post ? fmaf((y[i] - sy.x) * sy.y, pw[i], pb[i]) : y[i];
      if (a.gate) u *= gn_sigmoid<T>(g[i]);
      x[i] = gn_channel<VEC>(t, tpr, i) < C ? fmaf(sc[i], u, x[i]) : 0.f;  // h
    }
    if (live) gn_store<T, VEC>(static_cast<T*>(a.h) + r * C, t, tpr, C, x);
    if (a.has_pre) {
      sh = gn_stats<T, VEC, MULTI>(x, t, a, red, turn);
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) x[i] = fmaf((x[i] - sh.x) * sh.y, nw[i], nb[i]);
      if (live) gn_store<T, VEC>(static_cast<T*>(a.n) + r * C, t, tpr, C, x);
    }
    if (live && a.stats && t == 0) reinterpret_cast<float4*>(a.stats)[r] = make_float4(sy.x, sy.y, sh.x, sh.y);
  }
}

// Adds each thread's 8 sums over the block's row slots; slot 0 is left with the total.
template <int VEC>
__device__ __forceinline__ void slot_sum(float* f, float* buf, int t, int slot, int slots, int tpr) {
  if (slots == 1) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGnVals; ++i) buf[(slot * kGnVals + i) * tpr + t] = f[i];
  __syncthreads();
  if (slot == 0)
    for (int s = 1; s < slots; ++s)
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) f[i] += buf[(s * kGnVals + i) * tpr + t];
}

// Block b takes group b / splits, share b % splits of its rows, then on by the grid.
template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) gnorm_backward_kernel(GnormArgs a) {
  constexpr bool MULTI = THREADS > 128;
  __shared__ float red[MULTI ? 128 : 1];
  extern __shared__ float buf[];
  int turn = 0;
  const int tpr = a.tpr, t = threadIdx.x % tpr, slot = threadIdx.x / tpr, slots = blockDim.x / tpr, C = a.C;
  const float inv = 1.f / C;
  float pw[kGnVals], pb[kGnVals], sc[kGnVals], nw[kGnVals];
  gn_weight<T, VEC>(a.post_w, a.w_io, t, tpr, C, 1.f, pw);
  gn_weight<T, VEC>(a.post_b, a.w_io, t, tpr, C, 0.f, pb);
  gn_weight<T, VEC>(a.res_s, a.w_io, t, tpr, C, 1.f, sc);
  gn_weight<T, VEC>(a.pre_w, a.w_io, t, tpr, C, 1.f, nw);
  float apw[kGnVals] = {}, apb[kGnVals] = {}, asc[kGnVals] = {}, anw[kGnVals] = {}, anb[kGnVals] = {};
  const int share = blockIdx.x % a.splits;
  for (int64_t grp = blockIdx.x / a.splits; grp < a.groups; grp += gridDim.x / a.splits) {
    float ag[kGnVals] = {};
    const int64_t end = (grp + 1) * a.group_rows;
    const int64_t step = static_cast<int64_t>(a.splits) * slots;
    for (int64_t r0 = grp * a.group_rows + share * slots; r0 < end; r0 += step) {
      const bool live = r0 + slot < end;
      const int64_t r = live ? r0 + slot : end - 1;
      float x[kGnVals], y[kGnVals], g[kGnVals], dh[kGnVals], dn[kGnVals];
      gn_load<T, VEC>(static_cast<const T*>(a.x) + r * a.xs, t, tpr, C, x);
      gn_load<T, VEC>(static_cast<const T*>(a.y) + r * a.ys, t, tpr, C, y);
      if (a.gate) gn_load<T, VEC>(static_cast<const T*>(a.gate) + (a.shared ? grp : r) * a.gs, t, tpr, C, g);
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) dh[i] = dn[i] = 0.f;
      if (a.dh) gn_load<T, VEC>(static_cast<const T*>(a.dh) + r * a.dhs, t, tpr, C, dh);
      if (a.dn) gn_load<T, VEC>(static_cast<const T*>(a.dn) + r * a.dns, t, tpr, C, dn);
      const float4 st = reinterpret_cast<const float4*>(a.stats)[r];
      const float keep = live ? 1.f : 0.f;
      float s1 = 0.f, s2 = 0.f;
      // y: normalised y; g: sigmoid; x: normalised h; dn: d n * pre weight
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) {
        const bool in = gn_channel<VEC>(t, tpr, i) < C;
        if (a.has_post) y[i] = in ? (y[i] - st.x) * st.y : 0.f;
        g[i] = a.gate ? gn_sigmoid<T>(g[i]) : 1.f;
        if (a.has_pre) {
          const float u = a.has_post ? fmaf(y[i], pw[i], pb[i]) : y[i];
          const float h = fmaf(sc[i], u * g[i], x[i]);
          x[i] = in ? (h - st.z) * st.w : 0.f;
          anw[i] = fmaf(keep * dn[i], x[i], anw[i]);
          anb[i] = fmaf(keep, dn[i], anb[i]);
          dn[i] *= nw[i];
          s1 = fmaf(dn[i], x[i], s1);
          s2 += dn[i];
        }
      }
      if (a.has_pre) {
        const float2 s = row_sum<MULTI>(s1, s2, tpr, red, turn);
        const float m1 = s.x * inv, m2 = a.layer ? s.y * inv : 0.f;
#pragma unroll
        for (int i = 0; i < kGnVals; ++i) dh[i] = fmaf(st.w, dn[i] - x[i] * m1 - m2, dh[i]);
      }
      if (live) gn_store<T, VEC>(static_cast<T*>(a.dx) + r * C, t, tpr, C, dh);
      s1 = s2 = 0.f;
      // dh: d y^ ; dn: d gate
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) {
        const float u = a.has_post ? fmaf(y[i], pw[i], pb[i]) : y[i];
        asc[i] = fmaf(keep * dh[i], u * g[i], asc[i]);
        const float dr = dh[i] * sc[i];
        dn[i] = dr * u * g[i] * (1.f - g[i]);
        ag[i] = fmaf(keep, dn[i], ag[i]);
        const float du = dr * g[i];
        if (a.has_post) {
          apw[i] = fmaf(keep * du, y[i], apw[i]);
          apb[i] = fmaf(keep, du, apb[i]);
        }
        dh[i] = a.has_post ? du * pw[i] : du;
        if (gn_channel<VEC>(t, tpr, i) >= C) dh[i] = 0.f;
        s1 = fmaf(dh[i], y[i], s1);
        s2 += dh[i];
      }
      if (live && a.gate && !a.shared) gn_store<T, VEC>(static_cast<T*>(a.dgate) + r * C, t, tpr, C, dn);
      if (a.has_post) {
        const float2 s = row_sum<MULTI>(s1, s2, tpr, red, turn);
        const float m1 = s.x * inv, m2 = a.layer ? s.y * inv : 0.f;
#pragma unroll
        for (int i = 0; i < kGnVals; ++i) dh[i] = st.y * (dh[i] - y[i] * m1 - m2);
      }
      if (live) gn_store<T, VEC>(static_cast<T*>(a.dy) + r * C, t, tpr, C, dh);
    }
    if (a.shared) {
      slot_sum<VEC>(ag, buf, t, slot, slots, tpr);
      if (slot == 0) {
        if (a.gpart) {
          float* p = a.gpart + (grp * a.splits + share) * C;
#pragma unroll
          for (int i = 0; i < kGnVals; ++i) {
            const int c = gn_channel<VEC>(t, tpr, i);
            if (c < C) p[c] = ag[i];
          }
        } else {
          gn_store<T, VEC>(static_cast<T*>(a.dgate) + grp * C, t, tpr, C, ag);
        }
      }
    }
  }
  float* const acc[5] = {apw, apb, asc, anw, anb};
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    slot_sum<VEC>(acc[k], buf, t, slot, slots, tpr);
    if (slot == 0) {
      float* p = a.part + (static_cast<int64_t>(blockIdx.x) * 5 + k) * C;
#pragma unroll
      for (int i = 0; i < kGnVals; ++i) {
        const int c = gn_channel<VEC>(t, tpr, i);
        if (c < C) p[c] = acc[k][i];
      }
    }
  }
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
  const int64_t most = sms * (p.threads <= 128 ? 8 : p.threads <= 256 ? 4 : 2);
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
  const size_t smem = p.slots > 1 ? static_cast<size_t>(p.threads) * kGnVals * 4 : 0;
  int rc = gnorm_dispatch(dtype, fits, p.tpr, [&](auto t, auto v, auto m) {
    gnorm_backward_kernel<decltype(t), decltype(v)::value, decltype(m)::value>
        <<<static_cast<unsigned>(p.bblocks), p.threads, smem, st>>>(a);
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
