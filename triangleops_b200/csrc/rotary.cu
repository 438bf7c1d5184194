// rotary.cu — rotary positions with several axes, for the queries and the keys in one launch.
//
// Frequency f belongs to axis[f]; its pair of channels (f, D/2 + f), or (2f, 2f + 1) when
// interleaved, turns by the angle positions[axis[f]][b][n] * inv_freq[f]:
//   (a, b) -> (a cos - b sin, a sin + b cos)
// The backward pass is the same turn by the negated angle. Channels of no pair are copied.
//
// Bound by memory (q and k read once and written once); the angles are shared by the heads of a
// token, so a block takes some tokens, computes their cosines and sines once into shared memory
// and walks over all heads. The angle is formed and brought into one turn in fp64: a position of
// some thousands times a frequency near 1 would lose three digits of the angle in fp32.
#include <cuda_runtime.h>
#include "sm100.cuh"
#include "status.h"

namespace tops {

struct RotaryArgs {
  int64_t B, N;
  int Hq, Hk, D, P, A;  // P pairs, 2 P <= D; A axes
  int interleaved, wide, negate;  // wide: int64 positions
  int tok;                        // tokens a block
  const void *q, *k;
  int64_t qs[3], ks[3], ps[3];  // strides of (batch, token, head) and of positions (axis, batch, token)
  const void* pos;
  const float* inv_freq;
  const int* axis;
  void *qo, *ko;  // contiguous (B, N, H, D)
};

constexpr int kRotThreads = 256;

// cosine and sine of pos * freq, the angle in half turns of one turn
__device__ __forceinline__ float2 turn_of(double pos, float freq) {
  const double half = pos * freq * 0.31830988618379067154;  // 1 / pi
  float s, c;
  sincospif(static_cast<float>(fma(rint(0.5 * half), -2.0, half)), &s, &c);
  return make_float2(c, s);
}

// Two pieces of VEC channels of a head at a time, 16 bytes each, one from either half (VEC 1: channel
// by channel): the two halves' channels of VEC pairs, or VEC neighbouring pairs. Block (x, y): tokens
// x * tok.., share y of the heads.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 cs[];  // [tok][P]
  const uint32_t t0 = blockIdx.x * a.tok, tokens = static_cast<uint32_t>(a.B * a.N), N = static_cast<uint32_t>(a.N);
  const uint32_t nt = min(static_cast<uint32_t>(a.tok), tokens - t0), P = a.P;
  for (uint32_t i = threadIdx.x; i < nt * P; i += kRotThreads) {
    const uint32_t tok = t0 + i / P, f = i % P;
    const int ax = a.axis[f];
    float2 v = make_float2(1.f, 0.f);  // no such axis: the pair stays as it is
    if (ax >= 0 && ax < a.A) {
      const int64_t at = ax * a.ps[0] + tok / N * a.ps[1] + tok % N * a.ps[2];
      const double p = a.wide ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                              : static_cast<double>(static_cast<const int*>(a.pos)[at]);
      v = turn_of(p, a.inv_freq[f]);
      if (a.negate) v.y = -v.y;
    }
    cs[i] = v;
  }
  __syncthreads();
  const uint32_t H = a.Hq + a.Hk, half = a.D / 2;
  const uint32_t h_lo = H * blockIdx.y / gridDim.y, nh = H * (blockIdx.y + 1) / gridDim.y - h_lo;
  // items of a head: pieces of the first half with those of the second; channel by channel, with (odd
  // D) the last one alone, or every channel where its mate is its neighbour
  const uint32_t items = VEC > 1 ? half / VEC : a.interleaved ? a.D : a.D - half;
  for (uint32_t i = threadIdx.x; i < nt * nh * items; i += kRotThreads) {
    const uint32_t hi = i / items, e = i % items, ti = hi / nh, h = h_lo + hi % nh;
    const uint32_t tok = t0 + ti, b = tok / N, n = tok % N;
    const bool isq = h < static_cast<uint32_t>(a.Hq);
    const uint32_t hh = isq ? h : h - a.Hq;
    const T* src = isq ? static_cast<const T*>(a.q) + b * a.qs[0] + n * a.qs[1] + hh * a.qs[2]
                       : static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[1] + hh * a.ks[2];
    T* dst = isq ? static_cast<T*>(a.qo) + (static_cast<int64_t>(tok) * a.Hq + hh) * a.D
                 : static_cast<T*>(a.ko) + (static_cast<int64_t>(tok) * a.Hk + hh) * a.D;
    const float2* w = cs + ti * P;
    if constexpr (VEC == 1) {
      const uint32_t f = a.interleaved ? e / 2 : e;
      const uint32_t d = e, mate = a.interleaved ? e ^ 1 : e + half;
      if (a.interleaved) {
        if (f >= P) {
          dst[d] = src[d];
        } else {
          const float u = static_cast<float>(src[d]), v = static_cast<float>(src[mate]);
          dst[d] = static_cast<T>(e & 1 ? fmaf(u, w[f].x, v * w[f].y) : fmaf(u, w[f].x, -(v * w[f].y)));
        }
      } else if (f >= P) {
        if (f < half) dst[d] = src[d];
        dst[mate] = src[mate];
      } else {
        const float u = static_cast<float>(src[d]), v = static_cast<float>(src[mate]);
        dst[d] = static_cast<T>(fmaf(u, w[f].x, -(v * w[f].y)));
        dst[mate] = static_cast<T>(fmaf(v, w[f].x, u * w[f].y));
      }
    } else {
      union Piece {
        uint4 w;
        T v[VEC];
      };
      Piece p, r;
      p.w = *reinterpret_cast<const uint4*>(src + e * VEC);
      r.w = *reinterpret_cast<const uint4*>(src + half + e * VEC);
      auto turn = [&](T& x, T& y, uint32_t f) {
        if (f >= P) return;
        const float u = static_cast<float>(x), v = static_cast<float>(y);
        x = static_cast<T>(fmaf(u, w[f].x, -(v * w[f].y)));
        y = static_cast<T>(fmaf(v, w[f].x, u * w[f].y));
      };
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          turn(p.v[j], p.v[j + 1], (e * VEC + j) / 2);
          turn(r.v[j], r.v[j + 1], (half + e * VEC + j) / 2);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) turn(p.v[j], r.v[j], e * VEC + j);
      }
      *reinterpret_cast<uint4*>(dst + half + e * VEC) = r.w;
      *reinterpret_cast<uint4*>(dst + e * VEC) = p.w;
    }
  }
}

}  // namespace tops

using namespace tops;

extern "C" int tops_rotary(int dtype, int64_t B, int64_t N, int64_t Hq, int64_t Hk, int64_t D, int64_t P,
                           int64_t A, int interleaved, int negate, const void* q, const void* k, const int64_t* strides,
                           const void* positions, int wide, const int64_t* pos_strides, const float* inv_freq,
                           const int32_t* axis, void* q_out, void* k_out, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (B < 0 || N < 0 || Hq < 0 || Hk < 0 || Hq + Hk <= 0 || D <= 0 || D > 1024 || P <= 0 || 2 * P > D || A <= 0)
    return TOPS_ERR_SHAPE;
  if (Hq + Hk > 4096 || B * N >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  if (B == 0 || N == 0) return TOPS_OK;
  if ((Hq > 0 && (q == nullptr || q_out == nullptr)) || (Hk > 0 && (k == nullptr || k_out == nullptr)) ||
      strides == nullptr || positions == nullptr || pos_strides == nullptr || inv_freq == nullptr || axis == nullptr)
    return TOPS_ERR_ARG;
  RotaryArgs a = {};
  a.B = B, a.N = N, a.Hq = static_cast<int>(Hq), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.P = static_cast<int>(P), a.A = static_cast<int>(A), a.interleaved = interleaved, a.wide = wide, a.negate = negate;
  a.q = q, a.k = k, a.pos = positions, a.inv_freq = inv_freq, a.axis = axis, a.qo = q_out, a.ko = k_out;
  for (int i = 0; i < 3; ++i) a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.ps[i] = pos_strides[i];
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // few tokens: one a block, and the heads shared by blocks until the SMs are busy
  const int64_t tokens = B * N, sms = sm_count();
  a.tok = tokens >= 8 * sms ? 4 : 1;
  const int64_t blocks = (tokens + a.tok - 1) / a.tok;
  int64_t shares = tokens >= 8 * sms ? 1 : (2 * sms + blocks - 1) / blocks;
  shares = shares < Hq + Hk ? shares : Hq + Hk;
  const size_t smem = a.tok * P * sizeof(float2);
  return by_io_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = 16 / sizeof(T);
    auto fits = [&](const void* p, const void* o, const int64_t* st) {
      return aligned16(p) && aligned16(o) && st[0] % VEC == 0 && st[1] % VEC == 0 && st[2] % VEC == 0;
    };
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(shares));
    if (D % (2 * VEC) == 0 && (Hq == 0 || fits(q, q_out, a.qs)) &&
        (Hk == 0 || fits(k, k_out, a.ks)))
      rotary_kernel<T, VEC><<<grid, kRotThreads, smem, st>>>(a);
    else
      rotary_kernel<T, 1><<<grid, kRotThreads, smem, st>>>(a);
    return launch_status();
  });
}
