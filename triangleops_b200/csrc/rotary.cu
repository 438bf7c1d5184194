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
  const void *q, *k;
  int64_t qs[3], ks[3], ps[3];  // strides of (batch, token, head) and of positions (axis, batch, token)
  const void* pos;
  const float* inv_freq;
  const int* axis;
  void *qo, *ko;  // contiguous (B, N, H, D)
};

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;

__device__ __forceinline__ float2 turn_of(double pos, float freq) {
  const double a = pos * freq;
  const double turns = rint(a * 0.15915494309189533577);  // 1 / (2 pi)
  float s, c;
  sincosf(static_cast<float>(fma(turns, -6.283185307179586477, a)), &s, &c);
  return make_float2(c, s);
}

template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 cs[];  // [kRotTokens][P]
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kRotTokens, tokens = a.B * a.N;
  const int nt = static_cast<int>(tokens - t0 < kRotTokens ? tokens - t0 : kRotTokens);
  for (int i = threadIdx.x; i < nt * a.P; i += kRotThreads) {
    const int64_t tok = t0 + i / a.P;
    const int f = i % a.P;
    const int ax = a.axis[f];
    if (ax < 0 || ax >= a.A) {  // no such axis: the pair stays as it is
      cs[i] = make_float2(1.f, 0.f);
      continue;
    }
    const int64_t at = ax * a.ps[0] + tok / a.N * a.ps[1] + tok % a.N * a.ps[2];
    const double p = a.wide ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                            : static_cast<double>(static_cast<const int*>(a.pos)[at]);
    float2 v = turn_of(p, a.inv_freq[f]);
    if (a.negate) v.y = -v.y;
    cs[i] = v;
  }
  __syncthreads();
  const int H = a.Hq + a.Hk, half = a.D / 2;
  for (int i = threadIdx.x; i < nt * H * a.D; i += kRotThreads) {
    const int d = i % a.D, h = i / a.D % H, ti = i / a.D / H;
    const int64_t tok = t0 + ti, b = tok / a.N, n = tok % a.N;
    const bool isq = h < a.Hq;
    const int hh = isq ? h : h - a.Hq;
    const T* src = isq ? static_cast<const T*>(a.q) + b * a.qs[0] + n * a.qs[1] + hh * a.qs[2]
                       : static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[1] + hh * a.ks[2];
    T* dst = isq ? static_cast<T*>(a.qo) + (tok * a.Hq + hh) * a.D : static_cast<T*>(a.ko) + (tok * a.Hk + hh) * a.D;
    const int f = a.interleaved ? d / 2 : d % half;
    const bool second = a.interleaved ? d & 1 : d >= half;
    if (f >= a.P || (!a.interleaved && d >= 2 * half)) {
      dst[d] = src[d];
      continue;
    }
    const int mate = a.interleaved ? d ^ 1 : second ? d - half : d + half;
    const float2 w = cs[ti * a.P + f];
    const float u = static_cast<float>(src[d]), v = static_cast<float>(src[mate]);
    dst[d] = static_cast<T>(second ? fmaf(u, w.x, v * w.y) : fmaf(u, w.x, -(v * w.y)));
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
  const unsigned grid = static_cast<unsigned>((B * N + kRotTokens - 1) / kRotTokens);
  const size_t smem = kRotTokens * P * sizeof(float2);
  return by_io_type(dtype, [&](auto t) {
    rotary_kernel<decltype(t)><<<grid, kRotThreads, smem, st>>>(a);
    return launch_status();
  });
}
