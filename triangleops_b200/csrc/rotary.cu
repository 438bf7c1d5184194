// rotary.cu — rotary positions with several axes, for the queries and the keys in one launch.
//
// Frequency f belongs to axis[f]; its pair of channels (f, D/2 + f), or (2f, 2f + 1) when
// interleaved, turns by the angle positions[axis[f]][b][n] * inv_freq[f]:
//   (a, b) -> (a cos - b sin, a sin + b cos)
// The backward pass is the same turn by the negated angle. Channels of no pair are copied.
//
// Bound by memory (q and k read once and written once): 2 x 8192 tokens of 32 + 8 heads of 128
// channels in 16 bits, 336 MB, take 59 us, 5.7 TB/s. The angles are shared by the heads of a token,
// so a block takes some tokens, computes their cosines and sines once into shared memory and walks
// over all heads. The angle is formed and brought into one turn in fp64: a position of
// some thousands times a frequency near 1 would lose three digits of the angle in fp32.
#include <cuda_runtime.h>
#include "sm100.cuh"
#include "status.h"

namespace tops {

// n / d for n and d below 2^31 by a product: m = ceil(2^63 / d) makes it exact, and three instructions
// (the division's twenty, four times a piece, were a third of what the kernel issued).
struct Quotient {
  uint64_t m = 0;
  uint32_t d = 1;
  Quotient() = default;
  explicit Quotient(uint32_t d) : m(((uint64_t(1) << 63) + d - 1) / d), d(d) {}
  __device__ __forceinline__ uint32_t of(uint32_t n, uint32_t& rest) const {
    const uint64_t high = static_cast<uint64_t>(n) * static_cast<uint32_t>(m >> 32);
    const uint32_t q = static_cast<uint32_t>((high + __umulhi(n, static_cast<uint32_t>(m))) >> 31);
    rest = n - q * d;
    return q;
  }
};

struct RotaryArgs {
  int64_t B, N;
  int Hq, Hk, D, P, A;  // P pairs, 2 P <= D; A axes
  int interleaved, wide, negate;  // wide: int64 positions
  int tok;                        // tokens a block
  Quotient by_n, by_p, by_items, by_heads;  // tokens of a sequence, pairs, pieces of a head, a block's heads
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

// 16 bytes of a head as fp32 values and back
template <typename T>
__device__ __forceinline__ void rot_unpack(const uint4& w, float* f) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if constexpr (sizeof(T) == 4)
      f[i] = __uint_as_float(u[i]);
    else
      f[2 * i] = Elem<T>::lo(u[i]), f[2 * i + 1] = Elem<T>::hi(u[i]);
}
template <typename T>
__device__ __forceinline__ uint4 rot_pack(const float* f) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]),
                      Elem<T>::pack2(f[6], f[7]));
}

// Two pieces of VEC channels of a head at a time, 16 bytes each, one from either half (VEC 1: channel
// by channel): the two halves' channels of VEC pairs, or VEC neighbouring pairs. Block x takes the
// tokens x * tok.. and the heads y * by_heads.d... A thread's next pieces are on their way while it
// turns the present ones, the first ones while the block forms the angles.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 cs[];  // [tok][P]
  const uint32_t t0 = blockIdx.x * a.tok, tokens = static_cast<uint32_t>(a.B * a.N);
  const uint32_t nt = min(static_cast<uint32_t>(a.tok), tokens - t0), P = a.P, half = a.D / 2, Hq = a.Hq;
  const uint32_t h_lo = blockIdx.y * a.by_heads.d, nh = min(a.by_heads.d, Hq + a.Hk - h_lo);
  const uint32_t all = nt * a.by_heads.d * a.by_items.d;
  const T* src;
  T* dst;
  uint32_t e, ti, h;
  auto find = [&](uint32_t i) {  // item i of the block; false: a head past the block's share
    uint32_t b, n, hi;
    ti = a.by_heads.of(a.by_items.of(i, e), hi);
    if (i >= all || hi >= nh) return false;
    h = h_lo + hi;
    const uint32_t tok = t0 + ti;
    b = a.by_n.of(tok, n);
    const bool isq = h < Hq;
    const uint32_t hh = isq ? h : h - Hq;
    src = isq ? static_cast<const T*>(a.q) + b * a.qs[0] + n * a.qs[1] + hh * a.qs[2]
              : static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[1] + hh * a.ks[2];
    dst = isq ? static_cast<T*>(a.qo) + (static_cast<int64_t>(tok) * Hq + hh) * a.D
              : static_cast<T*>(a.ko) + (static_cast<int64_t>(tok) * a.Hk + hh) * a.D;
    return true;
  };
  uint32_t i = threadIdx.x;
  bool live = find(i);
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  auto load = [&] {
    if constexpr (VEC > 1) {
      if (!live) return;
      lo = *reinterpret_cast<const uint4*>(src + e * VEC);
      hi = *reinterpret_cast<const uint4*>(src + half + e * VEC);
    }
  };
  load();
  for (uint32_t j = threadIdx.x; j < nt * P; j += kRotThreads) {
    uint32_t f, n;
    const uint32_t tok = t0 + a.by_p.of(j, f), b = a.by_n.of(tok, n);
    const int ax = a.axis[f];
    float2 v = make_float2(1.f, 0.f);  // no such axis: the pair stays as it is
    if (ax >= 0 && ax < a.A) {
      const int64_t at = ax * a.ps[0] + b * a.ps[1] + n * a.ps[2];
      const double p = a.wide ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                              : static_cast<double>(static_cast<const int*>(a.pos)[at]);
      v = turn_of(p, a.inv_freq[f]);
      if (a.negate) v.y = -v.y;
    }
    cs[j] = v;
  }
  __syncthreads();
  while (i < all) {
    const uint32_t d = e;
    const float2* w = cs + ti * P;
    const T* from = src;
    T* to = dst;
    const uint4 p = lo, r = hi;
    const bool here = live;
    i += kRotThreads;
    live = find(i);
    load();
    if (!here) continue;
    if constexpr (VEC == 1) {
      const uint32_t f = a.interleaved ? d / 2 : d, mate = a.interleaved ? d ^ 1 : d + half;
      if (a.interleaved) {
        if (f >= P) {
          to[d] = from[d];
        } else {
          const float u = static_cast<float>(from[d]), v = static_cast<float>(from[mate]);
          to[d] = static_cast<T>(d & 1 ? fmaf(u, w[f].x, v * w[f].y) : fmaf(u, w[f].x, -(v * w[f].y)));
        }
      } else if (f >= P) {
        if (f < half) to[d] = from[d];
        to[mate] = from[mate];
      } else {
        const float u = static_cast<float>(from[d]), v = static_cast<float>(from[mate]);
        to[d] = static_cast<T>(fmaf(u, w[f].x, -(v * w[f].y)));
        to[mate] = static_cast<T>(fmaf(v, w[f].x, u * w[f].y));
      }
    } else {
      float x[VEC], y[VEC];
      rot_unpack<T>(p, x);
      rot_unpack<T>(r, y);
      auto turn = [&](float& u, float& v, uint32_t f) {
        if (f >= P) return;
        const float2 k = w[f];
        const float uc = fmaf(u, k.x, -(v * k.y));
        v = fmaf(v, k.x, u * k.y);
        u = uc;
      };
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          turn(x[j], x[j + 1], (d * VEC + j) / 2);
          turn(y[j], y[j + 1], (half + d * VEC + j) / 2);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) turn(x[j], y[j], d * VEC + j);
      }
      *reinterpret_cast<uint4*>(to + half + d * VEC) = rot_pack<T>(y);
      *reinterpret_cast<uint4*>(to + d * VEC) = rot_pack<T>(x);
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
  const int vec = dtype == TOPS_F32 ? 4 : 8;
  auto fits = [&](const void* p, const void* o, const int64_t* st) {
    return aligned16(p) && aligned16(o) && st[0] % vec == 0 && st[1] % vec == 0 && st[2] % vec == 0;
  };
  const bool whole = D % (2 * vec) == 0 && (Hq == 0 || fits(q, q_out, a.qs)) && (Hk == 0 || fits(k, k_out, a.ks));
  // items of a head: pieces of the first half with those of the second; channel by channel, with (odd
  // D) the last one alone, or every channel where its mate is its neighbour
  const int64_t H = Hq + Hk, items = whole ? D / 2 / vec : interleaved ? D : D - D / 2;
  // Three items a thread or more, so that loads are ahead of the work: 1, 2, 4, 8, 16 tokens a block take
  // 96, 57, 39, 35, 31 us at 48 items a token (8 x 4096 tokens) and 82, 70, 64, 64, 70 us at 320 (2 x 8192).
  // Few tokens: fewer a block, down to one with the heads shared by blocks, until the SMs are busy. And no
  // more than 48 KB of angles, what a block gets unasked (one token's are 4 KB at most).
  const int64_t tokens = B * N, sms = sm_count(), most = 48 * 1024 / (P * static_cast<int64_t>(sizeof(float2)));
  a.tok = 1;
  while (a.tok < 16 && 2 * a.tok <= most && a.tok * H * items < 3 * kRotThreads && tokens >= 4 * sms * a.tok)
    a.tok *= 2;
  const int64_t blocks = (tokens + a.tok - 1) / a.tok;
  int64_t shares = blocks >= 2 * sms ? 1 : (2 * sms + blocks - 1) / blocks;
  shares = shares < H ? shares : H;
  a.by_heads = Quotient(static_cast<uint32_t>((H + shares - 1) / shares));
  shares = (H + a.by_heads.d - 1) / a.by_heads.d;  // none of them empty
  a.by_n = Quotient(static_cast<uint32_t>(N)), a.by_p = Quotient(static_cast<uint32_t>(P));
  a.by_items = Quotient(static_cast<uint32_t>(items));
  const size_t smem = a.tok * P * sizeof(float2);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(shares));
  return by_io_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (whole)
      rotary_kernel<T, 16 / sizeof(T)><<<grid, kRotThreads, smem, st>>>(a);
    else
      rotary_kernel<T, 1><<<grid, kRotThreads, smem, st>>>(a);
    return launch_status();
  });
}
