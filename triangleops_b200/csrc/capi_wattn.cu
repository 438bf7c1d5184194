// capi_wattn.cu — C-ABI entry points of windowed attention with sinks. Declared in
// include/triangleops_b200.h.
#include <cuda_runtime.h>
#include "sm100.cuh"
#include "status.h"
#include "wattn.h"

namespace tops {

// The sizes that the kernels can count: sequences, heads and the channels of a token in 31 bits, keys in 30
// (a position plus a window fits 31).
inline int wattn_sizes(int64_t B, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D) {
  constexpr int64_t kInt = int64_t(1) << 31;
  if (B < 0 || Nk < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > 256) return TOPS_ERR_SHAPE;
  return B < kInt && Nk < kInt / 2 && Hq < kInt / D ? TOPS_OK : TOPS_ERR_SHAPE;
}

inline int wattn_args(WattnArgs& a, int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D,
                      const void* q, const void* k, const void* v, const int64_t* st, const uint8_t* mask,
                      int64_t left, int64_t right, int64_t sinks, float scale) {
  if (const int rc = wattn_sizes(B, Nk, Hq, Hkv, D)) return rc;
  if (Nq < 0 || Nk < Nq || (Nk > 0 && B * Hq > ((int64_t(1) << 33) - 1) / Nk)) return TOPS_ERR_SHAPE;
  if (left < 0 || right < 0 || sinks < 0) return TOPS_ERR_ARG;
  if (B > 0 && Nq > 0 && (q == nullptr || k == nullptr || v == nullptr || st == nullptr)) return TOPS_ERR_ARG;
  a.B = static_cast<int>(B);
  a.Nq = static_cast<int>(Nq);
  a.Nk = static_cast<int>(Nk);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.left = static_cast<int>(left < Nk ? left : Nk);
  a.right = static_cast<int>(right < Nk ? right : Nk);
  a.sinks = static_cast<int>(sinks < Nk ? sinks : Nk);
  a.q = q;
  a.k = k;
  a.v = v;
  if (st != nullptr)
    for (int i = 0; i < 3; ++i) {
      a.qs[i] = st[i];
      a.ks[i] = st[3 + i];
      a.vs[i] = st[6 + i];
    }
  a.mask = mask;
  a.lengths = nullptr;
  a.scale = scale;
  return TOPS_OK;
}

template <typename F>
int by_io_type(int dtype, F&& f) {
  if (dtype == TOPS_BF16) return f(__nv_bfloat16());
  if (dtype == TOPS_F16) return f(__half());
  if (dtype == TOPS_F32) return f(float());
  return TOPS_ERR_DTYPE;
}

}  // namespace tops

using namespace tops;

extern "C" int tops_window_attn_forward(int dtype, int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv,
                                        int64_t D, const void* q, const void* k, const void* v,
                                        const int64_t* strides, const uint8_t* mask, int64_t left, int64_t right,
                                        int64_t sinks, float scale, void* out, float* lse, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  WattnArgs a;
  if (const int rc = wattn_args(a, B, Nq, Nk, Hq, Hkv, D, q, k, v, strides, mask, left, right, sinks, scale)) return rc;
  if (B == 0 || Nq == 0) return TOPS_OK;
  if (out == nullptr) return TOPS_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (wattn_tensor(dtype, a) && aligned16(out))
    return dtype == TOPS_BF16 ? run_wattn_forward<__nv_bfloat16>(dtype, a, out, lse, st)
                              : run_wattn_forward<__half>(dtype, a, out, lse, st);
  return by_io_type(dtype, [&](auto t) { return run_wattn_generic<decltype(t)>(a, out, lse, st); });
}

extern "C" int tops_window_attn_backward(int dtype, int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv,
                                         int64_t D, const void* q, const void* k, const void* v,
                                         const int64_t* strides, const uint8_t* mask, int64_t left, int64_t right,
                                         int64_t sinks, float scale, const void* dout, const int64_t* dout_strides,
                                         const void* out, const float* lse, void* workspace, void* dq, void* dk,
                                         void* dv, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  WattnArgs a;
  if (const int rc = wattn_args(a, B, Nq, Nk, Hq, Hkv, D, q, k, v, strides, mask, left, right, sinks, scale)) return rc;
  if (B == 0 || Nk == 0) return TOPS_OK;
  if (dk == nullptr || dv == nullptr) return TOPS_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (Nq == 0) {  // no query reads a key: nothing else of the call is looked at
    const size_t bytes = static_cast<size_t>(B) * Nk * Hkv * D * (dtype == TOPS_F32 ? 4 : 2);
    return cudaMemsetAsync(dk, 0, bytes, st) == cudaSuccess && cudaMemsetAsync(dv, 0, bytes, st) == cudaSuccess
               ? launch_status()
               : TOPS_ERR_CUDA;
  }
  if (dout_strides == nullptr || workspace == nullptr || dout == nullptr || out == nullptr || lse == nullptr ||
      dq == nullptr)
    return TOPS_ERR_ARG;
  if (!aligned16(workspace)) return TOPS_ERR_ALIGN;
  float* delta = static_cast<float*>(workspace);
  if (wattn_tensor(dtype, a) && wattn_fits(dout, dout_strides, a.B, a.Nq, a.Hq) && aligned16(out) &&
      aligned16(dq) && aligned16(dk) && aligned16(dv))
    return dtype == TOPS_BF16
               ? run_wattn_backward<__nv_bfloat16>(dtype, a, dout, dout_strides, out, lse, delta, dq, dk, dv, st)
               : run_wattn_backward<__half>(dtype, a, dout, dout_strides, out, lse, delta, dq, dk, dv, st);
  return by_io_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (const int rc = run_wattn_delta<T>(a, dout, dout_strides, out, delta, st)) return rc;
    return run_wattn_generic_backward<T>(a, dout, dout_strides, lse, delta, dq, dk, dv, st);
  });
}

extern "C" int tops_window_attn_backward_workspace_bytes(int dtype, int64_t B, int64_t Nq, int64_t Nk, int64_t Hq,
                                                         int64_t Hkv, int64_t D, int64_t left, int64_t right,
                                                         int64_t sinks, int64_t* bytes) {
  if (bytes == nullptr) return TOPS_ERR_ARG;
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  WattnArgs a;
  if (const int rc = wattn_args(a, B, 0, Nk, Hq, Hkv, D, nullptr, nullptr, nullptr, nullptr, nullptr, left, right,
                                sinks, 1.f))
    return rc;
  if (Nq < 0 || Nq > Nk) return TOPS_ERR_SHAPE;
  const WattnBwdPlan p = wattn_bwd_plan(a, Nq);
  *bytes = (2 * p.stats + 4 + p.part) * 4;  // (the CUDA-core path needs less)
  return TOPS_OK;
}

extern "C" int tops_window_attn_decode_workspace_bytes(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D,
                                                       int64_t window, int64_t sinks, int64_t* bytes) {
  if (bytes == nullptr || window < 1 || sinks < 0) return TOPS_ERR_ARG;
  if (const int rc = wattn_sizes(B, N, Hq, Hkv, D)) return rc;
  // a plan divides the SMs among the sequences
  *bytes = B == 0 || N == 0 ? 0 : wattn_decode_plan(B, N, Hq, Hkv, D, window, sinks).part * 4;
  return TOPS_OK;
}

extern "C" int tops_window_attn_decode(int dtype, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D,
                                       const void* q, const void* k, const void* v, const int64_t* strides,
                                       const int32_t* lengths, int64_t window, int64_t sinks, float scale,
                                       void* workspace, void* out, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (window < 1 || sinks < 0) return TOPS_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (N == 0) {  // caches without a place: no sequence has a key
    if (const int rc = wattn_sizes(B, N, Hq, Hkv, D)) return rc;
    if (B == 0) return TOPS_OK;
    if (out == nullptr) return TOPS_ERR_ARG;
    const size_t bytes = static_cast<size_t>(B) * Hq * D * (dtype == TOPS_F32 ? 4 : 2);
    return cudaMemsetAsync(out, 0, bytes, st) == cudaSuccess ? TOPS_OK : TOPS_ERR_CUDA;
  }
  WattnArgs a;
  if (strides == nullptr) return TOPS_ERR_ARG;
  const int64_t full[9] = {strides[0], 0,          strides[1], strides[2], strides[3],
                           strides[4], strides[5], strides[6], strides[7]};
  if (const int rc = wattn_args(a, B, 1, N, Hq, Hkv, D, q, k, v, full, nullptr, window - 1, 0, sinks, scale)) return rc;
  if (B == 0) return TOPS_OK;
  if (lengths == nullptr || out == nullptr) return TOPS_ERR_ARG;
  a.lengths = lengths;
  if (dtype != TOPS_F32 && D % 8 == 0 && D <= 128 && wattn_decode_rows(q, a.qs[0], a.qs[2], 0) &&
      wattn_decode_rows(k, a.ks[0], a.ks[1], a.ks[2]) && wattn_decode_rows(v, a.vs[0], a.vs[1], a.vs[2])) {
    float* part = static_cast<float*>(workspace);
    return dtype == TOPS_BF16 ? run_wattn_decode<__nv_bfloat16>(a, window, out, part, st)
                              : run_wattn_decode<__half>(a, window, out, part, st);
  }
  return by_io_type(dtype, [&](auto t) { return run_wattn_generic<decltype(t)>(a, out, nullptr, st); });
}

extern "C" int tops_window_attn_store(int dtype, int64_t B, int64_t N, int64_t Hkv, int64_t D, const void* k, const void* v,
                                      const int64_t* strides, const int32_t* lengths, void* k_cache, void* v_cache,
                                      const int64_t* cache_strides, void* stream) {
  if (dtype != TOPS_BF16 && dtype != TOPS_F16 && dtype != TOPS_F32) return TOPS_ERR_DTYPE;
  if (const int rc = wattn_sizes(B, N, Hkv, Hkv, D)) return rc;
  if (B == 0 || N == 0) return TOPS_OK;
  if (k == nullptr || v == nullptr || strides == nullptr || lengths == nullptr || k_cache == nullptr ||
      v_cache == nullptr || cache_strides == nullptr)
    return TOPS_ERR_ARG;
  WattnStoreArgs a;
  for (int t = 0; t < 2; ++t) {
    for (int i = 0; i < 2; ++i) a.from[t][i] = strides[2 * t + i];
    for (int i = 0; i < 4; ++i) a.to[t][i] = cache_strides[4 * t + i];
  }
  a.src[0] = k, a.src[1] = v, a.dst[0] = k_cache, a.dst[1] = v_cache, a.lengths = lengths;
  a.N = static_cast<int>(N), a.H = static_cast<int>(Hkv), a.D = static_cast<int>(D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TOPS_F32)
    wattn_store_kernel<uint32_t><<<static_cast<unsigned>(B), 256, 0, st>>>(a);
  else
    wattn_store_kernel<uint16_t><<<static_cast<unsigned>(B), 256, 0, st>>>(a);
  return launch_status();
}
