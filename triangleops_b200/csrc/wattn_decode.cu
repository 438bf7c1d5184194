// wattn_decode.cu — windowed attention with sinks for one query a sequence (16-bit IO, D a multiple
// of 8 up to 128, 16-byte aligned rows).
//
// Bound by memory: each visible key and value is read once. The query heads of a key head (up to 16;
// more are done 16 at a time) are the rows of mma.sync tiles, so that a key read from memory meets
// all its queries; tcgen05 would want 128 rows.
//
// A warp walks over 16 keys at a time without shared memory: K and V go from memory to the
// registers of the MMA's B operand by 16-byte loads. The order of a contraction's terms and of an
// output's columns is free as long as both sides agree, so a lane's 8 neighbouring channels of K
// serve two contraction steps, and its 8 neighbouring channels of V eight tiles of output columns:
//   S: thread (key lane/4, part lane%4) holds channels 32 s + 8 (lane%4) ..+7 of its key
//   O: thread (column lane/4, keys 2 (lane%4) + {0, 1, 8, 9}) holds channels 64 u + 8 (lane/4) ..+7
// The next keys are on their way while the present ones are computed.
//
// 64 sequences of up to 8192 tokens, 32 heads of 128 on 8, window 4096: 192 us, 5.6 TB/s.
//
// The visible keys of one (sequence, key head) are shared by the warps of a block, by the blocks of a
// cluster (partial maxima, sums and outputs are joined through distributed shared memory), and, for
// few sequences with long windows, by several clusters, whose parts a second kernel joins.
#include "sm100.cuh"
#include "wattn.h"

namespace tops {

struct WattnDecodeArgs {
  int N, Hq, Hkv, group, D, window, sinks;
  int rtiles;  // 16-row tiles of a group
  int splits;  // clusters that share a (sequence, key head, row tile)
  const void *q, *k, *v;
  int64_t qs[2], ks[3], vs[3];
  const int* lengths;
  float c;  // scale * log2(e)
  void* out;
  float* part;  // [units][splits][16][DT + 2]: sums of p v, then the maximum and the sum of p
};

template <int DT, int NW>
struct WattnDecodeSmem {
  float o[NW][16][DT];
  float m[NW][16], l[NW][16];
  float cm[16], cl[16];  // the block's
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// a float of another block's shared memory, at the place that `p` has in this one's
__device__ __forceinline__ float peer_load(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (Elem<T>::kFmt == 1)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NW: warps a block; blocks of two share an SM by fours
template <typename T, int DT, int NW>
__global__ void __launch_bounds__(32 * NW, NW == 2 ? 4 : 1) wattn_decode_kernel(const WattnDecodeArgs a) {
  using E = Elem<T>;
  constexpr int NS = DT / 32, NU = DT / 64;
  // f16 ends at 2^-24: p, at most 1, is held at 2^15 times its size, the sums with it
  constexpr float kLift = E::kFmt == 0 ? 15.f : 0.f;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<WattnDecodeSmem<DT, NW>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, t4 = lane & 3;
  const uint32_t cs = cluster_size(), rank = cluster_rank();
  const int cl = blockIdx.x / cs;
  const int split = cl % a.splits, unit = cl / a.splits;
  const int rt = unit % a.rtiles, hk = unit / a.rtiles % a.Hkv, b = unit / a.rtiles / a.Hkv;
  const int rows = min(16, a.group - rt * 16), h0 = hk * a.group + rt * 16;

  const int n = min(max(a.lengths[b], 0), a.N);
  const int lo = max(0, n - a.window), ns = min(a.sinks, lo), total = ns + n - lo;
  // this block's tiles of 16 keys
  const int tiles = (total + 15) >> 4, parts = a.splits * cs, part = split * cs + rank;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * part / parts);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / parts);

  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  auto key_of = [&](int t) { return static_cast<int64_t>(t < ns ? t : lo + t - ns); };
  const uint4 zero = make_uint4(0, 0, 0, 0);

  // Q: rows quad and quad + 8, the same channels as this thread's of K
  uint32_t qa[2 * NS][4];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int d = 32 * s + 8 * t4;
    uint4 u[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = quad + 8 * r;
      u[r] = row < rows && d < a.D
                 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs[0] + (h0 + row) * a.qs[1] + d)
                 : zero;
    }
    qa[2 * s][0] = u[0].x, qa[2 * s][1] = u[1].x, qa[2 * s][2] = u[0].y, qa[2 * s][3] = u[1].y;
    qa[2 * s + 1][0] = u[0].z, qa[2 * s + 1][1] = u[1].z, qa[2 * s + 1][2] = u[0].w, qa[2 * s + 1][3] = u[1].w;
  }

  uint4 kr[2][NS];
  auto load_k = [&](int tile) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int t = tile * 16 + 8 * nt + quad;
      const T* row = k + key_of(t) * a.ks[1];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int d = 32 * s + 8 * t4;
        kr[nt][s] = t < total && d < a.D ? load_stream(row + d) : zero;
      }
    }
  };

  float o[8 * NU][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8 * NU; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  int tile = first + warp;
  if (tile < last) load_k(tile);
  for (; tile < last; tile += NW) {
    uint4 vr[4][NU];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = tile * 16 + 2 * t4 + (j & 1) + 8 * (j >> 1);
      const T* row = v + key_of(t) * a.vs[1];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int d = 64 * u + 8 * quad;
        vr[j][u] = t < total && d < a.D ? load_stream(row + d) : zero;
      }
    }
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        mma_16816<T>(s[nt], qa[2 * i], kr[nt][i].x, kr[nt][i].y);
        mma_16816<T>(s[nt], qa[2 * i + 1], kr[nt][i].z, kr[nt][i].w);
      }
    }
    if (tile + NW < last) load_k(tile + NW);
    // rows quad (elements 0, 1) and quad + 8 (2, 3); keys 8 nt + 2 t4 + {0, 1}
    const int past = total - tile * 16;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = 8 * nt + 2 * t4 + (e & 1) < past ? s[nt][e] * a.c : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[nt][e]);
      }
    bool grown = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      grown = grown || mx[r] > m[r];
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float mn = fmaxf(m[r], mx[r]);
        const float f = mn == -INFINITY ? 1.f : ex2_approx(m[r] - mn);
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < 8 * NU; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r] - kLift;
        const float p0 = ex2_approx(s[nt][2 * r] - base), p1 = ex2_approx(s[nt][2 * r + 1] - base);
        l[r] += p0 + p1;
        pa[2 * nt + r] = E::pack2(p0, p1);
      }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vr[0][u]);
      const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vr[1][u]);
      const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vr[2][u]);
      const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vr[3][u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mma_16816<T>(o[8 * u + 2 * i], pa, __byte_perm(w0[i], w1[i], 0x5410), __byte_perm(w2[i], w3[i], 0x5410));
        mma_16816<T>(o[8 * u + 2 * i + 1], pa, __byte_perm(w0[i], w1[i], 0x7632), __byte_perm(w2[i], w3[i], 0x7632));
      }
    }
  }
  // ---------------- the block's warps ----------------
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t4 == 0) {
      sm.m[warp][quad + 8 * r] = m[r];
      sm.l[warp][quad + 8 * r] = l[r];
    }
    // o[8 u + e]: channel 64 u + 8 column + e, columns 2 t4 and 2 t4 + 1
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int col = 0; col < 2; ++col)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(&sm.o[warp][quad + 8 * r][64 * u + 8 * (2 * t4 + col) + e]) =
              make_float4(o[8 * u + e][2 * r + col], o[8 * u + e + 1][2 * r + col], o[8 * u + e + 2][2 * r + col],
                          o[8 * u + e + 3][2 * r + col]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * DT; i += 32 * NW) {
    const int row = i / DT, d = i % DT;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sm.m[w][row]);
    float x = 0.f, y = 0.f;
    if (top > -INFINITY)
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = ex2_approx(sm.m[w][row] - top);
        x = fmaf(sm.o[w][row][d], f, x);
        y = fmaf(sm.l[w][row], f, y);
      }
    sm.o[0][row][d] = x;  // no other thread reads this element
    if (d == 0) sm.cm[row] = top, sm.cl[row] = y;
  }
  // ---------------- the cluster's blocks, each a share of the elements ----------------
  if (cs > 1)
    cluster_sync();
  else
    __syncthreads();
  const int count = rows * DT / cs;
  for (int j = threadIdx.x; j < count; j += 32 * NW) {
    const int i = rank * count + j, row = i / DT, d = i % DT;
    float top = sm.cm[row], x, y;
    if (cs == 1) {
      x = sm.o[0][row][d], y = sm.cl[row];
    } else {
      for (uint32_t r = 0; r < cs; ++r) top = fmaxf(top, peer_load(&sm.cm[row], r));
      x = y = 0.f;
      if (top > -INFINITY)
        for (uint32_t r = 0; r < cs; ++r) {
          const float f = ex2_approx(peer_load(&sm.cm[row], r) - top);
          x = fmaf(peer_load(&sm.o[0][row][d], r), f, x);
          y = fmaf(peer_load(&sm.cl[row], r), f, y);
        }
    }
    if (a.part != nullptr) {
      float* p = a.part + ((static_cast<int64_t>(unit) * a.splits + split) * 16 + row) * (DT + 2);
      p[d] = x;
      if (d == 0) p[DT] = top, p[DT + 1] = y;
    } else if (d < a.D) {
      static_cast<T*>(a.out)[(static_cast<int64_t>(b) * a.Hq + h0 + row) * a.D + d] = E::from_f(y == 0.f ? 0.f : x / y);
    }
  }
  if (cs > 1) cluster_sync();  // the others may still be reading this block's shared memory
}

// Joins the clusters' parts of a unit, in order.
template <typename T, int DT>
__global__ void __launch_bounds__(DT) wattn_decode_join_kernel(const WattnDecodeArgs a) {
  using E = Elem<T>;
  const int row = blockIdx.y, unit = blockIdx.x, d = threadIdx.x;
  const int rt = unit % a.rtiles, hk = unit / a.rtiles % a.Hkv, b = unit / a.rtiles / a.Hkv;
  if (rt * 16 + row >= a.group || d >= a.D) return;
  const float* p = a.part + (static_cast<int64_t>(unit) * a.splits * 16 + row) * (DT + 2);
  constexpr int step = 16 * (DT + 2);
  float top = -INFINITY, x = 0.f, y = 0.f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, p[s * step + DT]);
  if (top > -INFINITY)
    for (int s = 0; s < a.splits; ++s) {
      const float f = ex2_approx(p[s * step + DT] - top);
      x = fmaf(p[s * step + d], f, x);
      y = fmaf(p[s * step + DT + 1], f, y);
    }
  static_cast<T*>(a.out)[(static_cast<int64_t>(b) * a.Hq + hk * a.group + rt * 16 + row) * a.D + d] =
      E::from_f(y == 0.f ? 0.f : x / y);
}

// The key and value rows of one token a sequence to their place in the caches, W: the type's width. A
// place that the caches do not have is not written.
struct WattnStoreArgs {
  int64_t from[2][2], to[2][4];  // strides of k and v (batch, head), of the caches (batch, token, head, channel)
  const void* src[2];
  void* dst[2];
  const int* lengths;
  int N, H, D;
};
template <typename W>
__global__ void __launch_bounds__(256) wattn_store_kernel(const WattnStoreArgs a) {
  const int64_t b = blockIdx.x;
  const int at = a.lengths[b], row = a.H * a.D;
  if (at < 0 || at >= a.N) return;
  for (int i = threadIdx.x; i < row; i += 256)
#pragma unroll
    for (int t = 0; t < 2; ++t)
      static_cast<W*>(a.dst[t])[b * a.to[t][0] + at * a.to[t][1] + i / a.D * a.to[t][2] + i % a.D * a.to[t][3]] =
          static_cast<const W*>(a.src[t])[b * a.from[t][0] + i / a.D * a.from[t][1] + i % a.D];
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct WattnDecodePlan {
  int warps, cluster, splits;
  int64_t units, part;
};

inline WattnDecodePlan wattn_decode_plan(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                                         int64_t sinks) {
  WattnDecodePlan p;
  const int64_t sms = sm_count(), w = window < N ? window : N, s = sinks < N - w ? sinks : N - w;
  const int64_t tiles = (w + s + 15) / 16;
  p.units = B * Hkv * ((Hq / Hkv + 15) / 16);
  // Few units: blocks of 8 warps, so that a cluster has 64 (one sequence, 2 key heads, window 1024:
  // 6.7 us against 7.9 with blocks of 2). Else blocks of 2, four an SM, whose starts and ends overlap
  // (8 sequences x 8 key heads, window 4096: 27 us against 56; 64 sequences: 192 against 206).
  p.warps = p.units * 8 < sms ? 8 : 2;
  p.cluster = 1;
  // more blocks while the SMs are not all busy and a warp has a tile to itself, or while the last
  // round of blocks would idle many SMs and there is work enough to share
  while (p.cluster < 8 && ((p.units * p.cluster < sms && tiles > p.cluster * p.warps) ||
                           (p.units * p.cluster < 6 * sms && tiles >= 8 * p.cluster * p.warps)))
    p.cluster *= 2;
  // Few units with long windows (more than 4 tiles a warp): as many parts as fill the SMs once, joined
  // by a second kernel. Clusters of 2 then, since those of 8 leave SMs over in every GPC (one sequence,
  // window 65536: 25 us against 32).
  p.splits = 1;
  if (p.warps == 8 && tiles > 4 * 8 * p.warps) {
    p.cluster = 2;
    const int64_t room = sms / (p.units * p.cluster), most = tiles / (2 * p.cluster * p.warps);
    p.splits = static_cast<int>(room < most ? room : most);
    if (p.splits < 1) p.splits = 1;
  }
  p.part = p.splits > 1 ? p.units * p.splits * 16 * ((D <= 64 ? 64 : 128) + 2) : 0;
  return p;
}

template <typename T, int DT, int NW>
static int launch_wattn_decode(const WattnArgs& a, const WattnDecodePlan& p, int64_t window, void* out, float* part,
                               cudaStream_t st) {
  WattnDecodeArgs f;
  f.N = a.Nk, f.Hq = a.Hq, f.Hkv = a.Hkv, f.group = a.Hq / a.Hkv, f.D = a.D;
  f.window = static_cast<int>(window < a.Nk ? window : a.Nk), f.sinks = a.sinks;
  f.rtiles = (f.group + 15) / 16, f.splits = p.splits;
  f.q = a.q, f.k = a.k, f.v = a.v;
  f.qs[0] = a.qs[0], f.qs[1] = a.qs[2];
  for (int i = 0; i < 3; ++i) f.ks[i] = a.ks[i], f.vs[i] = a.vs[i];
  f.lengths = a.lengths, f.c = a.scale * kLog2e, f.out = out, f.part = p.splits > 1 ? part : nullptr;
  if (p.splits > 1 && (part == nullptr || !aligned16(part))) return TOPS_ERR_ARG;
  const int64_t grid = p.units * p.splits * p.cluster;
  if (grid >= (int64_t(1) << 31)) return TOPS_ERR_SHAPE;
  const size_t smem = sizeof(WattnDecodeSmem<DT, NW>);
  auto kern = wattn_decode_kernel<T, DT, NW>;
  static std::atomic<uint64_t> done{0};
  set_smem_once(kern, smem, done);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(32 * NW);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, f);
  if (const int rc = launch_status()) return rc;
  if (p.splits == 1) return TOPS_OK;
  wattn_decode_join_kernel<T, DT><<<dim3(static_cast<unsigned>(p.units), 16), DT, 0, st>>>(f);
  return launch_status();
}

template <typename T>
int run_wattn_decode(const WattnArgs& a, int64_t window, void* out, float* part, cudaStream_t st) {
  const WattnDecodePlan p = wattn_decode_plan(a.B, a.Nk, a.Hq, a.Hkv, a.D, window, a.sinks);
  if (p.warps == 8)
    return a.D <= 64 ? launch_wattn_decode<T, 64, 8>(a, p, window, out, part, st)
                     : launch_wattn_decode<T, 128, 8>(a, p, window, out, part, st);
  return a.D <= 64 ? launch_wattn_decode<T, 64, 2>(a, p, window, out, part, st)
                   : launch_wattn_decode<T, 128, 2>(a, p, window, out, part, st);
}

// 16-byte rows; strides of zero are fine here
inline bool wattn_decode_rows(const void* p, int64_t s0, int64_t s1, int64_t s2) {
  return aligned16(p) && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
}

}  // namespace tops
