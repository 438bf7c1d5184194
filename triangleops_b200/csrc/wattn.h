// wattn.h — what the windowed-attention kernels share: the arguments of a call and which
// keys a query sees.
//
// Query i of a sequence with `nq` queries and `nk` keys stands at key position
// p = i + nk - nq (the queries are the last ones). It sees key j iff
//   j <= p + right  and  (j >= p - left  or  j < sinks)  and  mask[b][j] != 0.
#pragma once
#include <cstdint>

namespace tops {

struct WattnArgs {
  int B, Nq, Nk, Hq, Hkv, D;
  int left, right, sinks;  // left, right <= Nk (clamped on the host)
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // strides of (batch, token, head) in elements; channels are contiguous
  const uint8_t* mask;          // [B][Nk] (0: the key is not seen) or null
  const int* lengths;           // [B]: keys each sequence has in k and v (decode), or null: Nk
  float scale;
};

// The keys a query at position p sees, before the key mask: [0, n_sink) and [lo, hi).
struct Seen {
  int n_sink, lo, hi;
};
__host__ __device__ inline Seen seen_keys(int p, int left, int right, int sinks, int nk) {
  Seen s;
  s.hi = p + right + 1 < nk ? p + right + 1 : nk;
  if (s.hi < 0) s.hi = 0;
  s.lo = p > left ? p - left : 0;
  if (s.lo > s.hi) s.lo = s.hi;
  s.n_sink = sinks < s.lo ? sinks : s.lo;
  return s;
}

// The queries (as positions) that see key j: positions [lo, hi), all of [lo, nk) for a sink.
__host__ __device__ inline void seen_by(int j, int left, int right, int sinks, int nk, int& lo, int& hi) {
  lo = j > right ? j - right : 0;
  hi = j < sinks || j + left + 1 > nk ? nk : j + left + 1;
}

}  // namespace tops
