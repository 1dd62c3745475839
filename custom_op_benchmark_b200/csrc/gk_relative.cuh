// The bucket of every edge from the positions of its two ends, in whole numbers.
//
// With x = src_pos[other] - dst_pos[node], a direction has n_limits + 1 buckets: a distance d belongs to the number of limits that
// are at most d.  both = 0: d = max(-x, 0).  both = 1: d = |x|, and positions ahead (x > 0) use a second set of buckets.  A position of
// no chunk gets -1.  Bound by the streams: 4 bytes of node and of endpoint in, 4 bytes out per edge, the positions out of the L2.
#pragma once
#include "gk_host.cuh"

namespace gk {

constexpr int kMostLimits = 1023;
struct Limits { int n; int both; long long at[kMostLimits]; };

template <typename P>
__global__ void __launch_bounds__(256)
relative_buckets_kernel(const int32_t* __restrict__ erow, const int32_t* __restrict__ other, long long E, const P* __restrict__ dst_pos,
                        const P* __restrict__ src_pos, const __grid_constant__ Limits limits, int32_t* __restrict__ out) {
  __shared__ long long s_at[kMostLimits + 1];
  for (int i = threadIdx.x; i < limits.n; i += 256) s_at[i] = limits.at[i];
  __syncthreads();
  const long long stride = (long long)gridDim.x * 256;
  for (long long j = (long long)blockIdx.x * 256 + threadIdx.x; j < E; j += stride) {
    const int r = __ldg(erow + j), c = __ldg(other + j);
    if (r < 0) { out[j] = -1; continue; }
    const long long to = src_pos ? (long long)__ldg(src_pos + c) : c, from = dst_pos ? (long long)__ldg(dst_pos + r) : r;
    const bool ahead = to > from;
    // without a sign: 64-bit positions may lie 2^63 and more apart
    unsigned long long d = ahead ? (unsigned long long)to - (unsigned long long)from : (unsigned long long)from - (unsigned long long)to;
    if (ahead && !limits.both) d = 0;
    int lo = 0, hi = limits.n;   // limits before lo are at most d, those from hi on are more
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((unsigned long long)s_at[mid] <= d) lo = mid + 1;
      else hi = mid;
    }
    out[j] = lo + (limits.both && ahead ? limits.n + 1 : 0);
  }
}

template <typename P, class GS>
inline int relative_buckets(const GS& gs, long long C, long long E, const P* dst_pos, const P* src_pos, const int64_t* limits, int n_limits,
                            int both, int32_t* out, void* ws, size_t wsb, cudaStream_t st) {
  GK_TRY(check_sizes(C, E, 0, 0, 1, 1));
  if (n_limits < 0 || (n_limits && !limits)) return GRAPHOP_ERR_INVALID_ARGUMENT;
  if (n_limits > kMostLimits) return GRAPHOP_ERR_UNSUPPORTED;
  Limits l;
  l.n = n_limits;
  l.both = both != 0;
  for (int i = 0; i < n_limits; ++i) {
    if (limits[i] < (i ? limits[i - 1] : 0)) return GRAPHOP_ERR_INVALID_ARGUMENT;
    l.at[i] = limits[i];
  }
  if (E == 0) return GRAPHOP_OK;
  if (!gs.valid(true) || !out) return GRAPHOP_ERR_INVALID_ARGUMENT;
  Arena ar(ws, wsb);
  GraphView g;
  GK_TRY(gs(ar, -1, st, &g));
  const long long blocks = (E + 255) / 256;
  relative_buckets_kernel<P><<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, st>>>(g.erow, g.other, E, dst_pos, src_pos, l, out);
  GK_LAUNCHED("relative_buckets");
  return GRAPHOP_OK;
}

}  // namespace gk
