// The bucket of every edge from the positions of its two ends, in whole numbers.
//
// With x = src_pos[other] - dst_pos[node], a direction has n_limits + 1 buckets: a distance d belongs to the number of limits that
// are at most d.  both = 0: d = max(-x, 0).  both = 1: d = |x|, and positions ahead (x > 0) use a second set of buckets.  A position of
// no chunk gets -1.  Bound by the streams: 4 bytes of node and of endpoint in, 4 bytes out per edge, the positions out of the L2.
//
// On chunk tables a chunk's node is known where its positions are: nothing is stored but the buckets.
#pragma once
#include "gk_host.cuh"

namespace gk {

constexpr int kMostLimits = 1023;
// Distances in D: 32 bits between 32-bit positions (limits beyond that are never reached, and left out), and between 64-bit ones where
// the limits fit, a distance beyond 32 bits standing as the largest that does; else 64.
// all: with those left out; top: the largest power of two <= n; near: the last limit where that is at most kNear, else -1.
template <typename D> struct Limits { int n, all, both, top, near; D at[kMostLimits]; };

constexpr int kRelPer = 8;   // positions per thread: their searches run side by side
constexpr int kNear = 1024;
// What a block keeps of the limits.  All distances from the last limit on share a bucket, so that limits of up to kNear (those of local
// attention) make a table by distance: one read per position instead of a search, 36 -> 22 us for 8.4M edges of bands and 31 limits (19 with 32-bit
// positions: 3.5 TB/s).
template <typename D> struct Shared { D at[kMostLimits + 1]; unsigned short near[kNear + 1]; };
template <typename D, int N>
__device__ __forceinline__ void search(int (&at)[N], const D (&d)[N], const Shared<D>& s, const Limits<D>& l) {
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = 0;
  for (int step = l.top; step; step >>= 1) {   // limits before at[i] are at most d[i]
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int next = at[i] + step;
      if (next <= l.n && s.at[next - 1] <= d[i]) at[i] = next;
    }
  }
}
// by the whole block
template <typename D>
__device__ __forceinline__ void load_limits(Shared<D>& s, const Limits<D>& l) {
  for (int i = threadIdx.x; i < l.n; i += blockDim.x) s.at[i] = l.at[i];
  __syncthreads();
  for (int i = threadIdx.x; i <= l.near; i += blockDim.x) {
    int at[1];
    const D d[1] = {(D)i};
    search<D, 1>(at, d, s, l);
    s.near[i] = (unsigned short)at[0];
  }
  __syncthreads();
}
template <typename D, int N>
__device__ __forceinline__ void buckets_of(int (&out)[N], const D (&d)[N], const bool (&ahead)[N], const Shared<D>& s, const Limits<D>& l) {
  int at[N];
  if (l.near >= 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] = s.near[d[i] < (D)l.near ? (int)d[i] : l.near];
  } else {
    search<D, N>(at, d, s, l);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = at[i] + (l.both && ahead[i] ? l.all + 1 : 0);
}
// without a sign: 64-bit positions may lie 2^63 and more apart
template <typename D, typename P>
__device__ __forceinline__ D distance(P from, P to, int both, bool& ahead) {
  using U = std::conditional_t<sizeof(P) == 4, unsigned, unsigned long long>;
  ahead = to > from;
  const U d = ahead ? (U)to - (U)from : (U)from - (U)to;
  if (ahead && !both) return D(0);
  if constexpr (sizeof(D) < sizeof(U)) return d > (U)~D(0) ? ~D(0) : (D)d;
  else return (D)d;
}

template <typename P, typename D>
__global__ void __launch_bounds__(256)
relative_planned_kernel(const int32_t* __restrict__ erow, const int32_t* __restrict__ other, long long E, const P* __restrict__ dst_pos,
                        const P* __restrict__ src_pos, const __grid_constant__ Limits<D> limits, int32_t* __restrict__ out) {
  __shared__ Shared<D> s_at;
  load_limits(s_at, limits);
  const long long j0 = ((long long)blockIdx.x * 256 + threadIdx.x) * kRelPer;
  if (j0 >= E) return;
  int r[kRelPer], c[kRelPer], b[kRelPer];
  // a plan's tables are aligned; the caller's own endpoints and the result need not be
  const bool whole = j0 + kRelPer <= E, wide = whole && ((((uintptr_t)other | (uintptr_t)out) & 15) == 0);
#pragma unroll
  for (int i = 0; i < kRelPer; i += 4) {
    if (wide) {
      *reinterpret_cast<int4*>(r + i) = __ldg(reinterpret_cast<const int4*>(erow + j0 + i));
      *reinterpret_cast<int4*>(c + i) = __ldg(reinterpret_cast<const int4*>(other + j0 + i));
    } else {
#pragma unroll
      for (int k = i; k < i + 4; ++k) {
        r[k] = j0 + k < E ? __ldg(erow + j0 + k) : -1;
        c[k] = j0 + k < E ? __ldg(other + j0 + k) : 0;
      }
    }
  }
  D d[kRelPer];
  bool ahead[kRelPer];
#pragma unroll
  for (int i = 0; i < kRelPer; ++i) {
    const bool in = r[i] >= 0;
    const P to = src_pos ? (in ? __ldg(src_pos + c[i]) : P(0)) : (P)c[i], from = dst_pos ? (in ? __ldg(dst_pos + r[i]) : P(0)) : (P)r[i];
    d[i] = distance<D, P>(from, to, limits.both, ahead[i]);
  }
  buckets_of<D, kRelPer>(b, d, ahead, s_at, limits);
#pragma unroll
  for (int i = 0; i < kRelPer; ++i)
    if (r[i] < 0) b[i] = -1;
#pragma unroll
  for (int i = 0; i < kRelPer; i += 4) {
    if (wide) *reinterpret_cast<int4*>(out + j0 + i) = *reinterpret_cast<int4*>(b + i);
    else
#pragma unroll
      for (int k = i; k < i + 4; ++k)
        if (j0 + k < E) out[j0 + k] = b[k];
  }
}

constexpr int kRelTile = 256 * kRelPer;
constexpr int kRelLong = 512;   // chunks from this length on are taken by the whole block
// A warp takes up to 32 chunks, one per lane to find their ends and the positions of their nodes, then four at a time with a lane per
// position.  The block comes back to its long chunks (rows that were not cut) together.
template <typename I, typename D>
__global__ void __launch_bounds__(256)
relative_chunks_kernel(const I* __restrict__ row, const I* __restrict__ indptr, long long C, long long E, int per_warp,
                       const I* __restrict__ indices, const I* __restrict__ dst_pos, const I* __restrict__ src_pos,
                       const __grid_constant__ Limits<D> limits, int32_t* __restrict__ out) {
  constexpr int U = 4;
  __shared__ Shared<D> s_at;
  __shared__ unsigned s_lo[256], s_hi[256];   // fewer than 2^31 positions
  __shared__ I s_node[256];
  __shared__ int s_long[8];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const long long c0 = ((long long)blockIdx.x * 8 + w) * per_warp, mine = c0 + lane;
  unsigned s = 0, e = 0;
  I from = I(0);
  if (lane < per_warp && mine < C) {
    s = (unsigned)indptr[mine];
    e = (unsigned)indptr[mine + 1];
    const I r = row[mine];
    from = dst_pos ? dst_pos[r] : r;
  }
  const bool is_long = e > s && e - s >= kRelLong;
  const unsigned long_lanes = __ballot_sync(kFull, is_long);
  if (is_long) {
    const int at = w * 32 + __popc(long_lanes & ((1u << lane) - 1));
    s_lo[at] = s; s_hi[at] = e; s_node[at] = from;
    e = s;
  }
  if (lane == 0) s_long[w] = __popc(long_lanes);
  load_limits(s_at, limits);   // after the chunks' loads were asked for; its barriers are s_lo's too
  const auto some = [&](const unsigned (&p)[U], const bool (&in)[U], const I (&at)[U]) {
    I to[U];
    D d[U];
    bool ahead[U];
    int b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) to[u] = in[u] ? __ldg(indices + p[u]) : I(0);
    if (src_pos) {
#pragma unroll
      for (int u = 0; u < U; ++u) to[u] = in[u] ? __ldg(src_pos + to[u]) : I(0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) d[u] = distance<D, I>(at[u], to[u], limits.both, ahead[u]);
    buckets_of<D, U>(b, d, ahead, s_at, limits);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (in[u]) out[p[u]] = b[u];
  };
  for (int k = 0; k < per_warp && c0 + k < C; k += U) {
    unsigned p[U], end[U];
    I at[U];
    bool in[U], more = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = __shfl_sync(kFull, s, k + u) + lane;
      end[u] = __shfl_sync(kFull, e, k + u);
      at[u] = __shfl_sync(kFull, from, k + u);
    }
    while (more) {
      more = false;
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = p[u] < end[u];
      some(p, in, at);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        p[u] += 32;
        more = more || p[u] < end[u];
      }
      more = __any_sync(kFull, more);
    }
  }
  for (int v = 0; v < 8; ++v)
    for (int k = 0; k < s_long[v]; ++k) {
      const unsigned hi = s_hi[v * 32 + k];
      I at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) at[u] = s_node[v * 32 + k];
      for (unsigned q = s_lo[v * 32 + k]; q < hi; q += 256 * U) {
        unsigned p[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          p[u] = q + u * 256 + tid;
          in[u] = p[u] < hi;
        }
        some(p, in, at);
      }
    }
  // positions of no chunk: before the first one and after the last one
  if (blockIdx.x == 0 || blockIdx.x == gridDim.x - 1) {
    const long long base = (long long)indptr[0], last = (long long)indptr[C], end = last < base ? base : last;
    if (blockIdx.x == 0)
      for (long long p = tid; p < base && p < E; p += 256) out[p] = -1;
    if (blockIdx.x == gridDim.x - 1)
      for (long long p = end + tid; p < E; p += 256) out[p] = -1;
  }
}

template <typename P, typename D>
inline int fill_limits(Limits<D>& l, const int64_t* limits, int n_limits, int both) {
  l.n = 0;
  l.all = n_limits;
  l.both = both != 0;
  for (int i = 0; i < n_limits; ++i) {
    if (limits[i] < (i ? limits[i - 1] : 0)) return GRAPHOP_ERR_INVALID_ARGUMENT;
    if (sizeof(D) == 8 || limits[i] <= 0xffffffffll) l.at[l.n++] = (D)limits[i];
  }
  l.top = 1;
  while (2 * l.top <= l.n) l.top *= 2;
  l.near = l.n == 0 ? 0 : l.at[l.n - 1] <= (D)kNear ? (int)l.at[l.n - 1] : -1;
  return GRAPHOP_OK;
}
inline int relative_check(long long C, long long E, const int64_t* limits, int n_limits) {
  GK_TRY(check_sizes(C, E, 0, 0, 1, 1));
  if (n_limits < 0 || (n_limits && !limits)) return GRAPHOP_ERR_INVALID_ARGUMENT;
  return n_limits > kMostLimits ? GRAPHOP_ERR_UNSUPPORTED : GRAPHOP_OK;
}
// f(a value of the type of the distances)
template <typename I, class F>
inline int with_distance(const int64_t* limits, int n_limits, F&& f) {
  if constexpr (sizeof(I) == 8)
    if (n_limits > 0 && limits[n_limits - 1] > 0xffffffffll) return f(0ull);
  return f(0u);
}

template <typename I>
inline int relative_chunks(const I* row, const I* indptr, const I* indices, long long C, long long E, const I* dst_pos, const I* src_pos,
                           const int64_t* limits, int n_limits, int both, int32_t* out, cudaStream_t st) {
  GK_TRY(relative_check(C, E, limits, n_limits));
  return with_distance<I>(limits, n_limits, [&](auto zero) -> int {
    using D = decltype(zero);
    Limits<D> l;
    GK_TRY((fill_limits<I, D>(l, limits, n_limits, both)));
    if (E == 0) return GRAPHOP_OK;
    if (!row || !indptr || !indices || !out) return GRAPHOP_ERR_INVALID_ARGUMENT;
    // as many chunks per warp as leave the chip full
    long long per_warp = C / (148 * 32);
    per_warp = per_warp < 1 ? 1 : per_warp > 32 ? 32 : per_warp;
    const long long blocks = (C + 8 * per_warp - 1) / (8 * per_warp);
    relative_chunks_kernel<I, D><<<(unsigned)(blocks ? blocks : 1), 256, 0, st>>>(row, indptr, C, E, (int)per_warp, indices, dst_pos, src_pos,
                                                                                 l, out);
    GK_LAUNCHED("relative_buckets");
    return GRAPHOP_OK;
  });
}
template <typename P>
inline int relative_planned(const graphop_plan_t* plan, const P* dst_pos, const P* src_pos, const int64_t* limits, int n_limits, int both,
                            int32_t* out, cudaStream_t st) {
  if (!plan) return GRAPHOP_ERR_INVALID_ARGUMENT;
  GK_TRY(relative_check(plan->n_chunks, plan->n_edges, limits, n_limits));
  return with_distance<P>(limits, n_limits, [&](auto zero) -> int {
    using D = decltype(zero);
    Limits<D> l;
    GK_TRY((fill_limits<P, D>(l, limits, n_limits, both)));
    const long long E = plan->n_edges;
    if (E == 0) return GRAPHOP_OK;
    if (!plan->erow || !plan->other || !out) return GRAPHOP_ERR_INVALID_ARGUMENT;
    relative_planned_kernel<P, D><<<(unsigned)((E + kRelTile - 1) / kRelTile), 256, 0, st>>>(plan->erow, plan->other, E, dst_pos, src_pos, l,
                                                                                            out);
    GK_LAUNCHED("relative_buckets");
    return GRAPHOP_OK;
  });
}

}  // namespace gk
