// What the dense-band path of the layers with learned score terms (gk_terms_banded.cuh) takes, and when it is taken: shared by its
// launches and by the workspace's size.  And its sums by bucket.
#pragma once
#include "gk_band_tiles.cuh"
#include "gk_terms.cuh"

namespace gk {
namespace banded {

constexpr int kMostBandBuckets = 255;
// What a tile says of itself: a product was not finite, and it is done again edge by edge; a wait ran out, and its results are NaN.
constexpr int kTileAgain = 1, kTileLost = 2;

// A block of the sums by bucket has a table per thread; as many blocks as share the SMs' memory, a piece or more for every thread.
struct BandSumShape { int threads, smem, blocks; };
inline BandSumShape band_sum_shape(long long elements, int buckets, int columns) {
  BandSumShape s;
  s.threads = 128;
  while (s.threads > 32 && (buckets + 1) * s.threads * (int)sizeof(float) > 56 * 1024) s.threads >>= 1;
  s.smem = (buckets + 1) * s.threads * (int)sizeof(float);
  long long per_sm = 200 * 1024 / (s.smem + 1024);
  per_sm = per_sm > 10 ? 10 : per_sm;
  long long blocks = per_sm * 148 / columns, most = elements / 8 / s.threads + 1;
  blocks = blocks < 1 ? 1 : blocks < most ? blocks : most;
  s.blocks = (int)blocks;
  return s;
}

inline int band_pitch(const graphop_plan_t* plan) { return (plan->band_span + kKeys - 1) / kKeys * kKeys; }
inline long long band_tiles_of(long long n) { return (n + kTileM - 1) / kTileM; }
// The tiles compute `pitch` columns for every node, the walkers its own neighbours.  Time of the tiles over that of the walkers,
// forward and backward together, bands of 1 x 300 to 8 x 40000 nodes (and blocks of that many nodes, 16384 in all), 1 and 8 heads, one
// and two maps, with a bias and without: 9 neighbours (pitch 192) 0.66 to 1.50, 17 neighbours (192) 0.54 to 1.04, 25 (192) 0.37 to
// 0.89, 129 (256) 0.12 to 0.70; 5 neighbours 0.70 to 2.1, 3 neighbours up to 2.7; blocks of 4 1.2 to 1.6, of 8 (pitch 128) 0.87 to 1.2,
// of 16 0.49 to 0.81.  They are even at about a neighbour per 16 columns.
inline bool band_pays(const graphop_plan_t* plan) { return plan->n_edges * 16 >= plan->n_nodes * (long long)band_pitch(plan); }
inline bool band_plan_ok(const graphop_plan_t* plan, long long n, int H) {
  return (plan->flags & GRAPHOP_PLAN_DENSE_BAND) && plan->band_span > 0 && plan->band_span <= kSpan && plan->node_lo && plan->node_deg &&
         plan->node_first && plan->tile_lo && n >= 1 && n <= plan->n_nodes && H <= 65535 && band_pays(plan);
}
// Heads of 64 features of v, up to 255 buckets, in bfloat16, on bands that pay.  plan_t: null for a forward.
inline bool band_serves(const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, long long n_dst, long long n_src, int H, int row_d,
                        int buckets) {
  return row_d == kD && buckets <= kMostBandBuckets && n_src >= 1 && band_plan_ok(plan_r, n_dst, H) &&
         (!plan_t || band_plan_ok(plan_t, n_src, H));
}

// A call's part of the workspace.
struct BandRoom {
  unsigned char *ids = nullptr, *ids_t = nullptr;   // of the tiles of either orientation
  int *dirty = nullptr, *dirty_t = nullptr;
  float2* stat = nullptr;
  float* t2 = nullptr;
  unsigned short* g = nullptr;                      // score gradients, upper and lower plane
  unsigned char* g_low = nullptr;
  double* partial = nullptr;
  long long elements = 0;                           // of the destination's tiles
  BandSumShape sum{};
  size_t bytes = 0;                                 // of all of it
};
inline BandRoom band_room_forward(Arena& ar, const graphop_plan_t* plan, long long n_dst, int H, int buckets) {
  BandRoom b;
  const long long tiles = band_tiles_of(n_dst);
  if (buckets) b.ids = (unsigned char*)ar.take((size_t)tiles * band_pitch(plan) * kTileM);
  b.dirty = (int*)ar.take((size_t)tiles * H * sizeof(int));
  b.bytes = ar.used;
  return b;
}
// Leaves room for the sums of lam's gradient behind what it took.
inline BandRoom band_room_backward(Arena& ar, const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, long long n_dst, long long n_src,
                                   int H, int maps, int buckets) {
  BandRoom b;
  const long long tiles = band_tiles_of(n_dst), tiles_t = band_tiles_of(n_src);
  const int columns = H * maps;
  b.elements = tiles * band_pitch(plan_r) * kTileM;
  b.stat = (float2*)ar.take((size_t)n_dst * columns * sizeof(float2));
  b.dirty = (int*)ar.take((size_t)tiles * H * sizeof(int));
  b.dirty_t = (int*)ar.take((size_t)tiles_t * H * sizeof(int));
  if (maps == 2) b.t2 = (float*)ar.take((size_t)n_dst * H * sizeof(float));
  if (buckets) {
    b.sum = band_sum_shape(b.elements, buckets, columns);
    b.ids = (unsigned char*)ar.take((size_t)b.elements);
    b.ids_t = (unsigned char*)ar.take((size_t)tiles_t * band_pitch(plan_t) * kTileM);
    b.g = (unsigned short*)ar.take((size_t)columns * b.elements * 2);
    b.g_low = (unsigned char*)ar.take((size_t)columns * b.elements);
    b.partial = (double*)ar.take((size_t)b.sum.blocks * buckets * columns * sizeof(double));
  }
  const size_t used = ar.used;
  if (maps == 2) ar.take(bucket_sum_bytes(n_dst, H, 1, 4));
  b.bytes = ar.used;
  ar.used = used;
  return b;
}

// ---------------------------------------------------------------------------------------------------------
// dT: sums of g by bucket, over the tiles' elements in the threads' order
// ---------------------------------------------------------------------------------------------------------
// grid: (blocks, H * maps).  A thread takes 8 elements at a time, so that a warp's loads are whole lines, and asks for kAhead such
// pieces at once; they go into a table of its own, cell b of thread t at b * NT + t: a warp's 32 cells lie in 32 banks.  An element
// that takes no part has a gradient of zero and goes to one cell more.  Bound by its instructions, about ten per element (with a test
// per element and the table's stride not known, 14), then by reading the gradients: 6.3M elements of 8 heads 43 us (3.6 TB/s; 28 when
// the gradients were bfloat16).
template <int NT>
__global__ void __launch_bounds__(NT)
band_bucket_sum_kernel(const unsigned char* __restrict__ ids, const unsigned short* __restrict__ g, const unsigned char* __restrict__ g_low,
                       const int* __restrict__ dirty, long long elements, int tiles, int buckets, int columns, int maps,
                       double* __restrict__ partial) {
  extern __shared__ float cells[];
  constexpr int kAhead = 4;
  const int tid = threadIdx.x, column = blockIdx.y;
  const long long pieces = elements / 8, stride = (long long)gridDim.x * NT;
  const uint2* idp = reinterpret_cast<const uint2*>(ids);
  const uint4* src = reinterpret_cast<const uint4*>(g + (size_t)column * elements);
  const uint2* src_low = reinterpret_cast<const uint2*>(g_low + (size_t)column * elements);
  float* mine = cells + tid;
  for (int b = 0; b <= buckets; ++b) mine[b * NT] = 0.f;
  const unsigned none = (unsigned)buckets;
  for (long long i = (long long)blockIdx.x * NT + tid; i < pieces; i += kAhead * stride) {
    uint2 id[kAhead];
    uint4 w[kAhead];
    uint2 l[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) id[k] = i + k * stride < pieces ? __ldg(idp + i + k * stride) : make_uint2(0xffffffffu, 0xffffffffu);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if ((id[k].x & id[k].y) != 0xffffffffu) {   // else nothing takes part, and nothing was stored
        w[k] = __ldg(src + i + k * stride);
        l[k] = __ldg(src_low + i + k * stride);
      }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if ((id[k].x & id[k].y) == 0xffffffffu) continue;
      const unsigned v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned b = min(((j < 4 ? id[k].x : id[k].y) >> (8 * (j & 3))) & 255u, none);
        // bytes of the float, from the highest: two of the upper plane, one of the lower, zero
        const unsigned high = (j & 1) ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16, next = j < 4 ? l[k].x : l[k].y;
        mine[b * NT] += __uint_as_float(__byte_perm(high, next, 0x3200 | ((4 + (j & 3)) << 4)));
      }
    }
  }
  // a lost tile's score gradients were not all written: the sums of its head are not known
  bool lost = false;
  if (blockIdx.x == 0)
    for (int i = tid; i < tiles; i += NT) lost = lost || __ldg(dirty + (size_t)(column / maps) * tiles + i) == kTileLost;
  lost = __syncthreads_or(lost);
  const int warp = tid >> 5, lane = tid & 31;
  for (int b = warp; b < buckets; b += NT / 32) {   // a bucket per warp: the threads' cells in order, by halves
    double s = 0;
#pragma unroll
    for (int t = 0; t < NT; t += 32) s += (double)cells[b * NT + t + lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (lane == 0) partial[((size_t)blockIdx.x * buckets + b) * columns + column] = lost ? (double)NAN : s;
  }
}
template <typename T>
inline int run_band_bucket_sum(const BandRoom& r, int tiles, int buckets, int H, int maps, T* out, cudaStream_t st) {
  const int columns = H * maps;
  const auto launch = [&](auto kernel, std::atomic<bool> (&configured)[64]) -> int {
    GK_TRY(allow_smem(kernel, 56 * 1024, configured));
    kernel<<<dim3((unsigned)r.sum.blocks, (unsigned)columns), r.sum.threads, r.sum.smem, st>>>(r.ids, r.g, r.g_low, r.dirty, r.elements, tiles, buckets,
                                                                                             columns, maps, r.partial);
    GK_LAUNCHED("band_bucket_sum");
    return GRAPHOP_OK;
  };
  static std::atomic<bool> c128[64], c64[64], c32[64];
  if (r.sum.threads == 128) GK_TRY(launch(band_bucket_sum_kernel<128>, c128));
  else if (r.sum.threads == 64) GK_TRY(launch(band_bucket_sum_kernel<64>, c64));
  else GK_TRY(launch(band_bucket_sum_kernel<32>, c32));
  const int cells = buckets * columns;
  bucket_total_kernel<T><<<(cells + 7) / 8, 256, 0, st>>>(r.partial, r.sum.blocks, cells, 1.0, out);
  GK_LAUNCHED("bucket_total");
  return GRAPHOP_OK;
}

}  // namespace banded
}  // namespace gk
