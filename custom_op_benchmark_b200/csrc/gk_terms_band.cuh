// What the dense-band path of the layers with learned score terms (gk_terms_banded.cuh) takes, and when it is taken: shared by its
// launches and by the workspace's size.
#pragma once
#include "gk_band_tiles.cuh"
#include "gk_terms.cuh"

namespace gk {
namespace banded {

constexpr int kMostBandBuckets = 255;

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

}  // namespace banded
}  // namespace gk
