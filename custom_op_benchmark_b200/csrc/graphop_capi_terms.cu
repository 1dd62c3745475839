// C ABI entry points of include/graphop_terms.h that do not depend on the element type: workspace sizes and the bucket of every edge.
#include "../../include/graphop_terms.h"
#include "gk_relative.cuh"
#include "gk_terms_band.cuh"

extern "C" size_t graphop_terms_workspace_bytes(int op, int64_t n_edges, int64_t n_nodes, int H, int D, int n_buckets, int elem_bytes,
                                                int index_bytes) {
  using namespace gk;
  if (n_edges < 0 || n_nodes < 0 || H < 1 || D < 1 || n_buckets < 0 || n_buckets > kMostBuckets) return 0;
  switch (op) {
    case GRAPHOP_TERMS_BUCKET_FWD:
    case GRAPHOP_TERMS_BUCKET_BWD:
      return terms_bytes(false, op == GRAPHOP_TERMS_BUCKET_BWD, n_edges, n_nodes, H, D, n_buckets, elem_bytes, index_bytes);
    case GRAPHOP_TERMS_DIFF_FWD:
    case GRAPHOP_TERMS_DIFF_BWD:
      return terms_bytes(true, op == GRAPHOP_TERMS_DIFF_BWD, n_edges, n_nodes, H, D, n_buckets, elem_bytes, index_bytes);
    default:
      return 0;
  }
}

extern "C" size_t graphop_terms_workspace_bytes_planned(int op, const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, int64_t n_dst,
                                                        int64_t n_src, int H, int D, int n_buckets, int elem_bytes) {
  using namespace gk;
  const bool diff = op == GRAPHOP_TERMS_DIFF_FWD || op == GRAPHOP_TERMS_DIFF_BWD;
  const bool backward = op == GRAPHOP_TERMS_BUCKET_BWD || op == GRAPHOP_TERMS_DIFF_BWD;
  if (!plan_r || (backward && !plan_t) || n_dst < 0 || n_src < 0) return 0;
  const size_t walkers = graphop_terms_workspace_bytes(op, plan_r->n_edges, n_dst > n_src ? n_dst : n_src, H, D, n_buckets, elem_bytes, 4);
  if (!walkers || elem_bytes != 2 ||
      !banded::band_serves(plan_r, backward ? plan_t : nullptr, n_dst, n_src, H, diff ? 2 * D : D, n_buckets))
    return walkers;
  Arena none(nullptr, 0);
  const size_t tiles = backward ? banded::band_room_backward(none, plan_r, plan_t, n_dst, n_src, H, diff ? 2 : 1, n_buckets).bytes
                                : banded::band_room_forward(none, plan_r, n_dst, H, n_buckets).bytes;
  return tiles > walkers ? tiles : walkers;
}

#define GRAPHOP_DEFINE_RELATIVE(SUF, I)                                                                                              \
  extern "C" int graphop_relative_buckets_##SUF(const I* row, const I* indptr, const I* indices, int64_t n_chunks, const I* dst_pos, \
                                                const I* src_pos, const int64_t* limits, int n_limits, int both, int32_t* bucket,    \
                                                int64_t n_edges, graphop_stream_t stream) {                                          \
    return gk::relative_chunks<I>(row, indptr, indices, n_chunks, n_edges, dst_pos, src_pos, limits, n_limits, both, bucket,         \
                                  (cudaStream_t)stream);                                                                             \
  }                                                                                                                                  \
  extern "C" int graphop_relative_buckets_planned_##SUF(const graphop_plan_t* plan, const I* dst_pos, const I* src_pos,              \
                                                        const int64_t* limits, int n_limits, int both, int32_t* bucket,              \
                                                        graphop_stream_t stream) {                                                   \
    return gk::relative_planned<I>(plan, dst_pos, src_pos, limits, n_limits, both, bucket, (cudaStream_t)stream);                    \
  }
GRAPHOP_DEFINE_RELATIVE(i32, int32_t)
GRAPHOP_DEFINE_RELATIVE(i64, int64_t)
