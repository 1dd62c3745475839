/*
 * graphop_terms: C ABI of the attention layers with learned score terms, in libgraphop_b200.so.
 *
 * The conventions are those of graphop_b200.h: device pointers of the current device, graph arguments (row, indptr, indices;
 * col, indptr_t, eid_t, indices_t of the transposed CSR), a 256-byte aligned workspace of the caller, work enqueued on `stream`,
 * a status code back, no synchronisation, the same bits on every run.  Names end in _<elem>_<index> (f32, f64, bf16; i32, i64) or, on
 * plans, in _planned_<elem>.  CT: uint16_t holds a bfloat16.
 *
 * Bias by buckets.  q (n_dst, H, D), k and v (n_src, H, D), bucket (n_edges) int32 by row-CSR position, table (n_buckets, H):
 *     score of position j and head h = scale * q[n, h].k[indices[j], h] + table[bucket[j], h]
 *     o (n_dst, H, D) = sum of softmax(score) * v;   lse (n_dst, H) = log of the softmax denominator, float (double for f64)
 * A position takes no part where bucket[j] is not in 0 .. n_buckets - 1 or its entry of the table is at most -1e38 (-inf, a type's
 * lowest value): nothing is read outside the table, and what lies in the position's rows does not matter.  A node of which nothing
 * takes part has o = 0, lse = -inf and no gradient.
 *
 * Differential attention.  H pairs of maps: q (n_dst, 2H, D), k (n_src, 2H, D), v (n_src, H, 2D), lam (H); with n_buckets > 0 the
 * bias above with table (n_buckets, 2H), else bucket and table are null:
 *     o (n_dst, H, 2D) = o1 - lam[h] * o2, o1 and o2 the softmax sums of v under the maps 2h and 2h + 1;   lse (n_dst, 2H)
 *
 * sums, for the backward (null where none follows): o before it is rounded, (n_dst, H, D), or o1 and o2, (n_dst, H, 2, 2D), as float
 * (double for f64).  Without maps, and where the element type is float or double, o itself serves.
 *
 * Backward: the transposed CSR must carry eid_t (the row-CSR position of each of its positions); without it
 * GRAPHOP_ERR_INVALID_ARGUMENT.  Gradients of table and lam have the element type and are summed in 32 bits and more.
 *
 * Shapes (else GRAPHOP_ERR_UNSUPPORTED): D * sizeof(elem) a power-of-two multiple of 16 bytes, a node's row of v at most 4 KiB,
 * n_buckets at most 16384, node tensors 16-byte aligned.  lse is aligned to a node's one head (2 * sizeof(float or double) for
 * the differential layer).
 */
#ifndef GRAPHOP_TERMS_H
#define GRAPHOP_TERMS_H
#include "graphop_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
  GRAPHOP_TERMS_BUCKET_FWD = 0, GRAPHOP_TERMS_BUCKET_BWD = 1, GRAPHOP_TERMS_DIFF_FWD = 2, GRAPHOP_TERMS_DIFF_BWD = 3
};

/* Bytes of workspace of one call.  n_nodes: the larger of n_dst and n_src; H, D, n_buckets as in the call. */
size_t graphop_terms_workspace_bytes(int op, int64_t n_edges, int64_t n_nodes, int H, int D, int n_buckets, int elem_bytes,
                                     int index_bytes);
/*
 * The same of one call on plans (plan_t: a backward's second one, else null).  Calls on a dense band run on the tensor cores where all of this
 * holds: bf16; 64 features of v a head; at most 255 buckets; no more node rows than the plan has nodes; a mean of at least a neighbour
 * per 16 columns of its span, rounded up to 64, in the plan, or in both plans of a backward; sums 32-byte aligned; a workspace of this
 * size.  It is more than the size above where a narrow band's tiles need it, for bucket ids and three bytes of score gradient per tile
 * element, head and map; with that size alone, and in every other case, a call runs the same kernels as on chunk tables.
 * On the tensor cores probabilities and score gradients are rounded to bf16 before the products with v, k, q and d_o (the
 * forward of two maps adds what that leaves off), in the other kernels they are not.
 */
size_t graphop_terms_workspace_bytes_planned(int op, const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, int64_t n_dst,
                                             int64_t n_src, int H, int D, int n_buckets, int elem_bytes);

#define GRAPHOP_DECLARE_TERMS(SUF, CT, I)                                                                                            \
  int graphop_attention_bucket_forward_##SUF(const I* row, const I* indptr, const I* indices, int64_t n_chunks, const CT* q,         \
                                             const CT* k, const CT* v, const int32_t* bucket, const CT* table, int n_buckets,        \
                                             double scale, CT* o, void* sums, void* lse, int64_t n_edges, int64_t n_dst,             \
                                             int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes,                   \
                                             graphop_stream_t stream);                                                               \
  int graphop_attention_bucket_backward_##SUF(                                                                                       \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const I* col, const I* indptr_t, const I* eid_t,            \
      const I* indices_t, int64_t n_chunks_t, const CT* q, const CT* k, const CT* v, const int32_t* bucket, const CT* table,         \
      int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv, CT* d_table,                 \
      int64_t n_edges, int64_t n_dst, int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes,                          \
      graphop_stream_t stream);                                                                                                      \
  int graphop_attention_diff_forward_##SUF(const I* row, const I* indptr, const I* indices, int64_t n_chunks, const CT* q,           \
                                           const CT* k, const CT* v, const CT* lam, const int32_t* bucket, const CT* table,          \
                                           int n_buckets, double scale, CT* o, void* sums, void* lse, int64_t n_edges,                \
                                           int64_t n_dst, int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes,      \
                                           graphop_stream_t stream);                                                                 \
  int graphop_attention_diff_backward_##SUF(                                                                                         \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const I* col, const I* indptr_t, const I* eid_t,            \
      const I* indices_t, int64_t n_chunks_t, const CT* q, const CT* k, const CT* v, const CT* lam, const int32_t* bucket,           \
      const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv,         \
      CT* d_lam, CT* d_table, int64_t n_edges, int64_t n_dst, int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes,  \
      graphop_stream_t stream);

#define GRAPHOP_DECLARE_TERMS_PLANNED(SUF, CT)                                                                                       \
  int graphop_attention_bucket_forward_planned_##SUF(const graphop_plan_t* plan, const CT* q, const CT* k, const CT* v,              \
                                                     const int32_t* bucket, const CT* table, int n_buckets, double scale, CT* o,     \
                                                     void* sums, void* lse, int64_t n_dst, int64_t n_src, int H, int D, void* workspace,         \
                                                     size_t workspace_bytes, graphop_stream_t stream);                               \
  int graphop_attention_bucket_backward_planned_##SUF(                                                                               \
      const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, const CT* q, const CT* k, const CT* v, const int32_t* bucket,      \
      const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv,             \
      CT* d_table, int64_t n_dst, int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes, graphop_stream_t stream);    \
  int graphop_attention_diff_forward_planned_##SUF(const graphop_plan_t* plan, const CT* q, const CT* k, const CT* v,                \
                                                   const CT* lam, const int32_t* bucket, const CT* table, int n_buckets,             \
                                                   double scale, CT* o, void* sums, void* lse, int64_t n_dst, int64_t n_src, int H,   \
                                                   int D, void* workspace, size_t workspace_bytes, graphop_stream_t stream);         \
  int graphop_attention_diff_backward_planned_##SUF(                                                                                 \
      const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, const CT* q, const CT* k, const CT* v, const CT* lam,              \
      const int32_t* bucket, const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq,  \
      CT* dk, CT* dv, CT* d_lam, CT* d_table, int64_t n_dst, int64_t n_src, int H, int D, void* workspace, size_t workspace_bytes,   \
      graphop_stream_t stream);

GRAPHOP_DECLARE_TERMS(f32_i32, float, int32_t)
GRAPHOP_DECLARE_TERMS(f32_i64, float, int64_t)
GRAPHOP_DECLARE_TERMS(f64_i32, double, int32_t)
GRAPHOP_DECLARE_TERMS(f64_i64, double, int64_t)
GRAPHOP_DECLARE_TERMS(bf16_i32, uint16_t, int32_t)
GRAPHOP_DECLARE_TERMS(bf16_i64, uint16_t, int64_t)
GRAPHOP_DECLARE_TERMS_PLANNED(f32, float)
GRAPHOP_DECLARE_TERMS_PLANNED(f64, double)
GRAPHOP_DECLARE_TERMS_PLANNED(bf16, uint16_t)

/*
 * bucket (n_edges) int32, by row-CSR position: with x = src_pos[indices[j]] - dst_pos[node] (positions of the index type; null: the
 * nodes' own numbers), the number of `limits` (HOST array, ascending, none negative) that are at most max(-x, 0) or, both != 0, |x|,
 * plus n_limits + 1 where x > 0.  -1 where no chunk covers the position.  n_limits at most 1023, else GRAPHOP_ERR_UNSUPPORTED.
 */
int graphop_relative_buckets_i32(const int32_t* row, const int32_t* indptr, const int32_t* indices, int64_t n_chunks,
                                 const int32_t* dst_pos, const int32_t* src_pos, const int64_t* limits, int n_limits, int both,
                                 int32_t* bucket, int64_t n_edges, graphop_stream_t stream);
int graphop_relative_buckets_i64(const int64_t* row, const int64_t* indptr, const int64_t* indices, int64_t n_chunks,
                                 const int64_t* dst_pos, const int64_t* src_pos, const int64_t* limits, int n_limits, int both,
                                 int32_t* bucket, int64_t n_edges, graphop_stream_t stream);
int graphop_relative_buckets_planned_i32(const graphop_plan_t* plan, const int32_t* dst_pos, const int32_t* src_pos,
                                         const int64_t* limits, int n_limits, int both, int32_t* bucket, graphop_stream_t stream);
int graphop_relative_buckets_planned_i64(const graphop_plan_t* plan, const int64_t* dst_pos, const int64_t* src_pos,
                                         const int64_t* limits, int n_limits, int both, int32_t* bucket, graphop_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* GRAPHOP_TERMS_H */
