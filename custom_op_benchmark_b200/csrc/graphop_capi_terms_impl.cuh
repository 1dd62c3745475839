// Expands to the extern "C" entry points of include/graphop_terms.h for one element type.
#pragma once
#include "../../include/graphop_terms.h"
#include "gk_terms.cuh"

#define GK_CH(I, row, indptr, eid, indices, C, E) gk::FromChunks<I>{row, indptr, eid, indices, (long long)(C), (long long)(E)}
#define GK_ST (cudaStream_t)stream
#define GK_TERMS(T, diff, q, k, v, table, lam, bucket, buckets, E) \
  gk::TermsCall<T>{diff, (const T*)(q), (const T*)(k), (const T*)(v), (const T*)(table), (const T*)(lam), bucket, buckets, scale, \
                   (long long)(E), n_dst, n_src, H, D}

#define GRAPHOP_DEFINE_TERMS_FORWARD(SUF, CT, T, I)                                                                                         \
  extern "C" int graphop_attention_bucket_forward_##SUF(                                                                             \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const CT* q, const CT* k, const CT* v,                      \
      const int32_t* bucket, const CT* table, int n_buckets, double scale, CT* o, void* sums, void* lse, int64_t n_edges,           \
      int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb, graphop_stream_t stream) {                                   \
    return gk::terms_forward<T>(GK_CH(I, row, indptr, (const I*)nullptr, indices, n_chunks, n_edges), n_chunks,                      \
                                GK_TERMS(T, false, q, k, v, table, nullptr, bucket, n_buckets, n_edges), (T*)o, sums, lse,           \
                                ws, wsb, GK_ST);                                                                                     \
  }                                                                                                                                  \
  extern "C" int graphop_attention_diff_forward_##SUF(                                                                               \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const CT* q, const CT* k, const CT* v, const CT* lam,       \
      const int32_t* bucket, const CT* table, int n_buckets, double scale, CT* o, void* sums, void* lse, int64_t n_edges,             \
      int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb, graphop_stream_t stream) {                                   \
    return gk::terms_forward<T>(GK_CH(I, row, indptr, (const I*)nullptr, indices, n_chunks, n_edges), n_chunks,                      \
                                GK_TERMS(T, true, q, k, v, table, lam, bucket, n_buckets, n_edges), (T*)o, sums, lse, ws, wsb,  \
                                GK_ST);                                                                                              \
  }

#define GRAPHOP_DEFINE_TERMS_BACKWARD(SUF, CT, T, I)                                                                                 \
  extern "C" int graphop_attention_bucket_backward_##SUF(                                                                            \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const I* col, const I* indptr_t, const I* eid_t,            \
      const I* indices_t, int64_t n_chunks_t, const CT* q, const CT* k, const CT* v, const int32_t* bucket, const CT* table,         \
      int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv, CT* d_table,                 \
      int64_t n_edges, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb, graphop_stream_t stream) {                  \
    return gk::terms_backward<T>(GK_CH(I, row, indptr, (const I*)nullptr, indices, n_chunks, n_edges),                               \
                                 GK_CH(I, col, indptr_t, eid_t, indices_t, n_chunks_t, n_edges), eid_t != nullptr, n_chunks,         \
                                 n_chunks_t, GK_TERMS(T, false, q, k, v, table, nullptr, bucket, n_buckets, n_edges), sums,          \
                                 lse, (const T*)d_o, (T*)dq, (T*)dk, (T*)dv, (T*)d_table, (T*)nullptr, ws, wsb, GK_ST);              \
  }                                                                                                                                  \
  extern "C" int graphop_attention_diff_backward_##SUF(                                                                              \
      const I* row, const I* indptr, const I* indices, int64_t n_chunks, const I* col, const I* indptr_t, const I* eid_t,            \
      const I* indices_t, int64_t n_chunks_t, const CT* q, const CT* k, const CT* v, const CT* lam, const int32_t* bucket,           \
      const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv,         \
      CT* d_lam, CT* d_table, int64_t n_edges, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb,                     \
      graphop_stream_t stream) {                                                                                                     \
    return gk::terms_backward<T>(GK_CH(I, row, indptr, (const I*)nullptr, indices, n_chunks, n_edges),                               \
                                 GK_CH(I, col, indptr_t, eid_t, indices_t, n_chunks_t, n_edges), eid_t != nullptr, n_chunks,         \
                                 n_chunks_t, GK_TERMS(T, true, q, k, v, table, lam, bucket, n_buckets, n_edges), sums,               \
                                 lse, (const T*)d_o, (T*)dq, (T*)dk, (T*)dv, (T*)d_table, (T*)d_lam, ws, wsb, GK_ST);                \
  }

// The same on plans.
#define GK_PL(plan) gk::FromPlan{plan}
#define GK_PE(plan) ((plan) ? (plan)->n_edges : -1)
#define GK_PC(plan) ((plan) ? (plan)->n_chunks : -1)

#define GRAPHOP_DEFINE_TERMS_FORWARD_PLANNED(SUF, CT, T)                                                                                     \
  extern "C" int graphop_attention_bucket_forward_planned_##SUF(                                                                     \
      const graphop_plan_t* plan, const CT* q, const CT* k, const CT* v, const int32_t* bucket, const CT* table, int n_buckets,      \
      double scale, CT* o, void* sums, void* lse, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb,                  \
      graphop_stream_t stream) {                                                                                                     \
    return gk::terms_forward<T>(GK_PL(plan), GK_PC(plan),                                                                            \
                                GK_TERMS(T, false, q, k, v, table, nullptr, bucket, n_buckets, GK_PE(plan)), (T*)o, sums,            \
                                lse, ws, wsb, GK_ST);                                                                                \
  }                                                                                                                                  \
  extern "C" int graphop_attention_diff_forward_planned_##SUF(                                                                       \
      const graphop_plan_t* plan, const CT* q, const CT* k, const CT* v, const CT* lam, const int32_t* bucket, const CT* table,      \
      int n_buckets, double scale, CT* o, void* sums, void* lse, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb,    \
      graphop_stream_t stream) {                                                                                                     \
    return gk::terms_forward<T>(GK_PL(plan), GK_PC(plan),                                                                            \
                                GK_TERMS(T, true, q, k, v, table, lam, bucket, n_buckets, GK_PE(plan)), (T*)o, sums, lse, ws,   \
                                wsb, GK_ST);                                                                                         \
  }

#define GRAPHOP_DEFINE_TERMS_BACKWARD_PLANNED(SUF, CT, T)                                                                            \
  extern "C" int graphop_attention_bucket_backward_planned_##SUF(                                                                    \
      const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, const CT* q, const CT* k, const CT* v, const int32_t* bucket,      \
      const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq, CT* dk, CT* dv,             \
      CT* d_table, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb, graphop_stream_t stream) {                      \
    return gk::terms_backward<T>(GK_PL(plan_r), GK_PL(plan_t), plan_t && plan_t->eid, GK_PC(plan_r), GK_PC(plan_t),                  \
                                 GK_TERMS(T, false, q, k, v, table, nullptr, bucket, n_buckets, GK_PE(plan_r)), sums, lse,           \
                                 (const T*)d_o, (T*)dq, (T*)dk, (T*)dv, (T*)d_table, (T*)nullptr, ws, wsb, GK_ST);                   \
  }                                                                                                                                  \
  extern "C" int graphop_attention_diff_backward_planned_##SUF(                                                                      \
      const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, const CT* q, const CT* k, const CT* v, const CT* lam,              \
      const int32_t* bucket, const CT* table, int n_buckets, const void* sums, const void* lse, const CT* d_o, double scale, CT* dq,  \
      CT* dk, CT* dv, CT* d_lam, CT* d_table, int64_t n_dst, int64_t n_src, int H, int D, void* ws, size_t wsb,                      \
      graphop_stream_t stream) {                                                                                                     \
    return gk::terms_backward<T>(GK_PL(plan_r), GK_PL(plan_t), plan_t && plan_t->eid, GK_PC(plan_r), GK_PC(plan_t),                  \
                                 GK_TERMS(T, true, q, k, v, table, lam, bucket, n_buckets, GK_PE(plan_r)), sums, lse,                \
                                 (const T*)d_o, (T*)dq, (T*)dk, (T*)dv, (T*)d_table, (T*)d_lam, ws, wsb, GK_ST);                     \
  }
