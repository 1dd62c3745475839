// C ABI entry points of the attention layers with learned score terms, forward, f64 element type.
#include "graphop_capi_terms_impl.cuh"
GRAPHOP_DEFINE_TERMS_FORWARD(f64_i32, double, double, int32_t)
GRAPHOP_DEFINE_TERMS_FORWARD(f64_i64, double, double, int64_t)
GRAPHOP_DEFINE_TERMS_FORWARD_PLANNED(f64, double, double)
