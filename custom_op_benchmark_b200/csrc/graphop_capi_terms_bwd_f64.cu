// C ABI entry points of the attention layers with learned score terms, backward, f64 element type.
#include "graphop_capi_terms_impl.cuh"
GRAPHOP_DEFINE_TERMS_BACKWARD(f64_i32, double, double, int32_t)
GRAPHOP_DEFINE_TERMS_BACKWARD(f64_i64, double, double, int64_t)
GRAPHOP_DEFINE_TERMS_BACKWARD_PLANNED(f64, double, double)
