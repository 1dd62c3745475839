// C ABI entry points of the attention layers with learned score terms, forward, f32 element type.
#include "graphop_capi_terms_impl.cuh"
GRAPHOP_DEFINE_TERMS_FORWARD(f32_i32, float, float, int32_t)
GRAPHOP_DEFINE_TERMS_FORWARD(f32_i64, float, float, int64_t)
GRAPHOP_DEFINE_TERMS_FORWARD_PLANNED(f32, float, float)
