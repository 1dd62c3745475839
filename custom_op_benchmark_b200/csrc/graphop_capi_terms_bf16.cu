// C ABI entry points of the attention layers with learned score terms, bf16 element type.
#include "graphop_capi_terms_impl.cuh"
GRAPHOP_DEFINE_TERMS(bf16_i32, uint16_t, __nv_bfloat16, int32_t)
GRAPHOP_DEFINE_TERMS(bf16_i64, uint16_t, __nv_bfloat16, int64_t)
GRAPHOP_DEFINE_TERMS_PLANNED(bf16, uint16_t, __nv_bfloat16)
