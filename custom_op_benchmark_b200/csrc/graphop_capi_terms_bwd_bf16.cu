// C ABI entry points of the attention layers with learned score terms, backward, bf16 element type.
#include "gk_terms_banded.cuh"
#include "graphop_capi_terms_impl.cuh"
GRAPHOP_DEFINE_TERMS_BACKWARD(bf16_i32, uint16_t, __nv_bfloat16, int32_t)
GRAPHOP_DEFINE_TERMS_BACKWARD(bf16_i64, uint16_t, __nv_bfloat16, int64_t)
GRAPHOP_DEFINE_TERMS_BACKWARD_PLANNED(bf16, uint16_t, __nv_bfloat16)
