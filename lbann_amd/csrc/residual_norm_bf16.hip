// Residual norm for bfloat16 storage: kernels and entry points of residual_norm.hpp.
#include "residual_norm.hpp"

extern "C" {

LBN_RESIDUAL_NORM_ENTRIES(bf16, void, lbn::bf16_t)

}  // extern "C"
