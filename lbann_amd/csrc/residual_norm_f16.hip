// Residual norm for IEEE binary16 storage: kernels and entry points of residual_norm.hpp.
#include "residual_norm.hpp"

extern "C" {

LBN_RESIDUAL_NORM_ENTRIES(f16, void, lbn::f16_t)

}  // extern "C"
