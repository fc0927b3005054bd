// Residual norm for fp32 storage: kernels and entry points of residual_norm.hpp.  The size query for all types is here.
#include "residual_norm.hpp"

extern "C" {

size_t lbn_residual_norm_bwd_workspace_bytes(int64_t size, int64_t width, int has_weight_grads, int64_t num_gate_grads,
                                             int elem_bytes)
{
  (void)elem_bytes;  // partial rows are fp32 whatever the storage type
  // what backward refuses needs nothing, and the plan takes whole gates of at least a column for granted
  if (size <= 0 || width <= 0 || num_gate_grads < 0 || (num_gate_grads > 0 && width % num_gate_grads != 0)) return 0;
  if (size > lbn::kRnMostFeatures || !lbn::drop_range_ok(size, width, 0)) return 0;
  return lbn::rn_bwd_plan(size, width, has_weight_grads, num_gate_grads).total();
}

LBN_RESIDUAL_NORM_ENTRIES(f32, float, float)

}  // extern "C"
