// Residual norm: what happens to a transformer's residual stream between two blocks, in one
// pass over the data (fp32, fp16 and bfloat16 storage, all arithmetic in fp32).  For column t,
// with o the block's output, r the residual stream, a and b scalars, g a gate,
//
//   u = N1(o),   v = keep ? u / q : 0,   h = a r + b g v,   y = N2(h),
//   N(v) = (v - mean) rsqrt(var + epsilon) scale + bias,
//
// where each of N1 (after the block) and N2 (before the next one) is no norm, the RMS norm (mean = 0,
// var = the mean of squares) or the layer norm.  y is formed from h before h is rounded to
// its storage type.  Backward, with xh and uh the normalised h and o:
//
//   p = dy scale2;      e  = dh + rstd2 (p - mean(p) - xh mean(p xh))
//   dr = a e;           dg = sum b e v;                du = keep ? b g e / q : 0
//   p1 = du scale1;     do = rstd1 (p1 - mean(p1) - uh mean(p1 uh))
//   dscale2 = sum dy xh, dbias2 = sum dy, dscale1 = sum du uh, dbias1 = sum du
//
// (the RMS norm drops mean(p)).  Sums over columns go through partial rows in the workspace,
// merged in a fixed order: no atomics, bitwise reproducible.  A gate column is shared by
// width / num_gates consecutive columns; a range of columns leaves one partial row per gate it
// meets, and range b and gate g use row b + g: ranges and gates are both contiguous, so b + g
// grows from one pair to the next and no row is used twice.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "residual_norm_rows.hpp"

namespace lbn {

// Sums the partial rows of ranges of columns: weight gradients over all ranges, a gate column
// over the ranges that meet it.
struct RnMergeArgs {
  const float* part[kGrads];
  float* out[kGrads];
  int64_t n, ranges, ld_dgate, num_gates, cols_per_gate, cols_per_range;
};

__global__ void __launch_bounds__(256)
rn_merge(RnMergeArgs a)
{
  const int64_t k = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (k >= a.n) return;
  for (int64_t item = blockIdx.y; item < kGradGate + a.num_gates; item += gridDim.y) {
    const int q = item < kGradGate ? static_cast<int>(item) : kGradGate;
    if (!a.out[q]) continue;
    if (q < kGradGate) {
      float s = 0.f;
      for (int64_t b = 0; b < a.ranges; ++b) s += a.part[q][b * a.n + k];
      a.out[q][k] = s;
    }
    else {
      const int64_t gate = item - kGradGate;
      const int64_t first = gate * a.cols_per_gate / a.cols_per_range;
      const int64_t last = ((gate + 1) * a.cols_per_gate - 1) / a.cols_per_range;
      float s = 0.f;
      for (int64_t b = first; b <= last; ++b) s += a.part[q][(b + gate) * a.n + k];
      a.out[q][gate * a.ld_dgate + k] = s;
    }
  }
}

// Ranges of columns that leave partial rows of their own.
static int64_t rn_ranges(int64_t width)
{
  const int64_t per = ceil_div(width, width < 256 ? width : 256);
  return ceil_div(width, per);
}

struct RnBwdPlan {
  int64_t ranges, cols_per_range;
  size_t sums_bytes, weight_bytes, gate_bytes;
  size_t total() const { return sums_bytes + weight_bytes + gate_bytes; }
};

static RnBwdPlan rn_bwd_plan(int64_t n, int64_t width, int weight_grads, int64_t gate_grads)
{
  RnBwdPlan p{};
  p.cols_per_range = ceil_div(width, rn_ranges(width));
  p.ranges = ceil_div(width, p.cols_per_range);
  auto round16 = [](int64_t b) { return static_cast<size_t>(ceil_div(b, 16) * 16); };
  p.sums_bytes = round16(width * 16);
  if (weight_grads) p.weight_bytes = round16(kGradGate * p.ranges * n * 4);
  if (gate_grads) p.gate_bytes = round16((p.ranges + gate_grads) * n * 4);
  return p;
}

static bool rn_ld_ok(const void* p, int64_t ld, int64_t height, int64_t width) { return !p || width <= 1 || ld >= height; }

static bool rn_norm_ok(int kind) { return kind >= kNormNone && kind <= kNormLayer; }

// How a column is shared: V units of eight entries per thread, a team of 16 lanes (`sub`) or of nw
// waves.  v == 0: it does not fit `max_v` units per thread of a full workgroup.
struct RnShape {
  int v, nw;
  bool sub;
  int threads() const { return sub || nw == 1 ? 256 : kWave * nw; }
  int teams() const { return sub ? 16 : (nw == 1 ? 4 : 1); }
};

static RnShape rn_shape(int64_t n, int max_v)
{
  const int64_t units = ceil_div(n, 8);
  if (units <= 16) return {1, 1, true};
  if (units <= 32) return {2, 1, true};
  for (int v = 1; v <= max_v; v *= 2)
    if (units <= 1024 * v) return {v, static_cast<int>(ceil_div(units, kWave * v)), false};
  return {0, 0, false};
}

template <typename T, int V, bool SUB>
static void rn_launch_fwd(hipStream_t st, const RnFwdArgs<T>& a, const RnShape& shape)
{
  const int64_t blocks = ceil_div(a.width, shape.teams());
  const int64_t resident = resident_blocks(rn_fwd_rows<T, V, SUB>, shape.threads());
  const int64_t grid = resident > 0 && blocks > resident ? resident : (blocks < (int64_t(1) << 30) ? blocks : (int64_t(1) << 30));
  hipLaunchKernelGGL((rn_fwd_rows<T, V, SUB>), dim3(static_cast<unsigned>(grid)), dim3(shape.threads()), 0, st, a, shape.nw);
}

template <typename T>
static int rn_fwd(lbn_stream_t stream, RnFwdArgs<T> a, int64_t num_gates, double keep_prob, uint64_t seed,
                  uint64_t offset, const uint64_t* step, int64_t column_offset)
{
  if (a.n < 0 || a.width < 0 || num_gates < 0 || column_offset < 0 || !rn_norm_ok(a.branch_norm) ||
      !rn_norm_ok(a.output_norm) || !drop_probability_ok(keep_prob))
    return LBN_ERR_INVALID_ARGUMENT;
  if (a.n == 0 || a.width == 0) return LBN_OK;
  if (!a.branch || (num_gates > 0) != (a.gate != nullptr) || (num_gates > 0 && a.width % num_gates != 0) ||
      (a.output_norm != kNormNone) != (a.y != nullptr) || (!a.y && !a.h))
    return LBN_ERR_INVALID_ARGUMENT;
  if (a.branch_norm == kNormNone && (a.branch_scale || a.branch_bias)) return LBN_ERR_INVALID_ARGUMENT;
  if (a.output_norm == kNormNone && (a.output_scale || a.output_bias)) return LBN_ERR_INVALID_ARGUMENT;
  if (!rn_ld_ok(a.branch, a.ld_branch, a.n, a.width) || !rn_ld_ok(a.residual, a.ld_residual, a.n, a.width) ||
      !rn_ld_ok(a.gate, a.ld_gate, a.n, num_gates) || !rn_ld_ok(a.h, a.ld_h, a.n, a.width) ||
      !rn_ld_ok(a.y, a.ld_y, a.n, a.width) || !rn_ld_ok(a.stats, a.ld_stats, 4, a.width))
    return LBN_ERR_INVALID_ARGUMENT;
  if (!drop_range_ok(a.n, a.width, column_offset)) return LBN_ERR_UNSUPPORTED;
  a.cols_per_gate = num_gates > 0 ? a.width / num_gates : a.width;
  a.drop = drop_args(keep_prob, seed, offset, step, column_offset);
  hipStream_t st = as_stream(stream);
  const RnShape shape = rn_shape(a.n, 2);
  switch (shape.v) {
  case 1: shape.sub ? rn_launch_fwd<T, 1, true>(st, a, shape) : rn_launch_fwd<T, 1, false>(st, a, shape); break;
  case 2: shape.sub ? rn_launch_fwd<T, 2, true>(st, a, shape) : rn_launch_fwd<T, 2, false>(st, a, shape); break;
  default: {
    const int64_t grid = a.width < (int64_t(1) << 30) ? a.width : (int64_t(1) << 30);
    hipLaunchKernelGGL((rn_fwd_long<T>), dim3(static_cast<unsigned>(grid)), dim3(kRnLongThreads), 0, st, a);
  }
  }
  return launch_status();
}

template <typename T>
static int rn_bwd(lbn_stream_t stream, RnBwdArgs<T> a, int64_t num_gates, double keep_prob, uint64_t seed,
                  uint64_t offset, const uint64_t* step, int64_t column_offset, float* dgate, int64_t ld_dgate,
                  float* const (&dweights)[kGradGate], void* workspace, size_t workspace_bytes)
{
  if (a.n < 0 || a.width < 0 || num_gates < 0 || column_offset < 0 || !rn_norm_ok(a.branch_norm) ||
      !rn_norm_ok(a.output_norm) || !drop_probability_ok(keep_prob))
    return LBN_ERR_INVALID_ARGUMENT;
  if (a.n == 0 || a.width == 0) return LBN_OK;
  const bool norm1 = a.branch_norm != kNormNone, norm2 = a.output_norm != kNormNone;
  if (!a.dbranch || (num_gates > 0) != (a.gate != nullptr) || (num_gates > 0 && a.width % num_gates != 0) ||
      norm2 != (a.dy != nullptr) || (norm2 && !a.h) || ((norm1 || norm2) && !a.stats) || (!norm2 && !a.dh) ||
      ((norm1 || dgate) && !a.branch) || (dgate && !a.gate))
    return LBN_ERR_INVALID_ARGUMENT;
  if (!norm1 && (a.branch_scale || a.branch_bias || dweights[kGradBranchScale] || dweights[kGradBranchBias]))
    return LBN_ERR_INVALID_ARGUMENT;
  if (!norm2 && (a.output_scale || dweights[kGradOutputScale] || dweights[kGradOutputBias]))
    return LBN_ERR_INVALID_ARGUMENT;
  if (!rn_ld_ok(a.branch, a.ld_branch, a.n, a.width) || !rn_ld_ok(a.h, a.ld_h, a.n, a.width) ||
      !rn_ld_ok(a.gate, a.ld_gate, a.n, num_gates) || !rn_ld_ok(dgate, ld_dgate, a.n, num_gates) ||
      !rn_ld_ok(a.stats, a.ld_stats, 4, a.width) || !rn_ld_ok(a.dy, a.ld_dy, a.n, a.width) ||
      !rn_ld_ok(a.dh, a.ld_dh, a.n, a.width) || !rn_ld_ok(a.dbranch, a.ld_dbranch, a.n, a.width) ||
      !rn_ld_ok(a.dresidual, a.ld_dresidual, a.n, a.width))
    return LBN_ERR_INVALID_ARGUMENT;
  if (!drop_range_ok(a.n, a.width, column_offset)) return LBN_ERR_UNSUPPORTED;
  if (!norm1 && !dgate) a.branch = nullptr;  // not needed, so not read
  a.cols_per_gate = num_gates > 0 ? a.width / num_gates : a.width;
  a.drop = drop_args(keep_prob, seed, offset, step, column_offset);
  bool weight_grads = false;
  for (float* d : dweights) weight_grads = weight_grads || d;
  const RnBwdPlan plan = rn_bwd_plan(a.n, a.width, weight_grads, dgate ? num_gates : 0);
  if (!workspace || workspace_bytes < plan.total() || !aligned16(workspace)) return LBN_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  a.sums = reinterpret_cast<float*>(ws);
  a.cols_per_range = plan.cols_per_range;
  float* weights = reinterpret_cast<float*>(ws + plan.sums_bytes);
  RnMergeArgs merge{};
  for (int q = 0; q < kGradGate; ++q) {
    a.part[q] = dweights[q] ? weights + q * plan.ranges * a.n : nullptr;
    merge.part[q] = a.part[q], merge.out[q] = dweights[q];
  }
  a.part[kGradGate] = dgate ? reinterpret_cast<float*>(ws + plan.sums_bytes + plan.weight_bytes) : nullptr;
  merge.part[kGradGate] = a.part[kGradGate], merge.out[kGradGate] = dgate;
  merge.n = a.n, merge.ranges = plan.ranges, merge.ld_dgate = ld_dgate, merge.num_gates = dgate ? num_gates : 0;
  merge.cols_per_gate = a.cols_per_gate, merge.cols_per_range = plan.cols_per_range;

  hipStream_t st = as_stream(stream);
  auto capped = [](int64_t blocks) { return static_cast<unsigned>(blocks < (int64_t(1) << 30) ? blocks : (int64_t(1) << 30)); };
  hipLaunchKernelGGL((rn_bwd_long_sums<T>), dim3(capped(a.width)), dim3(kRnLongThreads), 0, st, a);
  if (weight_grads || dgate) {
    hipLaunchKernelGGL((rn_bwd_long_columns<T>), dim3(capped(ceil_div(a.n, 2048)), static_cast<unsigned>(plan.ranges)), dim3(256),
                       0, st, a);
    const int64_t items = kGradGate + merge.num_gates;
    hipLaunchKernelGGL(rn_merge, dim3(capped(ceil_div(a.n, 256)), static_cast<unsigned>(items < 32768 ? items : 32768)),
                       dim3(256), 0, st, merge);
  }
  hipLaunchKernelGGL((rn_bwd_long_apply<T>), dim3(capped(ceil_div(a.n, 2048) * a.width)), dim3(256), 0, st, a);
  return launch_status();
}

}  // namespace lbn

extern "C" {

size_t lbn_residual_norm_bwd_workspace_bytes(int64_t size, int64_t width, int has_weight_grads, int64_t num_gate_grads,
                                             int elem_bytes)
{
  (void)elem_bytes;
  if (size <= 0 || width <= 0 || num_gate_grads < 0) return 0;
  return lbn::rn_bwd_plan(size, width, has_weight_grads, num_gate_grads).total();
}

#define LBN_RESIDUAL_NORM_ENTRIES(SUFFIX, ABI, T)                                                                    \
  int lbn_residual_norm_fwd_##SUFFIX(                                                                                \
    lbn_stream_t stream, int64_t size, int64_t width, int branch_norm, int output_norm, float epsilon,               \
    float residual_multiplier, float branch_multiplier, const ABI* branch, int64_t ld_branch, const ABI* residual,   \
    int64_t ld_residual, const float* gate, int64_t ld_gate, int64_t num_gates, const float* branch_scale,           \
    const float* branch_bias, const float* output_scale, const float* output_bias, double keep_prob, uint64_t seed,  \
    uint64_t offset, const uint64_t* step, int64_t column_offset, ABI* h, int64_t ld_h, ABI* y, int64_t ld_y,        \
    float* stats, int64_t ld_stats)                                                                                  \
  {                                                                                                                  \
    lbn::RnFwdArgs<T> a{};                                                                                           \
    a.n = size, a.width = width, a.branch_norm = branch_norm, a.output_norm = output_norm;                           \
    a.epsilon = epsilon, a.residual_mult = residual_multiplier, a.branch_mult = branch_multiplier;                   \
    a.branch = static_cast<const T*>(branch), a.ld_branch = ld_branch;                                               \
    a.residual = static_cast<const T*>(residual), a.ld_residual = ld_residual;                                       \
    a.gate = gate, a.ld_gate = ld_gate;                                                                              \
    a.branch_scale = branch_scale, a.branch_bias = branch_bias;                                                      \
    a.output_scale = output_scale, a.output_bias = output_bias;                                                      \
    a.h = static_cast<T*>(h), a.ld_h = ld_h, a.y = static_cast<T*>(y), a.ld_y = ld_y;                                \
    a.stats = stats, a.ld_stats = ld_stats;                                                                          \
    return lbn::rn_fwd<T>(stream, a, num_gates, keep_prob, seed, offset, step, column_offset);                       \
  }                                                                                                                  \
  int lbn_residual_norm_bwd_##SUFFIX(                                                                                \
    lbn_stream_t stream, int64_t size, int64_t width, int branch_norm, int output_norm, float epsilon,               \
    float residual_multiplier, float branch_multiplier, const ABI* branch, int64_t ld_branch, const ABI* h,          \
    int64_t ld_h, const float* gate, int64_t ld_gate, int64_t num_gates, const float* branch_scale,                  \
    const float* branch_bias, const float* output_scale, double keep_prob, uint64_t seed, uint64_t offset,           \
    const uint64_t* step, int64_t column_offset, const float* stats, int64_t ld_stats, const ABI* dy, int64_t ld_dy, \
    const ABI* dh, int64_t ld_dh, ABI* dbranch, int64_t ld_dbranch, ABI* dresidual, int64_t ld_dresidual,            \
    float* dgate, int64_t ld_dgate, float* dbranch_scale, float* dbranch_bias, float* doutput_scale,                 \
    float* doutput_bias, void* workspace, size_t workspace_bytes)                                                    \
  {                                                                                                                  \
    lbn::RnBwdArgs<T> a{};                                                                                           \
    a.n = size, a.width = width, a.branch_norm = branch_norm, a.output_norm = output_norm;                           \
    a.epsilon = epsilon, a.residual_mult = residual_multiplier, a.branch_mult = branch_multiplier;                   \
    a.branch = static_cast<const T*>(branch), a.ld_branch = ld_branch;                                               \
    a.h = static_cast<const T*>(h), a.ld_h = ld_h, a.gate = gate, a.ld_gate = ld_gate;                               \
    a.branch_scale = branch_scale, a.branch_bias = branch_bias, a.output_scale = output_scale;                       \
    a.stats = stats, a.ld_stats = ld_stats;                                                                          \
    a.dy = static_cast<const T*>(dy), a.ld_dy = ld_dy, a.dh = static_cast<const T*>(dh), a.ld_dh = ld_dh;            \
    a.dbranch = static_cast<T*>(dbranch), a.ld_dbranch = ld_dbranch;                                                 \
    a.dresidual = static_cast<T*>(dresidual), a.ld_dresidual = ld_dresidual;                                         \
    float* const dweights[lbn::kGradGate] = {doutput_scale, doutput_bias, dbranch_scale, dbranch_bias};              \
    return lbn::rn_bwd<T>(stream, a, num_gates, keep_prob, seed, offset, step, column_offset, dgate, ld_dgate,       \
                          dweights, workspace, workspace_bytes);                                                     \
  }

LBN_RESIDUAL_NORM_ENTRIES(f32, float, float)
LBN_RESIDUAL_NORM_ENTRIES(f16, void, lbn::f16_t)
LBN_RESIDUAL_NORM_ENTRIES(bf16, void, lbn::bf16_t)

#undef LBN_RESIDUAL_NORM_ENTRIES

}  // extern "C"
