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
// (the RMS norm drops mean(p)).  Sums over columns go through partial rows in the workspace, one for
// every range of columns, merged in a fixed order: no atomics, bitwise reproducible.  A gate column
// is shared by width / num_gates consecutive columns; ranges either lie within one gate's columns
// or hold all columns of the gates they meet.
#pragma once

#include "device_utils.hpp"
#include "host_utils.hpp"
#include "residual_norm_rows.hpp"

#include <initializer_list>

namespace lbn {

// Sums the partial rows of ranges of columns: weight gradients over all ranges, a gate column
// over its own.
struct RnMergeArgs {
  const float* part[kGrads];
  float* out[kGrads];
  int64_t n, ld_dgate;
  unsigned ranges, num_gates, ranges_per_gate;
  bool few;  // partial rows a gate, see kMergeFew
};

// A workgroup sums 64 neighbouring features: kMergeGroups groups of kMergeLanes lanes (four features each)
// take every kMergeGroups-th partial row, then a tree over the groups, all in a fixed order.
// Bound by latency: many groups, so that a thread has few loads and they are all in flight (256
// rows of 4096 features, three vectors: 4.9 us; 11.0 us with 16 groups of 64 single features).
constexpr int kMergeLanes = 16, kMergeGroups = 64;
// Gates of few partial rows have a group each, without a tree (27 gates of 8 rows of 5760 features and two scales:
// a workgroup each, 15.2 us; so, 5.7).
constexpr unsigned kMergeFew = 16;

static __global__ void __launch_bounds__(kMergeLanes * kMergeGroups)
rn_merge(RnMergeArgs a)
{
  __shared__ float sums[kMergeGroups][4 * kMergeLanes + 4];
  const int lane = threadIdx.x % kMergeLanes, group = threadIdx.x / kMergeLanes;
  const int64_t first_k = static_cast<int64_t>(blockIdx.x) * 4 * kMergeLanes, k = first_k + 4 * lane;
  const unsigned gate_items = a.few ? (a.num_gates + kMergeGroups - 1) / kMergeGroups : a.num_gates;
  for (uint64_t item = blockIdx.y; item < uint64_t(kGradGate) + gate_items; item += gridDim.y) {
    const int q = item < kGradGate ? static_cast<int>(item) : kGradGate;
    if (!a.out[q]) continue;
    if (q == kGradGate && a.few) {
      const uint64_t gate = (item - kGradGate) * kMergeGroups + group;
      if (gate < a.num_gates && k < a.n) {
        const float* from = a.part[q] + gate * a.ranges_per_gate * a.n + k;
        float s[4] = {};
        float* out = a.out[q] + gate * a.ld_dgate + k;
        if (k + 4 <= a.n) {
#pragma unroll 4
          for (unsigned b = 0; b < a.ranges_per_gate; ++b) {
            const typename Pack<float>::vec_t r = Pack<float>::load(from + b * a.n);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += r[j];
          }
          __builtin_memcpy(out, s, sizeof(s));
        }
        else {
          for (int j = 0; k + j < a.n; ++j) {
            float t = 0.f;
            for (unsigned b = 0; b < a.ranges_per_gate; ++b) t += from[b * a.n + j];
            out[j] = t;
          }
        }
      }
      continue;
    }
    const unsigned gate = static_cast<unsigned>(item) - kGradGate;  // the partial rows from `first` to `last`
    uint64_t first = 0, last = a.ranges - 1;
    float* out = a.out[q];
    if (q == kGradGate) {
      first = static_cast<uint64_t>(gate) * a.ranges_per_gate;
      last = first + a.ranges_per_gate - 1;
      out += gate * a.ld_dgate;
    }
    // The last features are read from further back, so that every read is whole: lanes that overlap
    // then write the same sums.
    const int64_t from = k + 4 <= a.n ? k : a.n - 4;
    if (k < a.n && from >= 0) {
      float s[4] = {};
#pragma unroll 4
      for (uint64_t b = first + group; b <= last; b += kMergeGroups) {
        const typename Pack<float>::vec_t r = Pack<float>::load(a.part[q] + b * a.n + from);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += r[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (from + j >= first_k) sums[group][from - first_k + j] = s[j];
    }
    else if (k < a.n) {  // fewer than four features
      for (int j = 0; j < a.n; ++j) {
        float s = 0.f;
        for (uint64_t b = first + group; b <= last; b += kMergeGroups) s += a.part[q][b * a.n + j];
        sums[group][j] = s;
      }
    }
    __syncthreads();
    // sixteen threads a feature, four groups each, then a row of lanes
    const int feature = threadIdx.x / 16, part = threadIdx.x % 16;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kMergeGroups / 16; ++i) t += sums[part + 16 * i][feature];
    t = row16_sum(t);
    if (part == 0 && first_k + feature < a.n) out[first_k + feature] = t;
    __syncthreads();
  }
}

static bool rn_ld_ok(const void* p, int64_t ld, int64_t height, int64_t width) { return !p || width <= 1 || ld >= height; }

static bool rn_norm_ok(int kind) { return kind >= kNormNone && kind <= kNormLayer; }

// How a column is shared: V units of eight entries per thread, a team of 16 lanes (`sub`) or of nw
// waves.  v == 0: it does not fit `max_v` units per thread of a full workgroup.
struct RnShape {
  int v, nw;
  bool sub;
  int threads() const { return sub || nw == 1 ? 256 : kWave * nw; }  // of a forward workgroup
  int teams() const { return sub ? 16 : (nw == 1 ? 4 : 1); }
  RowTeams row_teams(int teams) const { return {nw, teams, static_cast<unsigned>((65536 + nw - 1) / nw)}; }
};

// Calls that move this much read their inputs past the caches (4096 features, bf16, three sets of
// matrices in turn: 256 MiB forward in 51.4 -> 48.4 us, 384 MiB backward in 89 -> 78 us, but 128 MiB forward in
// 23 -> 25 us; sizes between were not measured).  Lengths that are no multiple of eight never do: their kernels exist with
// ordinary loads only.
constexpr int64_t kRnStreamBytes = int64_t(256) << 20;

constexpr int64_t kRnMostFeatures = int64_t(1) << 26;  // the merge of partial rows has a workgroup for 64 of them

// Whether a call takes the kernels for whole units and epsilons that leave no subnormal sum.  The others are for any
// length and epsilon (4096 x 8192 bf16 between two RMS norms with a gate without an epsilon: forward 45.7 us instead of
// 48.0, backward 108 instead of 77).
template <typename ARGS>
static bool rn_even(const ARGS& a)
{
  return a.n % 8 == 0 && (a.epsilon >= kRnNormalEpsilon || (a.branch_norm == kNormNone && a.output_norm == kNormNone));
}

static unsigned ld32(int64_t ld) { return static_cast<unsigned>(ld); }

// Leading dimensions (0 for a matrix that is not there) and widths that the row kernels' 32-bit indices hold.
// A leading dimension that no second column uses is not looked at.
static bool rn_fits32(int64_t width, std::initializer_list<int64_t> lds)
{
  if (width >= (int64_t(1) << 30)) return false;
  for (int64_t ld : lds)
    if (width > 1 && (ld < 0 || ld >= (int64_t(1) << 31))) return false;
  return true;
}

static RnShape rn_shape(int64_t n, int max_v = 1)
{
  const int64_t units = ceil_div(n, 8);
  if (n < 8) return {0, 0, false};  // no whole unit to read
  if (units <= 16) return {1, 1, true};
  if (units <= 32 && max_v >= 2) return {2, 1, true};
  for (int v = 1; v <= max_v; v *= 2)
    if (units <= 1024 * v) return {v, static_cast<int>(ceil_div(units, kWave * v)), false};
  return {0, 0, false};
}

// Backward: how many ranges of columns leave partial rows, and how a range is worked on.
struct RnBwdPlan {
  RnShape shape;  // v == 0: the long kernels
  int teams;
  int64_t ranges, cols_per_range, ranges_per_gate;
  bool twice;  // two workgroups a compute unit, where the kernel's registers allow it
  size_t sums_bytes, weight_bytes, gate_bytes;
  size_t total() const { return sums_bytes + weight_bytes + gate_bytes; }
  int threads() const { return (shape.sub ? 16 : kWave * shape.nw) * teams; }
  // Up to `most` ranges that do not cut across the end of a gate's columns.  A few more would be a second round of
  // workgroups (1024 x 4400 bf16 with 22 gates: 264 ranges 23.0 us, 242 of them 15.7).
  void cut(int64_t width, int64_t gates, int64_t most)
  {
    cols_per_range = ceil_div(width, most);
    if (cols_per_range < teams) cols_per_range = teams;
    ranges_per_gate = 0;
    if (gates > 0) {
      const int64_t per_gate = width / gates;
      if (per_gate > cols_per_range) {
        ranges_per_gate = ceil_div(per_gate, cols_per_range);
        if (ranges_per_gate > most / gates) ranges_per_gate = most / gates;
        cols_per_range = ceil_div(per_gate, ranges_per_gate);
        ranges = gates * ranges_per_gate;
        return;
      }
      cols_per_range = ceil_div(cols_per_range, per_gate) * per_gate;
    }
    ranges = ceil_div(width, cols_per_range);
  }
};

// One workgroup a compute unit, which keeps the partial rows few: 256 ranges of columns.  Where its
// teams leave a quarter of its lanes or more without entries, two (33.5 M entries, bf16: 256 features 76
// -> 65 us, 3000 features 73 -> 64, but 4096 features 59 -> 61).
constexpr int64_t kRnRanges = 256;

// gate_grads: the number of gates whose gradient is wanted.
static RnBwdPlan rn_bwd_plan(int64_t n, int64_t width, int weight_grads, int64_t gate_grads)
{
  RnBwdPlan p{};
  p.shape = rn_shape(n);
  p.teams = 1;
  int64_t most_ranges = kRnRanges;
  if (p.shape.v == 1) {
    // a workgroup of up to 8 waves (16 for the widest teams), no more teams than its range has columns
    const int64_t columns = ceil_div(width, kRnRanges);
    if (gate_grads > 1 && width / gate_grads < 16) {
      // few columns a gate: teams would wait for each other at the end of each, so single ones, more of them
      p.shape.sub = false;
      most_ranges = kRnRanges * (p.shape.nw <= 2 ? 4 : p.shape.nw <= 4 ? 2 : 1);
    }
    else {
      const int64_t most = p.shape.sub ? 32 : (p.shape.nw <= 8 ? 8 / p.shape.nw : 1);
      p.teams = static_cast<int>(columns < most ? columns : most);
      if (p.shape.sub) p.teams = static_cast<int>(ceil_div(p.teams, 4) * 4);  // whole waves
      p.twice = p.shape.nw <= 8 && ceil_div(n, 8) * p.teams <= 384;
      if (p.twice) most_ranges = 2 * kRnRanges;
    }
  }
  p.cut(width, gate_grads, most_ranges);
  auto round16 = [](int64_t b) { return static_cast<size_t>(ceil_div(b, 16) * 16); };
  p.sums_bytes = round16(width * 16);  // of the long kernels, which leading dimensions may call for
  if (weight_grads) p.weight_bytes = round16(kGradGate * p.ranges * n * 4);
  if (gate_grads && p.ranges_per_gate) p.gate_bytes = round16(p.ranges * n * 4);
  return p;
}

// The row kernel of a call.  Calls that are not `even` (rn_even) take, with a gate, the one that accumulates
// everything (without a gate that costs: 502 x 12100 bf16, two norms, 24.5 us against 19.3).
template <typename T, int TEAM>
static auto rn_bwd_kernel(bool norm, bool gate, bool bias, bool even, bool stream) -> void (*)(RnBwdRows<T>)
{
  auto of = [&](auto n, auto s) -> void (*)(RnBwdRows<T>) {
    constexpr bool N = decltype(n)::value, S = decltype(s)::value;
    if (gate) return bias ? rn_bwd_rows<T, TEAM, N, true, true, true, S> : rn_bwd_rows<T, TEAM, N, true, false, true, S>;
    return bias ? rn_bwd_rows<T, TEAM, N, false, true, true, S> : rn_bwd_rows<T, TEAM, N, false, false, true, S>;
  };
  if (!even && gate) return norm ? rn_bwd_rows<T, TEAM, true, true, true, false, false> : rn_bwd_rows<T, TEAM, false, true, true, false, false>;
  if (!even && norm) return bias ? rn_bwd_rows<T, TEAM, true, false, true, false, false> : rn_bwd_rows<T, TEAM, true, false, false, false, false>;
  if (!even) return bias ? rn_bwd_rows<T, TEAM, false, false, true, false, false> : rn_bwd_rows<T, TEAM, false, false, false, false, false>;
  if (stream) return norm ? of(std::true_type{}, std::true_type{}) : of(std::false_type{}, std::true_type{});
  return norm ? of(std::true_type{}, std::false_type{}) : of(std::false_type{}, std::false_type{});
}

template <typename T>
static auto rn_bwd_kernel(const RnBwdArgs<T>& g, const RnShape& shape, bool bias) -> void (*)(RnBwdRows<T>)
{
  const bool norm = g.branch_norm != kNormNone, gate = g.gate != nullptr, even = rn_even(g);
  const int64_t bytes = g.n * g.width * static_cast<int64_t>(sizeof(T)) * (1 + 2 * !!g.dy + !!g.dh + !!g.branch + !!g.dresidual);
  const bool stream = stream_call_inputs(bytes, kRnStreamBytes);
  if (shape.sub) return rn_bwd_kernel<T, 16>(norm, gate, bias, even, stream);
  if (shape.nw <= 8) return rn_bwd_kernel<T, 512>(norm, gate, bias, even, stream);
  return rn_bwd_kernel<T, 1024>(norm, gate, bias, even, stream);
}

template <typename T>
static void rn_launch_bwd(hipStream_t st, const RnBwdArgs<T>& g, const RnBwdPlan& plan, void (*kernel)(RnBwdRows<T>))
{
  RnBwdRows<T> a{};
  a.n = static_cast<int>(g.n), a.width = static_cast<int>(g.width);
  a.branch_norm = g.branch_norm, a.output_norm = g.output_norm, a.epsilon = g.epsilon;
  a.residual_mult = g.residual_mult, a.branch_mult = g.branch_mult;
  a.branch = g.branch, a.h = g.h, a.dy = g.dy, a.dh = g.dh, a.gate = g.gate, a.stats = g.stats;
  a.branch_scale = g.branch_scale, a.branch_bias = g.branch_bias, a.output_scale = g.output_scale;
  a.dbranch = g.dbranch, a.dresidual = g.dresidual, a.dgate = g.dgate;
  a.ld_branch = ld32(g.ld_branch), a.ld_h = ld32(g.ld_h), a.ld_dy = ld32(g.ld_dy), a.ld_dh = ld32(g.ld_dh);
  a.ld_gate = ld32(g.ld_gate), a.ld_stats = ld32(g.ld_stats), a.ld_dgate = ld32(g.ld_dgate);
  a.ld_dbranch = ld32(g.ld_dbranch), a.ld_dresidual = ld32(g.ld_dresidual);
  a.cols_per_gate = static_cast<unsigned>(g.cols_per_gate), a.cols_per_range = static_cast<unsigned>(g.cols_per_range);
  a.ranges_per_gate = static_cast<unsigned>(g.ranges_per_gate);
  a.drop = g.drop, a.teams = plan.shape.row_teams(plan.teams);
  for (int q = 0; q < kGrads; ++q) a.part[q] = g.part[q];
  const unsigned lds = plan.teams > 1 ? static_cast<unsigned>(kMergeRows * plan.threads() * 8 * sizeof(float)) : 0;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.ranges)), dim3(plan.threads()), lds, st, a);
}

template <typename T, int V, bool SUB, bool EVEN, bool STREAM>
static void rn_launch_fwd(hipStream_t st, const RnFwdArgs<T>& g, const RnShape& shape)
{
  RnFwdRows<T> a{};
  a.n = static_cast<int>(g.n), a.width = static_cast<int>(g.width);
  a.branch_norm = g.branch_norm, a.output_norm = g.output_norm, a.epsilon = g.epsilon;
  a.residual_mult = g.residual_mult, a.branch_mult = g.branch_mult;
  a.branch = g.branch, a.residual = g.residual, a.gate = g.gate, a.h = g.h, a.y = g.y, a.stats = g.stats;
  a.branch_scale = g.branch_scale, a.branch_bias = g.branch_bias;
  a.output_scale = g.output_scale, a.output_bias = g.output_bias;
  a.ld_branch = ld32(g.ld_branch), a.ld_residual = ld32(g.ld_residual), a.ld_gate = ld32(g.ld_gate);
  a.ld_h = ld32(g.ld_h), a.ld_y = ld32(g.ld_y), a.ld_stats = ld32(g.ld_stats);
  a.cols_per_gate = static_cast<unsigned>(g.cols_per_gate), a.drop = g.drop, a.teams = shape.row_teams(shape.teams());
  const int64_t blocks = ceil_div(g.width, shape.teams());
  const int64_t resident = resident_blocks(rn_fwd_rows<T, V, SUB, EVEN, STREAM>, shape.threads());
  const int64_t grid = resident > 0 && blocks > resident ? resident : blocks;
  hipLaunchKernelGGL((rn_fwd_rows<T, V, SUB, EVEN, STREAM>), dim3(walking_grid(grid)), dim3(shape.threads()), 0, st, a);
}

template <typename T, bool EVEN, bool STREAM>
static void rn_launch_fwd(hipStream_t st, const RnFwdArgs<T>& a, const RnShape& shape)
{
  if (shape.v == 1)
    shape.sub ? rn_launch_fwd<T, 1, true, EVEN, STREAM>(st, a, shape) : rn_launch_fwd<T, 1, false, EVEN, STREAM>(st, a, shape);
  else
    shape.sub ? rn_launch_fwd<T, 2, true, EVEN, STREAM>(st, a, shape) : rn_launch_fwd<T, 2, false, EVEN, STREAM>(st, a, shape);
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
  if (a.n > kRnMostFeatures || !drop_range_ok(a.n, a.width, column_offset)) return LBN_ERR_UNSUPPORTED;
  a.cols_per_gate = num_gates > 0 ? a.width / num_gates : a.width;
  a.drop = drop_args(keep_prob, seed, offset, step, column_offset);
  hipStream_t st = as_stream(stream);
  const RnShape shape = rn_shape(a.n, 2);
  if (shape.v && rn_fits32(a.width, {a.ld_branch, a.residual ? a.ld_residual : 0, a.gate ? a.ld_gate : 0, a.h ? a.ld_h : 0,
                                   a.y ? a.ld_y : 0, a.stats ? a.ld_stats : 0})) {
    const int64_t bytes = a.n * a.width * static_cast<int64_t>(sizeof(T)) * (1 + !!a.residual + !!a.h + !!a.y);
    if (!rn_even(a)) rn_launch_fwd<T, false, false>(st, a, shape);
    else if (stream_call_inputs(bytes, kRnStreamBytes)) rn_launch_fwd<T, true, true>(st, a, shape);
    else rn_launch_fwd<T, true, false>(st, a, shape);
  }
  else {
    hipLaunchKernelGGL((rn_fwd_long<T>), dim3(walking_grid(a.width)), dim3(kRnLongThreads), 0, st, a);
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
  if (a.n > kRnMostFeatures || !drop_range_ok(a.n, a.width, column_offset)) return LBN_ERR_UNSUPPORTED;
  if (!norm1 && !dgate) a.branch = nullptr;  // not needed, so not read
  a.cols_per_gate = num_gates > 0 ? a.width / num_gates : a.width;
  a.drop = drop_args(keep_prob, seed, offset, step, column_offset);
  bool weight_grads = false;
  for (float* d : dweights) weight_grads = weight_grads || d;
  RnBwdPlan plan = rn_bwd_plan(a.n, a.width, weight_grads, dgate ? num_gates : 0);
  if (!rn_fits32(a.width, {a.branch ? a.ld_branch : 0, a.h ? a.ld_h : 0, a.gate ? a.ld_gate : 0, a.stats ? a.ld_stats : 0,
                           a.dy ? a.ld_dy : 0, a.dh ? a.ld_dh : 0, a.ld_dbranch, a.dresidual ? a.ld_dresidual : 0,
                           dgate ? ld_dgate : 0}))
    plan.shape.v = 0;
  if (plan.total() && (!workspace || workspace_bytes < plan.total() || !aligned16(workspace))) return LBN_ERR_WORKSPACE;
  void (*kernel)(RnBwdRows<T>) = nullptr;
  if (plan.shape.v) {
    const bool bias = dweights[kGradOutputBias] || dweights[kGradBranchBias] || (dgate && a.branch_bias);
    kernel = rn_bwd_kernel<T>(a, plan.shape, bias);
    if (plan.twice && resident_blocks(kernel, plan.threads()) < 2 * kRnRanges)
      plan.cut(a.width, dgate ? num_gates : 0, kRnRanges);
  }
  char* ws = static_cast<char*>(workspace);
  a.sums = reinterpret_cast<float*>(ws);
  a.cols_per_range = plan.cols_per_range, a.ranges_per_gate = plan.ranges_per_gate;
  a.dgate = dgate, a.ld_dgate = ld_dgate;
  float* weights = reinterpret_cast<float*>(ws + plan.sums_bytes);
  RnMergeArgs merge{};
  for (int q = 0; q < kGradGate; ++q) {
    a.part[q] = !dweights[q] ? nullptr : plan.ranges == 1 ? dweights[q] : weights + q * plan.ranges * a.n;
    merge.part[q] = a.part[q], merge.out[q] = dweights[q];
  }
  if (dgate && plan.ranges_per_gate) {
    a.part[kGradGate] = reinterpret_cast<float*>(ws + plan.sums_bytes + plan.weight_bytes);
    merge.part[kGradGate] = a.part[kGradGate], merge.out[kGradGate] = dgate;
  }
  merge.n = a.n, merge.ld_dgate = ld_dgate, merge.ranges = static_cast<unsigned>(plan.ranges);
  merge.num_gates = merge.out[kGradGate] ? static_cast<unsigned>(num_gates) : 0;
  merge.ranges_per_gate = static_cast<unsigned>(plan.ranges_per_gate);
  merge.few = merge.num_gates > 1 && merge.ranges_per_gate <= kMergeFew;
  const int64_t items = kGradGate + (merge.few ? ceil_div(merge.num_gates, kMergeGroups) : int64_t(merge.num_gates));
  const dim3 merge_grid(static_cast<unsigned>(ceil_div(a.n, 4 * kMergeLanes)), static_cast<unsigned>(items < 32768 ? items : 32768));

  hipStream_t st = as_stream(stream);
  if (plan.shape.v) {
    rn_launch_bwd<T>(st, a, plan, kernel);
  }
  else {
    hipLaunchKernelGGL((rn_bwd_long_sums<T>), dim3(walking_grid(a.width)), dim3(kRnLongThreads), 0, st, a);
    const int64_t slices = ceil_div(a.n, 8 * kRnColumnThreads);
    hipLaunchKernelGGL((rn_bwd_long_columns<T>), dim3(static_cast<unsigned>(slices), static_cast<unsigned>(plan.ranges < 32768 ? plan.ranges : 32768)),
                       dim3(kRnColumnThreads), 0, st, a, plan.ranges);
  }
  // one range has written the gradients themselves
  if ((weight_grads && plan.ranges > 1) || merge.out[kGradGate])
    hipLaunchKernelGGL(rn_merge, merge_grid, dim3(kMergeLanes * kMergeGroups), 0, st, merge);
  return launch_status();
}

}  // namespace lbn

// The C entry points for one storage type.
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
