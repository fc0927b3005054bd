// Residual norm, the kernels that hold nothing across passes: any number of features, any
// alignment, any gate layout.  They serve the columns that are too long for one workgroup's
// registers.
//
// Bound by reading the column again: 33.5 M entries bf16 forward in 72 us at 20000 features and 104 at 100000 (four
// tensors once would take 52), backward in 126 us at 12288 (two passes over the inputs and the merge).
//
// Forward: one workgroup per column; the moments of the block's output, then those of the new
// residual stream, then both outputs, re-reading the column (from the caches) each time.
// Backward: (1) one workgroup per column forms the up to four row means the gradients need
// and leaves them in the workspace; (2) threads that own eight features walk a range of columns,
// write the gradients of the activations and leave partial sums of the weight and gate gradients;
// (3) those are merged in a fixed order (residual_norm.hpp).  A thread of (2) writes what it alone
// has read, so outputs may take the place of inputs.
#pragma once

#include "device_utils.hpp"
#include "philox.hpp"
#include "storage.hpp"

namespace lbn {

// Norm kinds of the ABI (LBN_NORM_*).
constexpr int kNormNone = 0, kNormRms = 1, kNormLayer = 2;

template <typename T>
struct RnFwdArgs {
  int64_t n, width;
  int branch_norm, output_norm;
  float epsilon, residual_mult, branch_mult;
  const T* branch;
  int64_t ld_branch;
  const T* residual;  // null: none
  int64_t ld_residual;
  const float* gate;  // null: none
  int64_t ld_gate, cols_per_gate;
  const float *branch_scale, *branch_bias, *output_scale, *output_bias;  // null: 1 resp. 0
  T* h;  // null: not wanted
  int64_t ld_h;
  T* y;
  int64_t ld_y;
  float* stats;  // null: not wanted
  int64_t ld_stats;
  DropArgs drop;
};

// Partial gradients: row b of part[q] is the sum over range b of the columns.
enum RnGrad { kGradOutputScale = 0, kGradOutputBias, kGradBranchScale, kGradBranchBias, kGradGate, kGrads };

template <typename T>
struct RnBwdArgs {
  int64_t n, width;
  int branch_norm, output_norm;
  float epsilon, residual_mult, branch_mult;
  const T* branch;  // null: not needed (no branch norm, no gate gradient)
  int64_t ld_branch;
  const T* h;  // null without an output norm
  int64_t ld_h;
  const float* gate;
  int64_t ld_gate, cols_per_gate;
  const float *branch_scale, *branch_bias, *output_scale;
  const float* stats;
  int64_t ld_stats;
  const T* dy;  // null without an output norm
  int64_t ld_dy;
  const T* dh;  // null: zero
  int64_t ld_dh;
  T* dbranch;
  int64_t ld_dbranch;
  T* dresidual;  // null: not wanted
  int64_t ld_dresidual;
  DropArgs drop;
  // partial gradients of ranges of columns; part[q] null: not wanted, or dgate written at once
  float* part[kGrads];
  float* dgate;
  int64_t ld_dgate;
  float* sums;            // long kernels: four means per column
  int64_t cols_per_range, ranges_per_gate;
};

// The columns of range b.  With ranges_per_gate > 0 no range reaches over the end of a gate's columns, each
// leaves one partial row of the gate's gradient; with 0, all columns of a gate lie in one range (or
// there is no gate), which writes the gate's gradient itself.
template <typename I>
__device__ __forceinline__ void rn_range(I b, I width, I cols_per_range, I cols_per_gate, I ranges_per_gate, I& first, I& last)
{
  if (ranges_per_gate) {
    const I gate = b / ranges_per_gate;
    first = gate * cols_per_gate + (b - gate * ranges_per_gate) * cols_per_range;
    last = min(first + cols_per_range, (gate + 1) * cols_per_gate);
  }
  else {
    first = b * cols_per_range;
    last = min(first + cols_per_range, width);
  }
}

// 1 / sqrt(v): 0 for an infinite variance and infinite for a zero one, as the formula has it
// (the Newton step alone would turn both into NaN).  v_rsq_f32 takes subnormal numbers for zeros: columns of
// entries below 2^-63 have such variances, and without an epsilon such sums, which are scaled then.
// SUBNORMAL: whether there can be any.  Where the epsilon is a normal number there are none, and the kernels that
// most calls take leave the scaling out: with it, backward of 768 and 1024 x 16384 bf16 between two RMS norms with a gate took
// 4 % longer, other calls up to 1 %.
template <bool SUBNORMAL = true>
__device__ __forceinline__ float rn_rstd(float v)
{
  const float r = rsqrt_refined(v);
  if constexpr (!SUBNORMAL) return v > 0.f && v < INFINITY ? r : __builtin_amdgcn_rsqf(v);
  return v >= 0x1p-126f && v < INFINITY ? r : __builtin_amdgcn_rsqf(v * 0x1p64f) * 0x1p32f;
}
constexpr float kRnNormalEpsilon = 0x1p-126f;  // from here on

template <int NW>
__device__ __forceinline__ void block_sum2(float& a, float& b, float (*slots)[2 * NW], int& turn, int wave, int lane)
{
  team_sum2<NW>(a, b, slots[turn], wave, lane);
  turn ^= 1;  // the other buffer's barrier separates two uses of this one
}

__device__ __forceinline__ void load_weights8(const float* w, int64_t k, int64_t valid, float fill, float (&out)[8])
{
  if (w) {
    load8(w + k, valid, out);
  }
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = fill;
  }
}

// u = N1(o) of eight entries, from its statistics.
__device__ __forceinline__ void rn_normalise8(float (&u)[8], float mean, float rstd, const float* scale, const float* bias,
                                              int64_t k, int64_t valid)
{
  float w[8], b[8];
  load_weights8(scale, k, valid, 1.f, w);
  load_weights8(bias, k, valid, 0.f, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = __builtin_fmaf((u[j] - mean) * rstd, w[j], b[j]);
}

// v = keep ? u / q : 0 of eight entries.
__device__ __forceinline__ void rn_drop8(float (&v)[8], const DropArgs& d, const DropStream& s, int64_t group, int64_t col)
{
  if (d.threshold < 65536u) {
    uint32_t w[4];
    drop_words(d, s, static_cast<uint32_t>(group), static_cast<uint32_t>(col), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = drop_kept(w, j, d.threshold) ? v[j] * d.inverse_keep : 0.f;
  }
}

constexpr int kRnLongThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kRnLongThreads)
rn_fwd_long(RnFwdArgs<T> a)
{
  constexpr int NW = kRnLongThreads / kWave;
  __shared__ float slots[2][2 * NW];
  int turn = 0;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const DropStream stream = drop_stream(a.drop);
  const int64_t groups = (a.n + 7) / 8;
  const float nf = static_cast<float>(a.n);
  for (int64_t col = blockIdx.x; col < a.width; col += gridDim.x) {
    const T* o = a.branch + col * a.ld_branch;
    const float* gate = a.gate ? a.gate + col / a.cols_per_gate * a.ld_gate : nullptr;
    // mean (centred norms only) and mean of squared deviations of what `value` yields
    auto moments = [&](int kind, auto value, float& mean, float& var) {
      float s = 0.f, unused = 0.f;
      mean = 0.f;
      if (kind == kNormLayer) {
        for (int64_t g = threadIdx.x; g < groups; g += kRnLongThreads) {
          float v[8];
          value(g, v);
          for (int j = 0; j < 8; ++j) s += 8 * g + j < a.n ? v[j] : 0.f;
        }
        block_sum2<NW>(s, unused, slots, turn, wave, lane);
        mean = s / nf;
      }
      float q = 0.f;
      for (int64_t g = threadIdx.x; g < groups; g += kRnLongThreads) {
        float v[8];
        value(g, v);
        for (int j = 0; j < 8; ++j) {
          const float d = 8 * g + j < a.n ? v[j] - mean : 0.f;
          q = __builtin_fmaf(d, d, q);
        }
      }
      block_sum2<NW>(q, unused, slots, turn, wave, lane);
      var = q / nf;
    };
    float mean1 = 0.f, var1 = 1.f, rstd1 = 1.f, mean2 = 0.f, var2 = 1.f, rstd2 = 1.f;
    if (a.branch_norm != kNormNone) {
      moments(a.branch_norm, [&](int64_t g, float (&v)[8]) { load8(o + 8 * g, a.n - 8 * g, v); }, mean1, var1);
      rstd1 = rn_rstd(var1 + a.epsilon);
    }
    auto stream_entry = [&](int64_t g, float (&v)[8]) {
      const int64_t k = 8 * g, valid = a.n - k;
      load8(o + k, valid, v);
      if (a.branch_norm != kNormNone) rn_normalise8(v, mean1, rstd1, a.branch_scale, a.branch_bias, k, valid);
      rn_drop8(v, a.drop, stream, g, col);
      float gt[8], r[8];
      load_weights8(gate, k, valid, 1.f, gt);
      if (a.residual) load8(a.residual + col * a.ld_residual + k, valid, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] *= a.branch_mult * gt[j];
        if (a.residual) v[j] = __builtin_fmaf(a.residual_mult, r[j], v[j]);
      }
    };
    if (a.output_norm != kNormNone) {
      moments(a.output_norm, stream_entry, mean2, var2);
      rstd2 = rn_rstd(var2 + a.epsilon);
    }
    for (int64_t g = threadIdx.x; g < groups; g += kRnLongThreads) {
      const int64_t k = 8 * g, valid = a.n - k;
      float v[8];
      stream_entry(g, v);
      if (a.h) store8(a.h + col * a.ld_h + k, valid, v);
      if (a.output_norm != kNormNone) {
        rn_normalise8(v, mean2, rstd2, a.output_scale, a.output_bias, k, valid);
        store8(a.y + col * a.ld_y + k, valid, v);
      }
    }
    if (a.stats && threadIdx.x == 0) {
      float* st = a.stats + col * a.ld_stats;
      st[0] = mean1, st[1] = var1, st[2] = mean2, st[3] = var2;
    }
  }
}

// ------------------------------------------------------------------ backward
// What the statistics of a column say.
struct RnColumnStats {
  float mean1, rstd1, mean2, rstd2;
};

template <typename T>
__device__ __forceinline__ RnColumnStats rn_column_stats(const RnBwdArgs<T>& a, int64_t col)
{
  RnColumnStats s{0.f, 1.f, 0.f, 1.f};
  const float* st = a.stats + col * a.ld_stats;
  if (a.branch_norm != kNormNone) s.mean1 = st[0], s.rstd1 = rn_rstd(st[1] + a.epsilon);
  if (a.output_norm != kNormNone) s.mean2 = st[2], s.rstd2 = rn_rstd(st[3] + a.epsilon);
  return s;
}

// e = dL/dh of eight entries, all contributions included; xh: the normalised stream.
template <typename T>
__device__ __forceinline__ void rn_stream_grad8(const RnBwdArgs<T>& a, const RnColumnStats& s, int64_t col, int64_t k,
                                                int64_t valid, float mean_p, float mean_px, float (&e)[8], float (&dy)[8],
                                                float (&xh)[8])
{
  if (a.dh) {
    load8(a.dh + col * a.ld_dh + k, valid, e);
  }
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = 0.f;
  }
  if (a.output_norm != kNormNone) {
    float w[8];
    load8(a.dy + col * a.ld_dy + k, valid, dy);
    load8(a.h + col * a.ld_h + k, valid, xh);
    load_weights8(a.output_scale, k, valid, 1.f, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xh[j] = (xh[j] - s.mean2) * s.rstd2;
      e[j] = __builtin_fmaf(s.rstd2, dy[j] * w[j] - mean_p - xh[j] * mean_px, e[j]);
    }
  }
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j) dy[j] = xh[j] = 0.f;
  }
}

// du = dL/du of eight entries from e; also uh, the normalised branch, and ev = b e v, the
// gate's gradient (both only where the branch is read).
template <typename T>
__device__ __forceinline__ void rn_branch_grad8(const RnBwdArgs<T>& a, const DropStream& stream, const RnColumnStats& s,
                                                int64_t col, int64_t k, int64_t valid, const float (&e)[8], float (&du)[8],
                                                float (&uh)[8], float (&ev)[8])
{
  float gt[8], keep[8];
  load_weights8(a.gate ? a.gate + col / a.cols_per_gate * a.ld_gate : nullptr, k, valid, 1.f, gt);
#pragma unroll
  for (int j = 0; j < 8; ++j) keep[j] = 1.f;
  rn_drop8(keep, a.drop, stream, k / 8, col);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = a.branch_mult * e[j];
    du[j] = keep[j] != 0.f ? f * gt[j] * keep[j] : 0.f;
    uh[j] = ev[j] = 0.f;
  }
  if (a.branch) {
    float u[8];
    load8(a.branch + col * a.ld_branch + k, valid, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = uh[j] = (u[j] - s.mean1) * s.rstd1;
    if (a.branch_norm != kNormNone) {
      float w[8], b[8];
      load_weights8(a.branch_scale, k, valid, 1.f, w);
      load_weights8(a.branch_bias, k, valid, 0.f, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = __builtin_fmaf(u[j], w[j], b[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ev[j] = keep[j] != 0.f ? a.branch_mult * e[j] * (u[j] * keep[j]) : 0.f;
  }
}

// (1) The means of p = dy scale2, p xh, p1 = du scale1, p1 uh of every column.
template <typename T>
__global__ void __launch_bounds__(kRnLongThreads)
rn_bwd_long_sums(RnBwdArgs<T> a)
{
  constexpr int NW = kRnLongThreads / kWave;
  __shared__ float slots[2][2 * NW];
  int turn = 0;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const DropStream stream = drop_stream(a.drop);
  const int64_t groups = (a.n + 7) / 8;
  const float nf = static_cast<float>(a.n);
  for (int64_t col = blockIdx.x; col < a.width; col += gridDim.x) {
    const RnColumnStats s = rn_column_stats(a, col);
    float m[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.output_norm != kNormNone) {
      float sp = 0.f, spx = 0.f;
      for (int64_t g = threadIdx.x; g < groups; g += kRnLongThreads) {
        const int64_t k = 8 * g, valid = a.n - k;
        float dy[8], x[8], w[8];
        load8(a.dy + col * a.ld_dy + k, valid, dy);
        load8(a.h + col * a.ld_h + k, valid, x);
        load_weights8(a.output_scale, k, valid, 1.f, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= valid) continue;  // the distance of a missing entry from the mean may overflow
          const float p = dy[j] * w[j];
          sp += p;
          spx = __builtin_fmaf(p, (x[j] - s.mean2) * s.rstd2, spx);
        }
      }
      block_sum2<NW>(sp, spx, slots, turn, wave, lane);
      m[0] = a.output_norm == kNormLayer ? sp / nf : 0.f;
      m[1] = spx / nf;
    }
    if (a.branch_norm != kNormNone) {
      float sp = 0.f, spu = 0.f;
      for (int64_t g = threadIdx.x; g < groups; g += kRnLongThreads) {
        const int64_t k = 8 * g, valid = a.n - k;
        float e[8], dy[8], xh[8], du[8], uh[8], ev[8], w[8];
        rn_stream_grad8(a, s, col, k, valid, m[0], m[1], e, dy, xh);
        rn_branch_grad8(a, stream, s, col, k, valid, e, du, uh, ev);
        load_weights8(a.branch_scale, k, valid, 1.f, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= valid) continue;
          const float p = du[j] * w[j];
          sp += p;
          spu = __builtin_fmaf(p, uh[j], spu);
        }
      }
      block_sum2<NW>(sp, spu, slots, turn, wave, lane);
      m[2] = a.branch_norm == kNormLayer ? sp / nf : 0.f;
      m[3] = spu / nf;
    }
    if (threadIdx.x == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) a.sums[4 * col + j] = m[j];
    }
  }
}

// (2) Gradients of the activations and partial sums: blockIdx.x is a slice of features, blockIdx.y a
// range of columns.
constexpr int kRnColumnThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kRnColumnThreads)
rn_bwd_long_columns(RnBwdArgs<T> a, int64_t ranges)
{
  const DropStream stream = drop_stream(a.drop);
  const int64_t group = static_cast<int64_t>(blockIdx.x) * kRnColumnThreads + threadIdx.x;
  const int64_t k = 8 * group, valid = a.n - k;
  if (valid <= 0) return;
  for (int64_t range = blockIdx.y; range < ranges; range += gridDim.y) {
    int64_t first, last;
    rn_range<int64_t>(range, a.width, a.cols_per_range, a.cols_per_gate, a.ranges_per_gate, first, last);
    float acc[kGrads][8] = {};
    for (int64_t col = first; col < last; ++col) {
      const RnColumnStats s = rn_column_stats(a, col);
      const float* m = a.sums + 4 * col;
      float e[8], dy[8], xh[8], du[8], uh[8], ev[8];
      rn_stream_grad8(a, s, col, k, valid, m[0], m[1], e, dy, xh);
      rn_branch_grad8(a, stream, s, col, k, valid, e, du, uh, ev);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[kGradOutputScale][j] = __builtin_fmaf(dy[j], xh[j], acc[kGradOutputScale][j]);
        acc[kGradOutputBias][j] += dy[j];
        acc[kGradBranchScale][j] = __builtin_fmaf(du[j], uh[j], acc[kGradBranchScale][j]);
        acc[kGradBranchBias][j] += du[j];
        acc[kGradGate][j] += ev[j];
      }
      if (a.dresidual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] *= a.residual_mult;
        store8(a.dresidual + col * a.ld_dresidual + k, valid, e);
      }
      if (a.branch_norm != kNormNone) {
        float w[8];
        load_weights8(a.branch_scale, k, valid, 1.f, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) du[j] = s.rstd1 * (du[j] * w[j] - m[2] - uh[j] * m[3]);
      }
      store8(a.dbranch + col * a.ld_dbranch + k, valid, du);
      if (a.dgate && a.ranges_per_gate == 0 && (col + 1) % a.cols_per_gate == 0) {
        store8(a.dgate + col / a.cols_per_gate * a.ld_dgate + k, valid, acc[kGradGate]);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[kGradGate][j] = 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < kGrads; ++q)
      if (a.part[q]) store8(a.part[q] + range * a.n + k, valid, acc[q]);
  }
}

}  // namespace lbn
