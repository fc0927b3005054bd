// Residual norm, the kernels that hold a column in registers: every tensor crosses HBM once.
//
// A "unit" is eight consecutive entries of a column, what one counter of the generator serves;
// a thread owns V units.  A team works on a column: 16 lanes (a DPP row) for up to 128 V
// features, otherwise NW whole waves, 512 V NW >= n; a workgroup holds several teams where a team
// is at most a wave, else one.  Teams walk columns with the next column's loads in flight and,
// for V = 1, the weights of their units in registers.
//
// One norm costs one workgroup barrier: a wave takes the mean and the squared deviations of its own
// entries from registers (two passes, no E[x^2] - mean^2 cancellation), and the pairs of the
// waves are merged as sums over parts are:  M2 = sum of M2_w + n_w (mean_w - mean)^2.
#pragma once

#include "residual_norm_long.hpp"

namespace lbn {

// Eight entries as they are stored.  A column whose length is no multiple of eight ends in a partial
// unit: it is read as the last eight entries of the column and moved down by `shift` entries when
// it is used, which leaves zeros where nothing is.  So every load is whole, waits for nothing and stays inside the
// column (columns have at least eight entries here), and only the wave with the partial unit moves
// anything.
template <typename T>
struct Unit {
  typedef T raw_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  static __device__ __forceinline__ raw_t load(const T* p) { return *reinterpret_cast<const raw_t*>(p); }
  // STREAM: past the caches, for calls that move more than they hold.
  template <bool STREAM>
  static __device__ __forceinline__ raw_t load(const T* p)
  {
    if constexpr (!STREAM) return load(p);
    constexpr int N = Pack<T>::N;
    raw_t r;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const typename Pack<T>::vec_t v = __builtin_nontemporal_load(reinterpret_cast<const typename Pack<T>::vec_t*>(p + i));
#pragma unroll
      for (int k = 0; k < N; ++k) r[i + k] = v[k];
    }
    return r;
  }
  // ROUND: what leaves at the bottom comes back at the top, so that missing entries are entries of the column.
  template <bool ROUND = false>
  static __device__ __forceinline__ raw_t moved(const raw_t& r, int shift)
  {
    constexpr int W = 2 * static_cast<int>(sizeof(T));  // words of a unit
    uint32_t d[W + 4];
    __builtin_memcpy(d, &r, 4 * W);
    if constexpr (sizeof(T) == 2) {
      if (shift & 1) {
        const uint32_t first = ROUND ? d[0] : 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) d[i] = d[i] >> 16 | (i + 1 < W ? d[i + 1] : first) << 16;
      }
      shift >>= 1;
    }
#pragma unroll
    for (int by = 1; by < W; by *= 2) {
      if (shift & by) {
        uint32_t first[W];
#pragma unroll
        for (int i = 0; i < W; ++i) first[i] = ROUND ? d[i] : 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) d[i] = i + by < W ? d[i + by] : first[i + by - W];
      }
    }
    if (!ROUND && (shift & W)) {
#pragma unroll
      for (int i = 0; i < W; ++i) d[i] = 0u;
    }
    raw_t out;
    __builtin_memcpy(&out, d, 4 * W);
    return out;
  }
  // EVEN: the length is a multiple of eight, a unit exists (shift 0) or does not (8).
  template <bool EVEN>
  static __device__ __forceinline__ void widen(raw_t r, int shift, float (&v)[8])
  {
    if constexpr (EVEN) {
      uint32_t d[sizeof(raw_t) / 4];
      __builtin_memcpy(d, &r, sizeof(d));
#pragma unroll
      for (uint32_t& w : d) w = shift ? 0u : w;
      __builtin_memcpy(&r, d, sizeof(d));
    }
    else if (shift) {
      r = moved(r, shift);
    }
    widen(r, v);
  }
  // For what a mean is taken from in backward.  A zero's distance from the mean may overflow when it is scaled (columns of one
  // large number), and infinity times the zero that stands beside it is no zero.  So missing entries of partial units
  // are entries of the column, which are as near to its mean as any; missing whole units: RowShare::epsilon.
  template <bool EVEN>
  static __device__ __forceinline__ void widen_centred(raw_t r, int shift, float (&v)[8])
  {
    if constexpr (EVEN) {
      widen<true>(r, shift, v);
    }
    else {
      if (shift) r = moved<true>(r, shift);
      widen(r, v);
    }
  }
  static __device__ __forceinline__ void widen(const raw_t& r, float (&v)[8])
  {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(r[j]);
  }
};

// Eight entries in the storage type: the whole unit, or its first `valid` ones in up to three pieces.
// NT: past the caches, for forward calls that are themselves too large for them: a training step writes
// its activations to fresh memory (4096 x 8192 bf16, eight sets of outputs in turn: 47.5 us, 50.7 with
// ordinary stores).  Gradients are read next and their memory soon used again: ordinary stores
// keep them in the last-level cache (backward of the same shape: 76.5 us against 86.0).
template <bool EVEN, bool NT = false, typename T>
__device__ __forceinline__ void store_unit(T* p, int valid, const float (&v)[8])
{
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = static_cast<T>(v[j]);
  if (valid == 8) {
    if constexpr (NT) store8(p, 8, v);
    else __builtin_memcpy(p, t, sizeof(t));
  }
  else if constexpr (!EVEN) {
    const bool four = valid & 4, two = valid & 2;
    if (four) __builtin_memcpy(p, t, 4 * sizeof(T));
    const T a[2] = {four ? t[4] : t[0], four ? t[5] : t[1]};
    const T c = four ? t[6] : t[2];
    if (two) __builtin_memcpy(p + (valid & 4), a, 2 * sizeof(T));
    if (valid & 1) p[valid & 6] = two ? c : a[0];
  }
}

// Which entries of its column a thread owns: unit(i) = t + i * lanes, of which valid[i] entries exist.
template <int V, bool EVEN>
struct RowShare {
  int unit[V], valid[V], at[V], shift[V];  // where the unit is read, and how far it is moved then
  __device__ __forceinline__ RowShare(int t, int lanes, int n)
  {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      unit[i] = t + i * lanes;
      const int left = n - 8 * unit[i];
      valid[i] = left < 0 ? 0 : (left > 8 ? 8 : left);
      at[i] = left < 8 ? n - 8 : 8 * unit[i];
      shift[i] = 8 - valid[i];
    }
  }
  // The epsilon of unit i.  Kernels for whole units: infinite where nothing exists, which makes 1 / sqrt(var + epsilon)
  // zero there (see Unit::widen_centred).
  __device__ __forceinline__ float epsilon(int i, float e) const { return !EVEN || valid[i] ? e : INFINITY; }
  // The thread's entries of a weight vector (null: `fill`); 0 where nothing exists.
  __device__ __forceinline__ void weights(const float* w, int i, float fill, float (&out)[8]) const
  {
    if (w) {
      Unit<float>::template widen<EVEN>(Unit<float>::load(w + at[i]), shift[i], out);
    }
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = j < valid[i] ? fill : 0.f;
    }
  }
};

template <bool SUB>
__device__ __forceinline__ float lanes_sum(float v)
{
  return SUB ? row16_sum(v) : wave_sum(v);
}

// Merges over the waves of a team, through sixteen slots a team.  Every team of the workgroup makes
// the same calls.
constexpr int kMergeSlots = 4 * 16;  // teams of two waves or more: at most four

struct TeamMerge {
  float2 (*slots)[kMergeSlots];  // two buffers, zero behind a team's wave nw
  int nw, wave, lane;
  int base;             // the team's first slot
  float count;          // entries of the column that wave (lane % 16) owns
  int turn = 0;

  __device__ __forceinline__ float2 exchange(float a, float b)
  {
    if (lane == 0) slots[turn][base + wave] = make_float2(a, b);
    __syncthreads();
    const float2 r = slots[turn][base + (lane & 15)];
    turn ^= 1;  // the other buffer's barrier separates two uses of this one
    return r;
  }
  __device__ __forceinline__ void sum2(float& a, float& b)
  {
    const float2 r = exchange(a, b);
    a = row16_sum(r.x);
    b = row16_sum(r.y);
  }
};

// Mean and variance of a column from registers.  Entries that do not exist are zeros and do not count.
template <int V, bool SUB, bool FULL, bool EVEN>
__device__ __forceinline__ void row_moments(const float (&x)[V][8], const RowShare<V, EVEN>& share, int kind, float inv_n,
                                            float inv_mine, TeamMerge& merge, float& mean, float& var)
{
  float part_mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += x[i][j];
    part_mean = lanes_sum<SUB>(s) * inv_mine;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = FULL || (EVEN ? share.valid[i] != 0 : j < share.valid[i]) ? x[i][j] - part_mean : 0.f;
      q = __builtin_fmaf(d, d, q);
    }
  q = lanes_sum<SUB>(q);
  mean = part_mean;
  if (!SUB && merge.nw > 1) {
    const float2 r = merge.exchange(part_mean, q);
    if (kind == kNormLayer) {
      mean = row16_sum(merge.count * r.x) * inv_n;
      const float d = r.x - mean;
      q = row16_sum(__builtin_fmaf(merge.count * d, d, r.y));
    }
    else {
      q = row16_sum(r.y);
    }
  }
  var = q * inv_n;
}

// How a workgroup is cut into teams; `of_wave`: 65536 / nw rounded up, so that wave * of_wave >> 16 is
// the wave's team (exact for up to 16 waves).
struct RowTeams {
  int nw, teams;
  unsigned of_wave;
};

// What a team needs to know about itself; block-wide set-up of the merge buffers included.
template <int V, bool SUB>
struct Team {
  int index, t;
  float inv_n, inv_mine;  // 1 / entries of the column, of this wave
  __device__ __forceinline__ Team(const RowTeams& shape, int n, float2 (*slots)[kMergeSlots], TeamMerge& merge)
  {
    const int tid = threadIdx.x, nw = shape.nw;
    const int lanes = SUB ? 16 : kWave * nw;
    index = SUB ? tid / 16 : static_cast<int>(wave_index() * shape.of_wave >> 16);
    t = tid - index * lanes;
    merge.slots = slots;
    merge.nw = nw;
    merge.lane = tid & (kWave - 1);
    merge.wave = SUB ? 0 : wave_index() - index * nw;
    merge.base = 16 * index;
    auto entries_of = [&](int wave) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int left = n - 8 * (wave * kWave + i * lanes);
        c += left < 0 ? 0 : (left > 8 * kWave ? 8 * kWave : left);
      }
      return c;
    };
    inv_n = 1.f / static_cast<float>(n);
    inv_mine = inv_n;
    merge.count = 0.f;
    if (!SUB && nw > 1) {
      const int mine = entries_of(merge.wave);
      inv_mine = mine > 0 ? 1.f / static_cast<float>(mine) : 0.f;
      merge.count = (merge.lane & 15) < nw ? static_cast<float>(entries_of(merge.lane & 15)) : 0.f;
      for (int i = tid; i < 2 * kMergeSlots; i += static_cast<int>(blockDim.x))
        slots[i / kMergeSlots][i % kMergeSlots] = make_float2(0.f, 0.f);
      __syncthreads();
    }
  }
};

// The arguments of the row kernels: columns and leading dimensions in 32 bits (the host sends larger
// ones to the long kernels).  64-bit products and divisions on the scalar unit were a third of the
// instructions of a kernel that walks only a few columns (backward over 777 columns of 1023 fp32: 21 -> 17 us
// without them).
template <typename T>
struct RnFwdRows {
  int n, width;
  int branch_norm, output_norm;
  float epsilon, residual_mult, branch_mult;
  const T *branch, *residual;
  const float *gate, *branch_scale, *branch_bias, *output_scale, *output_bias;
  T *h, *y;
  float* stats;
  unsigned ld_branch, ld_residual, ld_gate, ld_h, ld_y, ld_stats, cols_per_gate;
  DropArgs drop;
  RowTeams teams;
};

template <typename T>
struct RnBwdRows {
  int n, width;
  int branch_norm, output_norm;
  float epsilon, residual_mult, branch_mult;
  const T *branch, *h, *dy, *dh;
  const float *gate, *branch_scale, *branch_bias, *output_scale, *stats;
  T *dbranch, *dresidual;
  unsigned ld_branch, ld_h, ld_dy, ld_dh, ld_gate, ld_stats, ld_dbranch, ld_dresidual, ld_dgate, cols_per_gate, cols_per_range, ranges_per_gate;
  DropArgs drop;
  float* part[kGrads];
  float* dgate;
  RowTeams teams;
};

template <typename T>
__device__ __forceinline__ T* column(T* p, unsigned col, unsigned ld)
{
  return p + static_cast<uint64_t>(col) * ld;
}

// Forward.  Bound by HBM where the columns fill the chip: 4096 x 8192 fp16 with dropout, 256 MiB moved,
// in 49.3 us (5.4 TB/s; a copy reaches 5.1); 1151 x 3000 fp32 between two layer norms in 16.1 us (3.4
// TB/s: three rounds of columns a workgroup, of which the last is a third full).  A single column of 4096
// takes 3.2 us, of which about 3 is what an empty launch traces at.  One resident wave of
// workgroups walks the columns: with the weights in registers that beats workgroups of one, two or
// four columns (50.9 us against 57.0, 52.5 and 51.3 at 4096 x 8192).
template <typename T, int V, bool SUB, bool EVEN, bool STREAM>
__global__ void __launch_bounds__(SUB ? 256 : 1024)
rn_fwd_rows(RnFwdRows<T> a)
{
  using U = Unit<T>;
  constexpr bool kKeepWeights = V == 1 || SUB;  // of a thread's units, in registers from column to column
  constexpr bool kPrefetch = V == 1 || SUB;
  constexpr int WV = kKeepWeights ? V : 1;
  __shared__ float2 slots[2][kMergeSlots];
  TeamMerge merge;
  const int n = a.n, lanes = SUB ? 16 : kWave * a.teams.nw;
  const Team<V, SUB> team(a.teams, n, slots, merge);
  const RowShare<V, EVEN> share(team.t, lanes, n);
  const DropStream stream = drop_stream(a.drop);
  const bool dropping = a.drop.threshold < 65536u;
  const unsigned width = a.width;
  const bool one_gate = a.gate && a.cols_per_gate == width;

  auto gate_of = [&](unsigned col) { return a.gate ? column(a.gate, col / a.cols_per_gate, a.ld_gate) : nullptr; };
  auto weights = [&](const float* w, int i, float fill, float (&out)[8]) { share.weights(w, i, fill, out); };
  float w1[WV][8], b1[WV][8], w2[WV][8], b2[WV][8], gt[WV][8];
  if constexpr (kKeepWeights) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      weights(a.branch_scale, i, 1.f, w1[i]);
      weights(a.branch_bias, i, 0.f, b1[i]);
      weights(a.output_scale, i, 1.f, w2[i]);
      weights(a.output_bias, i, 0.f, b2[i]);
      weights(one_gate ? a.gate : nullptr, i, 1.f, gt[i]);
    }
  }

  typename U::raw_t qo[V], qr[V];
  auto issue = [&](unsigned col) {
    const T* o = column(a.branch, col, a.ld_branch);
#pragma unroll
    for (int i = 0; i < V; ++i) qo[i] = U::template load<STREAM>(o + share.at[i]);
    if (a.residual) {
      const T* r = column(a.residual, col, a.ld_residual);
#pragma unroll
      for (int i = 0; i < V; ++i) qr[i] = U::template load<STREAM>(r + share.at[i]);
    }
  };
  const unsigned step = gridDim.x * a.teams.teams;

  // full: every unit of every thread exists, nothing is masked
  auto walk = [&](auto full) {
    constexpr bool kFull = decltype(full)::value;
    unsigned col = blockIdx.x * a.teams.teams + team.index;
    if (kPrefetch && col < width) issue(col);
    for (; col < width; col += step) {
      if (!kPrefetch) issue(col);
      float x[V][8], r[V][8];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (kFull) U::widen(qo[i], x[i]);
        else U::template widen<EVEN>(qo[i], share.shift[i], x[i]);
      }
      if (a.residual) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if constexpr (kFull) U::widen(qr[i], r[i]);
          else U::template widen<EVEN>(qr[i], share.shift[i], r[i]);
        }
      }
      if (kPrefetch && col + step < width) issue(col + step);
      if (a.gate && !one_gate && kKeepWeights) {
#pragma unroll
        for (int i = 0; i < V; ++i) weights(gate_of(col), i, 1.f, gt[i]);
      }
      float mean1 = 0.f, var1 = 1.f, mean2 = 0.f, var2 = 1.f;
      if (a.branch_norm != kNormNone) {
        row_moments<V, SUB, kFull, EVEN>(x, share, a.branch_norm, team.inv_n, team.inv_mine, merge, mean1, var1);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float rstd = rn_rstd<!EVEN>(var1 + (kFull ? a.epsilon : share.epsilon(i, a.epsilon)));
          if constexpr (!kKeepWeights) {
            weights(a.branch_scale, i, 1.f, w1[0]);
            weights(a.branch_bias, i, 0.f, b1[0]);
          }
          constexpr bool kw = kKeepWeights;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            // partial units: the weight first, which is zero where nothing exists
            x[i][j] = EVEN ? __builtin_fmaf((x[i][j] - mean1) * rstd, w1[kw ? i : 0][j], b1[kw ? i : 0][j])
                           : __builtin_fmaf(x[i][j] - mean1, rstd * w1[kw ? i : 0][j], b1[kw ? i : 0][j]);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (dropping) {
          uint32_t w[4];
          drop_words(a.drop, stream, share.unit[i], col, w);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            x[i][j] = drop_kept(w, j, a.drop.threshold) ? x[i][j] * a.drop.inverse_keep : 0.f;
        }
        if constexpr (!kKeepWeights) weights(gate_of(col), i, 1.f, gt[0]);
        constexpr bool kw = kKeepWeights;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[i][j] *= a.branch_mult * gt[kw ? i : 0][j];
          if (a.residual) x[i][j] = __builtin_fmaf(a.residual_mult, r[i][j], x[i][j]);
        }
        if (a.h) store_unit<EVEN, STREAM>(column(a.h, col, a.ld_h) + 8 * share.unit[i], kFull ? 8 : share.valid[i], x[i]);
      }
      if (a.output_norm != kNormNone) {
        row_moments<V, SUB, kFull, EVEN>(x, share, a.output_norm, team.inv_n, team.inv_mine, merge, mean2, var2);
        const float rstd = rn_rstd<!EVEN>(var2 + a.epsilon);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if constexpr (!kKeepWeights) {
            weights(a.output_scale, i, 1.f, w2[0]);
            weights(a.output_bias, i, 0.f, b2[0]);
          }
          constexpr bool kw = kKeepWeights;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            x[i][j] = __builtin_fmaf((x[i][j] - mean2) * rstd, w2[kw ? i : 0][j], b2[kw ? i : 0][j]);
          store_unit<EVEN, STREAM>(column(a.y, col, a.ld_y) + 8 * share.unit[i], kFull ? 8 : share.valid[i], x[i]);
        }
      }
      if (a.stats && team.t == 0) {
        const float st[4] = {mean1, var1, mean2, var2};
        __builtin_memcpy(column(a.stats, col, a.ld_stats), st, sizeof(st));
      }
    }
  };
  if (EVEN && n == 8 * V * lanes) walk(std::integral_constant<bool, EVEN>{});
  else walk(std::false_type{});
}

// ------------------------------------------------------------------ backward
constexpr int kMergeRows = 3;

// A workgroup takes a contiguous range of columns; its teams (of 16 lanes or nw waves, one unit a
// thread) walk it with the next column's loads in flight and sum the gradients of weights and
// gate in registers.  At the end of the range, and for several gates at the end of each gate's
// columns, the teams' sums are merged through LDS and leave one partial row.
// BRANCH_NORM, GATE, BIAS: what there is to accumulate (BIAS: of any norm); GATE and BIAS may be
// set where there is none.  EVEN: the length is a multiple of eight and the epsilon a normal number.  STREAM: inputs
// past the caches.
//
// Entries that do not exist are loaded as zeros (partial units of what is normalised: as others of the column) and have
// zero weights, so that they add nothing to any sum that is kept and need no masks.
//
// Bound by HBM: 4096 x 8192 bf16 between two RMS norms with a gate, 384 MiB moved, in 76.8 us (5.2
// TB/s).  One workgroup a compute unit keeps the partial rows few (256 of them: 4.9 us to merge).
//
// TEAM: lanes of the largest team.  Up to 512 (256 registers a thread) the weights of a thread's unit stay in
// registers beside its up to five sums; teams of up to 1024 (128 registers) with many sums read the weights
// again for every column, from L2, and keep all sums but one in LDS.
template <typename T, int TEAM, bool BRANCH_NORM, bool GATE, bool BIAS, bool EVEN, bool STREAM>
__global__ void __launch_bounds__(TEAM <= 512 ? 512 : 1024)
rn_bwd_rows(RnBwdRows<T> a)
{
  using U = Unit<T>;
  constexpr bool SUB = TEAM == 16;
  constexpr bool kKeepWeights = TEAM <= 512 || (!GATE && (sizeof(T) == 2 ? !(BRANCH_NORM && BIAS) : !BRANCH_NORM));
  constexpr bool kLdsSums = !kKeepWeights;
  extern __shared__ __align__(16) float merged[];  // kMergeRows x blockDim x 8 floats if there are several teams
  // 16-byte pieces of the sums that are not in registers: piece i of thread t at [i][t]
  __shared__ v4f lds_sums[kLdsSums ? 2 * (kGrads - 1) : 1][kLdsSums ? TEAM : 1];
  __shared__ float* merged_rows[kMergeRows];
  __shared__ float2 slots[2][kMergeSlots];
  TeamMerge merge;
  const int n = a.n, nw = a.teams.nw, lanes = SUB ? 16 : kWave * nw;
  const Team<1, SUB> team(a.teams, n, slots, merge);
  const RowShare<1, EVEN> share(team.t, lanes, n);
  const int unit = share.unit[0], valid = share.valid[0], entry = 8 * unit, at = share.at[0], shift = share.shift[0];
  const int teams = a.teams.teams;
  const DropStream stream = drop_stream(a.drop);
  const bool dropping = a.drop.threshold < 65536u;
  const unsigned width = a.width;
  const bool several_gates = GATE && a.cols_per_gate < width;
  const bool output_norm = a.output_norm != kNormNone;
  const bool read_branch = BRANCH_NORM || (GATE && a.branch);
  const float epsilon = share.epsilon(0, a.epsilon);
  unsigned first, last;
  rn_range(blockIdx.x, width, a.cols_per_range, a.cols_per_gate, a.ranges_per_gate, first, last);

  auto weights = [&](const float* w, float fill, float (&out)[8]) {
    RowShare<1, EVEN> here = share;
    if constexpr (!kKeepWeights) asm volatile("" : "+v"(here.at[0]));  // read now: not kept from the last column
    here.weights(w, 0, fill, out);
  };
  float w2[8], w1[8], b1[8], gt[8];
  const float* gate_row = a.gate;
  auto load_output_weights = [&] { weights(a.output_scale, 1.f, w2); };
  auto load_branch_weights = [&] {
    if (BRANCH_NORM) weights(a.branch_scale, 1.f, w1);
    if (BRANCH_NORM && GATE && BIAS) weights(a.branch_bias, 0.f, b1);
  };
  auto load_gate = [&] {
    if (GATE) weights(gate_row, 1.f, gt);
  };
  if constexpr (kKeepWeights) {
    load_output_weights();
    load_branch_weights();
    load_gate();
  }

  float acc[kGrads][8] = {};
  // A thread's sum of quantity q: `next(j, sum)` is what entry j becomes.
  auto update = [&](auto quantity, auto next) {
    constexpr int q = decltype(quantity)::value;
    if constexpr (kLdsSums && q > 0) {
      v4f* const s = &lds_sums[2 * (q - 1)][threadIdx.x];
      v4f low = s[0], high = s[TEAM];
#pragma unroll
      for (int j = 0; j < 4; ++j) low[j] = next(j, low[j]), high[j] = next(4 + j, high[j]);
      s[0] = low, s[TEAM] = high;
    }
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[q][j] = next(j, acc[q][j]);
    }
  };
  if constexpr (kLdsSums) {
#pragma unroll
    for (int i = 0; i < 2 * (kGrads - 1); ++i) lds_sums[i][threadIdx.x] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  constexpr std::integral_constant<int, kGradOutputScale> output_scale_sum;
  constexpr std::integral_constant<int, kGradOutputBias> output_bias_sum;
  constexpr std::integral_constant<int, kGradBranchScale> branch_scale_sum;
  constexpr std::integral_constant<int, kGradBranchBias> branch_bias_sum;
  constexpr std::integral_constant<int, kGradGate> gate_sum;
  typename U::raw_t qy{}, qh{}, qs{}, qo{};
  RnColumnStats qstats{0.f, 1.f, 0.f, 1.f};
  auto issue = [&](unsigned col) {
    if (output_norm) {
      qy = U::template load<STREAM>(column(a.dy, col, a.ld_dy) + at);
      qs = U::template load<STREAM>(column(a.h, col, a.ld_h) + at);
    }
    if (a.dh) qh = U::template load<STREAM>(column(a.dh, col, a.ld_dh) + at);
    if (read_branch) qo = U::template load<STREAM>(column(a.branch, col, a.ld_branch) + at);
    if (BRANCH_NORM || output_norm) {
      const float* st = column(a.stats, col, a.ld_stats);
      qstats = {st[0], st[1], st[2], st[3]};  // variances, for now
    }
  };
  // The sums of the quantities from FIRST to LAST whose row is given, over all teams: one row each.
  // Several teams meet in LDS, kMergeRows rows at a time, in 16-byte pieces and by one piece of code for
  // all rows (one row after the other in single floats cost 1.5 us a row on short ranges).
  auto flush = [&](auto first_q, auto last_q, float* const (&rows)[kGrads]) {
    constexpr int kFirst = decltype(first_q)::value, kLast = decltype(last_q)::value;
    if (teams == 1) {
#pragma unroll
      for (int q = kFirst; q <= kLast; ++q) {
        if (!rows[q]) continue;
        if constexpr (kLdsSums) {
          if (q > 0) {
            const v4f low = lds_sums[2 * (q - 1)][threadIdx.x], high = lds_sums[2 * (q - 1) + 1][threadIdx.x];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[q][j] = low[j], acc[q][4 + j] = high[j];
          }
        }
        store_unit<EVEN>(rows[q] + entry, valid, acc[q]);
      }
    }
    else {
      const int stride = 8 * lanes, quads = (n + 3) / 4;
      auto round = [&](auto from_q, auto to_q) {
        int count = 0;
        __syncthreads();  // what was here has been read
#pragma unroll
        for (int q = decltype(from_q)::value; q <= decltype(to_q)::value; ++q) {
          if (rows[q]) {
            v4f* mine = reinterpret_cast<v4f*>(merged + (count * teams + team.index) * stride + 8 * team.t);
            mine[0] = v4f{acc[q][0], acc[q][1], acc[q][2], acc[q][3]};
            mine[1] = v4f{acc[q][4], acc[q][5], acc[q][6], acc[q][7]};
            if (threadIdx.x == 0) merged_rows[count] = rows[q];
            ++count;
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count * quads; i += static_cast<int>(blockDim.x)) {
          const int row = (i >= quads) + (i >= 2 * quads), k = 4 * (i - row * quads);
          const float* from = merged + row * teams * stride + k;
          v4f sum = *reinterpret_cast<const v4f*>(from);
#pragma unroll 3
          for (int j = 1; j < teams; ++j) sum += *reinterpret_cast<const v4f*>(from + j * stride);
          float* out = merged_rows[row] + k;
          if (EVEN || k + 4 <= n) {
            __builtin_memcpy(out, &sum, sizeof(sum));
          }
          else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
              if (k + j < n) out[j] = sum[j];
          }
        }
      };
      static_assert(kMergeRows == 3, "the row of a piece is found by two comparisons");
      constexpr int kMid = kFirst + kMergeRows - 1 < kLast ? kFirst + kMergeRows - 1 : kLast;
      round(std::integral_constant<int, kFirst>{}, std::integral_constant<int, kMid>{});
      if constexpr (kMid < kLast) round(std::integral_constant<int, kMid + 1>{}, std::integral_constant<int, kLast>{});
    }
  };

  bool in_flight = false;
  for (unsigned begin = first; begin < last;) {
    unsigned end = last, gate = 0;
    if (several_gates) {
      gate = begin / a.cols_per_gate;
      end = min(last, (gate + 1) * a.cols_per_gate);
      gate_row = column(a.gate, gate, a.ld_gate);
      if (kKeepWeights) load_gate();
    }
    unsigned col = begin + team.index;
    if (!in_flight && col < end) issue(col);
    for (unsigned turn = begin; turn < end; turn += teams, col += teams) {
      const bool active = col < end;
      float e[8], f[8], x[8];
      RnColumnStats s = qstats;
      s.rstd1 = BRANCH_NORM ? rn_rstd<!EVEN>(s.rstd1 + epsilon) : 1.f;
      s.rstd2 = rn_rstd<!EVEN>(s.rstd2 + epsilon);
      float o[8];
      U::template widen<EVEN>(qy, shift, f);
      U::template widen_centred<EVEN>(qs, shift, x);
      U::template widen<EVEN>(qh, shift, e);
      U::template widen_centred<EVEN>(qo, shift, o);
      // a single team carries the next column over the end of a gate's columns
      const unsigned next = col + teams;
      in_flight = teams == 1 && next < last;
      if (in_flight || next < end) issue(next);

      if (output_norm) {
        float sp = 0.f, spx = 0.f;
        if constexpr (!kKeepWeights) load_output_weights();
        if (active) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[j] = (x[j] - s.mean2) * s.rstd2;
          }
          update(output_scale_sum, [&](int j, float sum) { return __builtin_fmaf(f[j], x[j], sum); });
          if (BIAS) update(output_bias_sum, [&](int j, float sum) { return sum + f[j]; });
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            f[j] *= w2[j];
            sp += f[j];
            spx = __builtin_fmaf(f[j], x[j], spx);
          }
          sp = lanes_sum<SUB>(sp);
          spx = lanes_sum<SUB>(spx);
        }
        if (!SUB && nw > 1) merge.sum2(sp, spx);
        sp = a.output_norm == kNormLayer ? sp * team.inv_n : 0.f;
        spx *= team.inv_n;
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __builtin_fmaf(s.rstd2, f[j] - sp - x[j] * spx, e[j]);
      }
      if (active && a.dresidual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = a.residual_mult * e[j];
        store_unit<EVEN>(column(a.dresidual, col, a.ld_dresidual) + entry, valid, f);
      }
      // e becomes du; o the normalised branch
      if constexpr (!kKeepWeights) load_branch_weights();
      const float scale = dropping ? a.branch_mult * a.drop.inverse_keep : a.branch_mult;
      float ev[8];  // the gate's gradient
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (BRANCH_NORM) o[j] = (o[j] - s.mean1) * s.rstd1;
        e[j] *= scale;
        if (GATE) {
          const float u = BRANCH_NORM ? (BIAS ? __builtin_fmaf(o[j], w1[j], b1[j]) : o[j] * w1[j]) : o[j];
          ev[j] = e[j] * u;
        }
      }
      if constexpr (GATE) {
        if constexpr (!kKeepWeights) load_gate();
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] *= gt[j];
      }
      if (dropping) {
        uint32_t w[4];
        drop_words(a.drop, stream, unit, col, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool kept = drop_kept(w, j, a.drop.threshold);
          e[j] = kept ? e[j] : 0.f;
          if (GATE) ev[j] = kept ? ev[j] : 0.f;
        }
      }
      if (GATE && active && read_branch) update(gate_sum, [&](int j, float sum) { return sum + ev[j]; });
      if (BRANCH_NORM) {
        float sp = 0.f, spu = 0.f;
        if (active) {
          update(branch_scale_sum, [&](int j, float sum) { return __builtin_fmaf(e[j], o[j], sum); });
          if (BIAS) update(branch_bias_sum, [&](int j, float sum) { return sum + e[j]; });
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] *= w1[j];
            sp += e[j];
            spu = __builtin_fmaf(e[j], o[j], spu);
          }
          sp = lanes_sum<SUB>(sp);
          spu = lanes_sum<SUB>(spu);
        }
        if (!SUB && nw > 1) merge.sum2(sp, spu);
        sp = a.branch_norm == kNormLayer ? sp * team.inv_n : 0.f;
        spu *= team.inv_n;
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = s.rstd1 * (e[j] - sp - o[j] * spu);
      }
      if (active) store_unit<EVEN>(column(a.dbranch, col, a.ld_dbranch) + entry, valid, e);
    }
    if (GATE && a.dgate && a.ranges_per_gate == 0) {  // the gate's columns are all here
      float* rows[kGrads] = {};
      rows[kGradGate] = column(a.dgate, gate, a.ld_dgate);
      flush(std::integral_constant<int, kGradGate>{}, std::integral_constant<int, kGradGate>{}, rows);
      update(gate_sum, [](int, float) { return 0.f; });
    }
    begin = end;
  }
  float* rows[kGrads];
#pragma unroll
  for (int q = 0; q < kGrads; ++q) {
    const bool here = q == kGradOutputScale || (q == kGradOutputBias && BIAS) || (q == kGradBranchScale && BRANCH_NORM) ||
                      (q == kGradBranchBias && BRANCH_NORM && BIAS) || (q == kGradGate && GATE);
    rows[q] = here && a.part[q] ? column(a.part[q], blockIdx.x, n) : nullptr;
  }
  flush(std::integral_constant<int, 0>{}, std::integral_constant<int, kGradGate>{}, rows);
}

}  // namespace lbn
