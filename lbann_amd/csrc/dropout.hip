// Dropout from a counter-based generator (philox.hpp), forward and backward, fp32, fp16 and
// bfloat16 storage:  y = keep(row, column) ? x / q : 0,  dx = keep(row, column) ? dy / q : 0
// with the same keep(): one kernel serves both directions.
//
// A thread owns eight consecutive entries of a column, the unit of one counter.  Dropped
// entries are selected away, not multiplied by zero, so that an infinity or a NaN in a dropped
// place does not reach the output.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "philox.hpp"
#include "storage.hpp"

namespace lbn {

constexpr int kDropThreads = 256;

template <typename T>
constexpr int kDropUnits = sizeof(T) == 2 ? 2 : 1;

// `lanes` threads (a power of two) work on a column side by side, UNITS groups of eight each, and
// kDropThreads / lanes columns side by side in a workgroup.  Bound by HBM: two groups of 2-byte
// entries a thread, both loaded before the first is worked on, keep enough bytes in flight while the
// generator runs (4096 x 8192 bf16: 21.7 us, 6.2 TB/s, against 27.2 with one and 22.5 with four; 1001 x
// 20000: 15.7, 19.9, 16.5).  One group of fp32 entries is as many bytes (1001 x 20000: 28.2 us, 30.2 with two).
template <typename T>
__global__ void __launch_bounds__(kDropThreads)
dropout_apply(const T* x, int64_t ldx, T* y, int64_t ldy, int64_t height, int64_t width, int lanes, DropArgs drop)
{
  constexpr int UNITS = kDropUnits<T>;
  const int64_t groups = (height + 7) / 8;
  const int columns = kDropThreads / lanes;
  const int64_t tiles = (groups + UNITS * lanes - 1) / (UNITS * lanes);
  const int64_t strips = (width + columns - 1) / columns;
  const DropStream stream = drop_stream(drop);
  const int lane = static_cast<int>(threadIdx.x) & (lanes - 1);
  const int sub = static_cast<int>(threadIdx.x) / lanes;
  for (int64_t item = blockIdx.x; item < tiles * strips; item += gridDim.x) {
    const int64_t strip = item / tiles;
    const int64_t first = (item - strip * tiles) * UNITS * lanes + lane;
    const int64_t col = strip * columns + sub;
    if (col >= width) continue;
    float v[UNITS][8];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int64_t row = 8 * (first + i * lanes);
      if (row < height) load8(x + col * ldx + row, height - row, v[i]);
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int64_t group = first + i * lanes, row = 8 * group;
      if (row >= height) continue;
      if (drop.threshold < 65536u) {
        uint32_t w[4];
        drop_words(drop, stream, static_cast<uint32_t>(group), static_cast<uint32_t>(col), w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = drop_kept(w, k, drop.threshold) ? v[i][k] * drop.inverse_keep : 0.f;
      }
      store8(y + col * ldy + row, height - row, v[i]);
    }
  }
}

template <typename T>
static int dropout_launch(lbn_stream_t stream, int64_t height, int64_t width, double keep_prob, uint64_t seed,
                          uint64_t offset, const uint64_t* step, int64_t column_offset, const T* x, int64_t ldx, T* y,
                          int64_t ldy)
{
  if (height < 0 || width < 0 || column_offset < 0 || !drop_probability_ok(keep_prob)) return LBN_ERR_INVALID_ARGUMENT;
  if (height == 0 || width == 0) return LBN_OK;
  if (!x || !y || (width > 1 && (ldx < height || ldy < height))) return LBN_ERR_INVALID_ARGUMENT;
  if (!drop_range_ok(height, width, column_offset)) return LBN_ERR_UNSUPPORTED;
  hipStream_t st = as_stream(stream);
  const int64_t groups = ceil_div(height, 8);
  constexpr int units = kDropUnits<T>;
  int lanes = 1;
  while (units * lanes < groups && lanes < kDropThreads) lanes *= 2;
  const int64_t items = ceil_div(groups, units * lanes) * ceil_div(width, kDropThreads / lanes);
  hipLaunchKernelGGL((dropout_apply<T>), dim3(walking_grid(items)), dim3(kDropThreads), 0, st, x, ldx, y, ldy, height, width, lanes,
                     drop_args(keep_prob, seed, offset, step, column_offset));
  return launch_status();
}

}  // namespace lbn

extern "C" {

#define LBN_DROPOUT_ENTRY(NAME, ABI, T)                                                                              \
  int NAME(lbn_stream_t stream, int64_t height, int64_t width, double keep_prob, uint64_t seed, uint64_t offset,     \
           const uint64_t* step, int64_t column_offset, const ABI* x, int64_t ldx, ABI* y, int64_t ldy)              \
  {                                                                                                                  \
    return lbn::dropout_launch<T>(stream, height, width, keep_prob, seed, offset, step, column_offset,               \
                                  static_cast<const T*>(x), ldx, static_cast<T*>(y), ldy);                           \
  }

LBN_DROPOUT_ENTRY(lbn_dropout_fwd_f32, float, float)
LBN_DROPOUT_ENTRY(lbn_dropout_fwd_f16, void, lbn::f16_t)
LBN_DROPOUT_ENTRY(lbn_dropout_fwd_bf16, void, lbn::bf16_t)
LBN_DROPOUT_ENTRY(lbn_dropout_bwd_f32, float, float)
LBN_DROPOUT_ENTRY(lbn_dropout_bwd_f16, void, lbn::f16_t)
LBN_DROPOUT_ENTRY(lbn_dropout_bwd_bf16, void, lbn::bf16_t)

#undef LBN_DROPOUT_ENTRY

}  // extern "C"
