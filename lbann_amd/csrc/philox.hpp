// The counter-based generator behind dropout: Philox-4x32 with ten rounds (Salmon, Moraes,
// Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC11).
//
// The random bits of an entry are a function of (seed, offset, row, column) and nothing else:
// key = seed, counter = (row / 8, column, offset low, offset high); the 128 bits of one counter
// serve the eight entries 8*(row/8) .. 8*(row/8)+7 of a column, sixteen bits each (word
// (row % 8) / 2, its low half for even rows).  So no mask is stored, backward repeats
// forward's bits, and the mask depends neither on leading dimensions nor on storage types nor on how
// a mini-batch is cut into calls (`column0` is the global index of the call's first column).
//
// Sixteen bits an entry: one counter costs twenty 32 x 32 -> 64-bit products, some 560 cycles of
// a wave, which eight 2-byte entries a lane read and written at HBM speed just cover; 32 bits an
// entry would make the generator, not the memory, the bound.  The price is that keep_prob is
// rounded to a multiple of 2^-16; outputs are scaled with the inverse of the rounded value, so
// that they stay unbiased.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace lbn {

struct DropArgs {
  uint32_t threshold;    // an entry is kept if its sixteen bits are below; 65536: nothing is dropped
  float inverse_keep;    // 65536 / threshold
  uint32_t key0, key1;
  uint64_t offset;
  const uint64_t* step;  // device counter added to the offset (captured graphs), or null
  uint32_t column0;
};

struct DropStream {  // what every entry of a call shares, resolved on the device
  uint32_t key0, key1, off0, off1;
};

__device__ __forceinline__ DropStream drop_stream(const DropArgs& d)
{
  const uint64_t off = d.offset + (d.step ? *d.step : 0);
  return {d.key0, d.key1, static_cast<uint32_t>(off), static_cast<uint32_t>(off >> 32)};
}

__device__ __forceinline__ void philox_4x32_10(uint32_t (&c)[4], uint32_t k0, uint32_t k1)
{
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c[0];
    const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c[2];
    const uint32_t odd1 = c[1], odd3 = c[3];
    c[0] = static_cast<uint32_t>(p1 >> 32) ^ odd1 ^ k0;
    c[1] = static_cast<uint32_t>(p1);
    c[2] = static_cast<uint32_t>(p0 >> 32) ^ odd3 ^ k1;
    c[3] = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// The four words for the group of eight rows `group` of column `col` (a local index).
__device__ __forceinline__ void drop_words(const DropArgs& d, const DropStream& s, uint32_t group, uint32_t col,
                                           uint32_t (&w)[4])
{
  w[0] = group;
  w[1] = d.column0 + col;
  w[2] = s.off0;
  w[3] = s.off1;
  philox_4x32_10(w, s.key0, s.key1);
}

// Whether entry j (0..7) of the group is kept.
__device__ __forceinline__ bool drop_kept(const uint32_t (&w)[4], int j, uint32_t threshold)
{
  const uint32_t bits = (j & 1) ? (w[j >> 1] >> 16) : (w[j >> 1] & 0xFFFFu);
  return bits < threshold;
}

// keep_prob as a number of 65536ths, at least one.
inline uint32_t drop_threshold(double keep_prob)
{
  const double t = std::floor(keep_prob * 65536.0 + 0.5);
  return t < 1.0 ? 1u : (t > 65536.0 ? 65536u : static_cast<uint32_t>(t));
}

inline DropArgs drop_args(double keep_prob, uint64_t seed, uint64_t offset, const uint64_t* step, int64_t column_offset)
{
  DropArgs d;
  d.threshold = drop_threshold(keep_prob);
  d.inverse_keep = static_cast<float>(65536.0 / d.threshold);
  d.key0 = static_cast<uint32_t>(seed);
  d.key1 = static_cast<uint32_t>(seed >> 32);
  d.offset = offset;
  d.step = step;
  d.column0 = static_cast<uint32_t>(column_offset);
  return d;
}

// Argument checks shared by every entry point that drops: the probability, and that the
// counter's 32-bit row group and column hold the matrix.
inline bool drop_probability_ok(double keep_prob) { return keep_prob > 0.0 && keep_prob <= 1.0; }  // false for NaN
inline bool drop_range_ok(int64_t height, int64_t width, int64_t column_offset)
{
  return height <= (int64_t(1) << 34) && column_offset <= (int64_t(1) << 32) - width;
}

}  // namespace lbn
