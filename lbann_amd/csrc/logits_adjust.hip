// Penalties for repeated tokens, bias lists and grammar masks on the logits of a batch of
// sequences, one pass over the logits (fp32, fp16 and bfloat16 storage, fp32 arithmetic).  For
// entry v of column s, with c the number of times v was generated and "seen" if v occurs in
// the prompt or was generated,
//
//   z = x;  seen: z = z > 0 ? z / repetition : z * repetition
//   z = z - (frequency c + presence [c > 0]) + bias_v;  z = -inf where the grammar forbids v.
//
// A workgroup takes a slab of one column: it counts the tokens of the sequence's history that
// fall into the slab in a table in LDS (integer atomics: the order does not matter), then streams the
// slab's logits through it.  Nothing is kept between calls and no table goes through memory:
// the history, a few thousand tokens, is read once per slab from the caches instead.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "storage.hpp"

namespace lbn {

constexpr int kLogitsThreads = 512;
constexpr uint32_t kInPrompt = 0x80000000u;  // beside the count of generated occurrences

template <typename T>
struct LogitsArgs {
  int64_t vocabulary, width;
  const T* x;
  int64_t ldx;
  T* y;
  int64_t ldy;
  const int32_t* tokens;
  int64_t ld_tokens, max_tokens;
  const int32_t *lengths, *prompt_lengths;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_tokens;
  const float* bias_values;
  int64_t ld_bias_tokens, ld_bias_values, num_biases;
  const uint32_t* mask;
  int64_t ld_mask, num_masks;
  const int32_t* mask_index;
  int slab;        // entries per workgroup, a multiple of 8
  int64_t slabs;   // per column
};

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads)
logits_adjust_slab(LogitsArgs<T> a)
{
  extern __shared__ uint32_t table[];  // occurrences of the slab's entries; behind them 1 + their bias list entry
  uint32_t* bias_at = table + a.slab;
  for (int64_t item = blockIdx.x; item < a.slabs * a.width; item += gridDim.x) {
    const int64_t col = item / a.slabs;
    const int64_t first = (item - col * a.slabs) * a.slab;
    const uint32_t here = static_cast<uint32_t>(imin64(a.slab, a.vocabulary - first));
    for (int i = threadIdx.x; i < a.slab; i += kLogitsThreads) {
      table[i] = 0;
      if (a.num_biases) bias_at[i] = 0;
    }
    __syncthreads();
    if (a.max_tokens) {
      // lengths are data: whatever they hold, only the max_tokens places of the column are read
      const int64_t length = a.lengths ? imin64(a.lengths[col], a.max_tokens) : a.max_tokens;
      const int64_t prompt = a.prompt_lengths ? a.prompt_lengths[col] : 0;
      const int32_t* history = a.tokens + col * a.ld_tokens;
      for (int64_t i = threadIdx.x; i < length; i += kLogitsThreads) {
        const int64_t at = history[i] - first;
        if (at >= 0 && at < here) {
          if (i < prompt) atomicOr(&table[at], kInPrompt);
          else atomicAdd(&table[at], 1u);
        }
      }
    }
    for (int64_t i = threadIdx.x; i < a.num_biases; i += kLogitsThreads) {
      const int64_t at = a.bias_tokens[col * a.ld_bias_tokens + i] - first;
      if (at >= 0 && at < here) atomicMax(&bias_at[at], static_cast<uint32_t>(i) + 1u);
    }
    __syncthreads();
    const float repetition = a.repetition ? a.repetition[col] : 1.f;
    const float presence = a.presence ? a.presence[col] : 0.f;
    const float frequency = a.frequency ? a.frequency[col] : 0.f;
    const uint32_t* mask = nullptr;
    bool all_forbidden = false;
    if (a.mask) {
      const int64_t index = a.mask_index ? a.mask_index[col] : (a.num_masks == 1 ? 0 : col);
      all_forbidden = index >= a.num_masks;  // no such grammar: nothing passes
      if (index >= 0 && !all_forbidden) mask = a.mask + index * a.ld_mask;
    }
    const T* x = a.x + col * a.ldx + first;
    T* y = a.y + col * a.ldy + first;
    for (uint32_t k = 8 * threadIdx.x; k < here; k += 8 * kLogitsThreads) {
      float v[8];
      load8(x + k, here - k, v);
      uint32_t allowed = all_forbidden ? 0u : 0xFFu;
      if (mask) allowed = mask[(first + k) >> 5] >> ((first + k) & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t t = table[k + j];
        if (t) {
          v[j] = v[j] > 0.f ? v[j] / repetition : v[j] * repetition;
          const uint32_t c = t & ~kInPrompt;
          v[j] -= frequency * static_cast<float>(c) + (c ? presence : 0.f);
        }
        if (a.num_biases) {
          const uint32_t b = bias_at[k + j];
          if (b) v[j] += a.bias_values[col * a.ld_bias_values + b - 1];
        }
        if (!(allowed >> j & 1u)) v[j] = -INFINITY;
      }
      store8(y + k, here - k, v);
    }
    __syncthreads();
  }
}

template <typename T>
static int logits_adjust(lbn_stream_t stream, LogitsArgs<T> a)
{
  if (a.vocabulary < 0 || a.width < 0 || a.max_tokens < 0 || a.num_biases < 0 || a.num_masks < 0) return LBN_ERR_INVALID_ARGUMENT;
  if (a.vocabulary == 0 || a.width == 0) return LBN_OK;
  const bool many = a.width > 1;
  if (!a.x || !a.y || (many && (a.ldx < a.vocabulary || a.ldy < a.vocabulary))) return LBN_ERR_INVALID_ARGUMENT;
  if (a.max_tokens && (!a.tokens || (many && a.ld_tokens < a.max_tokens))) return LBN_ERR_INVALID_ARGUMENT;
  if (a.num_biases && (!a.bias_tokens || !a.bias_values ||
                       (many && (a.ld_bias_tokens < a.num_biases || a.ld_bias_values < a.num_biases))))
    return LBN_ERR_INVALID_ARGUMENT;
  if ((a.num_masks > 0) != (a.mask != nullptr) || (a.num_masks > 1 && a.ld_mask < ceil_div(a.vocabulary, 32)) ||
      (a.num_masks > 1 && !a.mask_index && a.num_masks != a.width))
    return LBN_ERR_INVALID_ARGUMENT;
  const int64_t limit = (int64_t(1) << 31) - 1;
  if (a.vocabulary > limit || a.max_tokens > limit || a.num_biases >= limit) return LBN_ERR_UNSUPPORTED;
  a.slab = 4096;
  a.slabs = ceil_div(a.vocabulary, a.slab);
  const int64_t items = a.slabs * a.width;
  const unsigned grid = static_cast<unsigned>(items < (int64_t(1) << 30) ? items : (int64_t(1) << 30));
  const unsigned lds = static_cast<unsigned>(a.slab * sizeof(uint32_t) * (a.num_biases ? 2 : 1));
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL((logits_adjust_slab<T>), dim3(grid), dim3(kLogitsThreads), lds, st, a);
  return launch_status();
}

}  // namespace lbn

extern "C" {

#define LBN_LOGITS_ADJUST_ENTRY(SUFFIX, ABI, T)                                                                      \
  int lbn_logits_adjust_##SUFFIX(                                                                                    \
    lbn_stream_t stream, int64_t vocabulary, int64_t width, const ABI* x, int64_t ldx, ABI* y, int64_t ldy,          \
    const int32_t* tokens, int64_t ld_tokens, int64_t max_tokens, const int32_t* lengths,                            \
    const int32_t* prompt_lengths, const float* repetition, const float* presence, const float* frequency,           \
    const int32_t* bias_tokens, int64_t ld_bias_tokens, const float* bias_values, int64_t ld_bias_values,            \
    int64_t num_biases, const uint32_t* mask, int64_t ld_mask, int64_t num_masks, const int32_t* mask_index)         \
  {                                                                                                                  \
    lbn::LogitsArgs<T> a{};                                                                                          \
    a.vocabulary = vocabulary, a.width = width;                                                                      \
    a.x = static_cast<const T*>(x), a.ldx = ldx, a.y = static_cast<T*>(y), a.ldy = ldy;                              \
    a.tokens = tokens, a.ld_tokens = ld_tokens, a.max_tokens = max_tokens;                                           \
    a.lengths = lengths, a.prompt_lengths = prompt_lengths;                                                          \
    a.repetition = repetition, a.presence = presence, a.frequency = frequency;                                       \
    a.bias_tokens = bias_tokens, a.ld_bias_tokens = ld_bias_tokens;                                                  \
    a.bias_values = bias_values, a.ld_bias_values = ld_bias_values, a.num_biases = num_biases;                       \
    a.mask = mask, a.ld_mask = ld_mask, a.num_masks = num_masks, a.mask_index = mask_index;                          \
    return lbn::logits_adjust<T>(stream, a);                                                                         \
  }

LBN_LOGITS_ADJUST_ENTRY(f32, float, float)
LBN_LOGITS_ADJUST_ENTRY(f16, void, lbn::f16_t)
LBN_LOGITS_ADJUST_ENTRY(bf16, void, lbn::bf16_t)

#undef LBN_LOGITS_ADJUST_ENTRY

}  // extern "C"
