// Penalties for repeated tokens, bias lists and grammar masks on the logits of a batch of
// sequences, one pass over the logits (fp32, fp16 and bfloat16 storage, fp32 arithmetic).  For
// entry v of column s, with c the number of times v was generated and "seen" if v occurs in
// the prompt or was generated,
//
//   z = x;  seen: z = z > 0 ? z / repetition : z * repetition
//   z = z - (frequency c + presence [c > 0]) + bias_v;  z = -inf where the grammar forbids v.
//
// A workgroup takes a slab of one column, U units of eight entries a thread: it counts the tokens
// of the sequence's history that fall into the slab in a table in LDS (integer atomics: their order
// does not matter), then passes the slab's logits through it.  Nothing is kept between calls and no
// table goes through memory: the history, a few thousand tokens, is read once per slab instead, from
// the L2 of the die that has all slabs of the column.  Bound by latency rather than by bytes, so
// the logits, the mask and the first tokens are all asked for before anything waits: 32768 x 512 fp16 with
// 2048 tokens, 64 biases and grammars in 23.4 us (3.1 TB/s; 15.5 us without a history).
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "storage.hpp"

namespace lbn {

// A table word holds, from below: the count of generated occurrences (count_bits), 1 + the place
// in the bias list, whether the entry occurs in the prompt.
constexpr uint32_t kInPrompt = 0x80000000u;

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
  unsigned slabs;  // per column
  int count_bits;
};

template <typename T, int U>
__global__ void __launch_bounds__(1024)
logits_adjust_slab(LogitsArgs<T> a)
{
  typedef T raw_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  typedef int32_t four_t __attribute__((ext_vector_type(4), aligned(4)));
  extern __shared__ uint32_t table[];  // one word for every entry of the slab
  const unsigned threads = blockDim.x, slab = 8 * U * threads, tid = threadIdx.x;
  const unsigned item = item_of_block_by_die(blockIdx.x, gridDim.x);
  const unsigned col = item / a.slabs;
  const int first = static_cast<int>((item - col * a.slabs) * slab);
  const unsigned here = min(slab, static_cast<unsigned>(a.vocabulary) - first);
  const T* x = a.x + col * a.ldx + first;
  T* y = a.y + col * a.ldy + first;
  const int max_tokens = static_cast<int>(a.max_tokens), biases = static_cast<int>(a.num_biases);

  raw_t q[U];
  uint32_t allowed[U];
  const uint32_t* mask = nullptr;
  bool none_allowed = false;
  if (a.mask) {
    const int64_t index = a.mask_index ? a.mask_index[col] : (a.num_masks == 1 ? 0 : static_cast<int64_t>(col));
    none_allowed = index >= a.num_masks;  // no such grammar: nothing passes
    if (index >= 0 && !none_allowed) mask = a.mask + index * a.ld_mask;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const unsigned k = 8 * (tid + i * threads);
    if (k + 8 <= here) q[i] = *reinterpret_cast<const raw_t*>(x + k);
    allowed[i] = none_allowed ? 0u : 0xFFu;
    if (mask && k < here) allowed[i] = mask[(first + k) >> 5] >> ((first + k) & 31);
  }
  const int32_t* history = a.tokens + col * a.ld_tokens;
  // Four tokens from place `at` on, in one load: near the end of the column from further back, and the places
  // before `at`, which are another thread's, do not count then.
  const int last_load = max_tokens - 4;
  auto tokens_at = [&](int at) {
    four_t t = {-1, -1, -1, -1};
    if (last_load >= 0) {
      if (at < max_tokens) t = *reinterpret_cast<const four_t*>(history + min(at, last_load));
    }
    else if (at == 0) {
      for (int j = 0; j < max_tokens; ++j) t[3 - j] = history[max_tokens - 1 - j];  // as if from place `last_load`
    }
    return t;
  };
  const int stride = 4 * static_cast<int>(threads);
  four_t t = tokens_at(4 * tid);
  const int32_t* bias_tokens = a.bias_tokens + col * a.ld_bias_tokens;
  int bias_token = static_cast<int>(tid) < biases ? bias_tokens[tid] : -1;
  // lengths are data: whatever they hold, only the max_tokens places of the column are read
  const int length = max_tokens ? (a.lengths ? min(a.lengths[col], max_tokens) : max_tokens) : 0;
  const int prompt = max_tokens && a.prompt_lengths ? a.prompt_lengths[col] : 0;
  const float repetition = a.repetition ? a.repetition[col] : 1.f;
  const float presence = a.presence ? a.presence[col] : 0.f;
  const float frequency = a.frequency ? a.frequency[col] : 0.f;

  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (unsigned i = tid; i < slab / 4; i += threads) reinterpret_cast<uint4*>(table)[i] = zero;
  __syncthreads();
  if (biases) {  // before the counts: the larger place wins, and there is nothing below it yet
    for (int i = tid; i < biases;) {
      const unsigned entry = static_cast<unsigned>(bias_token) - first;
      if (entry < here && bias_token >= 0) atomicMax(&table[entry], static_cast<uint32_t>(i + 1) << a.count_bits);
      i += static_cast<int>(threads);
      if (i < biases) bias_token = bias_tokens[i];
    }
    __syncthreads();
  }
  for (int own = 4 * static_cast<int>(tid); own < length;) {
    const four_t now = t;
    const int at = own, from = min(at, last_load);
    own += stride;
    if (own < length) t = tokens_at(own);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned entry = static_cast<unsigned>(now[j]) - first;
      if (entry < here && now[j] >= 0 && from + j >= at && from + j < length) {
        if (from + j < prompt) atomicOr(&table[entry], kInPrompt);
        else atomicAdd(&table[entry], 1u);
      }
    }
  }
  __syncthreads();

#pragma unroll
  for (int i = 0; i < U; ++i) {
    const unsigned k = 8 * (tid + i * threads);
    if (k >= here) continue;
    float v[8];
    if (k + 8 <= here) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(q[i][j]);
    }
    else {
      load8(x + k, here - k, v);
    }
    uint32_t word[8], any = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) any |= word[j] = table[k + j];
    if (any) {
      const uint32_t count_mask = (1u << a.count_bits) - 1u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t c = word[j] & count_mask;
        if (word[j] & (kInPrompt | count_mask)) {
          v[j] = v[j] > 0.f ? v[j] / repetition : v[j] * repetition;
          v[j] -= frequency * static_cast<float>(c) + (c ? presence : 0.f);
        }
        const uint32_t listed = (word[j] & ~kInPrompt) >> a.count_bits;
        if (listed) v[j] += a.bias_values[col * a.ld_bias_values + listed - 1];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = allowed[i] >> j & 1u ? v[j] : -INFINITY;
    store8(y + k, here - k, v);
  }
}

// Every slab reads the whole history, so long histories take large slabs, and many threads to read
// them; short ones take small workgroups, which start and end sooner.  us by threads x units:
//                                     256x1   512x1   512x2   1024x2
//   131072 x 64 fp16,   128 tokens     11.5    12.1    12.2    12.2
//    32768 x 512 fp16, 2048 tokens     24.6    24.1    23.2    23.0
//   131072 x 64 fp16,  4096 tokens     15.1    14.4    14.5    13.9
//   262144 x 16 bf16, 16384 tokens     14.5    12.1    11.5    10.2
//    50257 x 1 fp32,    300 tokens      4.4     4.8     5.8     6.5
struct LogitsShape {
  int threads, units;
  int slab() const { return 8 * units * threads; }
};

static LogitsShape logits_shape(int64_t max_tokens)
{
  if (max_tokens >= 4096) return {1024, 2};
  if (max_tokens >= 1024) return {512, 2};
  return {256, 1};
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
  if (a.vocabulary > limit - (1 << 14) || a.width > limit || a.max_tokens > limit - (1 << 14) || a.num_biases > limit)
    return LBN_ERR_UNSUPPORTED;
  while ((int64_t(1) << a.count_bits) <= a.max_tokens) ++a.count_bits;
  if (a.num_biases >> (31 - a.count_bits)) return LBN_ERR_UNSUPPORTED;
  const LogitsShape shape = logits_shape(a.max_tokens);
  a.slabs = static_cast<unsigned>(ceil_div(a.vocabulary, shape.slab()));
  if (a.slabs * a.width * shape.threads > limit) return LBN_ERR_UNSUPPORTED;  // threads of a launch
  const dim3 grid(static_cast<unsigned>(a.slabs * a.width));
  const unsigned lds = static_cast<unsigned>(shape.slab() * sizeof(uint32_t));
  hipStream_t st = as_stream(stream);
  if (shape.units == 1) hipLaunchKernelGGL((logits_adjust_slab<T, 1>), grid, dim3(shape.threads), lds, st, a);
  else hipLaunchKernelGGL((logits_adjust_slab<T, 2>), grid, dim3(shape.threads), lds, st, a);
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
