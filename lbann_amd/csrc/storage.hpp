// Storage types of the operators around the residual stream and the logits: fp32, IEEE
// binary16 and bfloat16, always widened to fp32 registers.
//
// Vectors are 16 bytes at the alignment of ONE entry: gfx950 takes a 16-byte access at any
// entry boundary with the same instruction (256 MiB copies: 5.1 to 5.2 TB/s off the 16-byte
// grid against 5.4 to 5.5 on it), so one kernel serves every leading dimension and every
// buffer offset.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace lbn {

using f16_t = _Float16;
using bf16_t = __bf16;

template <typename T>
struct Pack {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));

  static __device__ __forceinline__ vec_t load(const T* p) { return *reinterpret_cast<const vec_t*>(p); }
  static __device__ __forceinline__ void widen(const vec_t& r, float (&v)[N])
  {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = static_cast<float>(r[k]);
  }
  // Round to nearest even, once, at the store.
  static __device__ __forceinline__ void store(T* p, const float (&v)[N])
  {
    vec_t r;
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = static_cast<T>(v[k]);
    __builtin_nontemporal_store(r, reinterpret_cast<vec_t*>(p));
  }
};

// Eight consecutive entries, the unit the generator works in; `valid` of them exist (the rest
// reads as 0 and is not written).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t valid, float (&v)[8])
{
  constexpr int N = Pack<T>::N;
  if (valid >= 8) {
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      float t[N];
      Pack<T>::widen(Pack<T>::load(p + i), t);
#pragma unroll
      for (int k = 0; k < N; ++k) v[i + k] = t[k];
    }
  }
  else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < valid ? static_cast<float>(p[k]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t valid, const float (&v)[8])
{
  constexpr int N = Pack<T>::N;
  if (valid >= 8) {
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      float t[N];
#pragma unroll
      for (int k = 0; k < N; ++k) t[k] = v[i + k];
      Pack<T>::store(p + i, t);
    }
  }
  else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < valid) p[k] = static_cast<T>(v[k]);
  }
}

}  // namespace lbn
