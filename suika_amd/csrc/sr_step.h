// sr_step.h -- what the kernels of the training-step operators share (not
// part of the C ABI): element types, 16-byte vectors at element alignment and
// reductions over a wave or a workgroup.
#ifndef SR_STEP_H
#define SR_STEP_H

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sr_internal.h"

namespace sr_step {

using sr_internal::fail;

#define SR_STEP_TRY(expr)                                                                          \
  do {                                                                                             \
    hipError_t e_ = (expr);                                                                        \
    if (e_ != hipSuccess) return sr_internal::fail(SR_EHIP, "%s failed: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

constexpr int kWave = 64;

typedef __bf16 bf16;
typedef _Float16 f16;

// Vectors of N elements that are aligned as one element is: the hardware takes
// 16-byte accesses at any address.
template <typename T, int N> struct VecAt {
  typedef T packed __attribute__((ext_vector_type(N)));
  typedef packed type __attribute__((aligned(alignof(T))));
};
template <typename T, int N> using Vec = typename VecAt<T, N>::type;

template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float (&f)[N]) {
  const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = static_cast<float>(v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void load_stream(const T* p, float (&f)[N]) {
  const Vec<T, N> v = __builtin_nontemporal_load(reinterpret_cast<const Vec<T, N>*>(p));
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = static_cast<float>(v[i]);
}

// Rounds to nearest even where T is narrower.
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&f)[N]) {
  Vec<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = static_cast<T>(f[i]);
  *reinterpret_cast<Vec<T, N>*>(p) = v;
}

template <typename T, int N>
__device__ __forceinline__ void store_stream(T* p, const float (&f)[N]) {
  Vec<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = static_cast<T>(f[i]);
  __builtin_nontemporal_store(v, reinterpret_cast<Vec<T, N>*>(p));
}

template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SR_OK : fail(SR_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace sr_step

#endif  // SR_STEP_H
