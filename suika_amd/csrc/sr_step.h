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

// A device address out of a table of kernel arguments: known to be global
// memory, which a flat access would not be.
template <typename T>
__device__ __forceinline__ T* global(uint64_t address) {
  typedef __attribute__((address_space(1))) T* Global;
  return (T*)(Global)address;
}

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

// Memory from an address on as a buffer resource, for stores with a cache
// policy: 32-bit offsets, and what lies outside `bytes` is dropped.
typedef __amdgpu_buffer_rsrc_t Region;

__device__ __forceinline__ Region region(void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, int(bytes), 0x00027000);
}

constexpr int kThrough = 16;     // sc1: whole lines go through the L2

template <int POLICY, typename T, int N>
__device__ __forceinline__ void store_region(Region r, uint32_t at, const float (&f)[N]) {
  static_assert(N * sizeof(T) == 16, "a whole vector");
  typename VecAt<T, N>::packed v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = static_cast<T>(f[i]);
  typedef unsigned int Words __attribute__((ext_vector_type(4)));
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Words, v), r, at, 0, POLICY);
}

template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// Eight values of a row, n of which exist.
template <typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[8], uint32_t n) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      store<T, 8>(p, v);
    } else {
      const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
      store<T, 4>(p, lo);
      store<T, 4>(p + 4, hi);
    }
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
      if (e < n) p[e] = static_cast<T>(v[e]);
  }
}

template <typename T>
__device__ __forceinline__ void load_row(const T* p, float (&v)[8], uint32_t n) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      load<T, 8>(p, v);
    } else {
      float lo[4], hi[4];
      load<T, 4>(p, lo);
      load<T, 4>(p + 4, hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
    }
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = e < n ? static_cast<float>(p[e]) : 0.0f;
  }
}

// The factor that gradients are clipped by: min(1, max_norm / (norm + 1e-6));
// NaN stays NaN.
__device__ __forceinline__ float clip_factor(double square_sum, float max_norm) {
  const double f = double(max_norm) / (sqrt(square_sum) + 1e-6);
  return f > 1.0 ? 1.0f : float(f);
}

// Work items in the order of memory, an eighth of them for each of the 8 dies
// that workgroups go to in turn: the items in flight then come from 8 distant
// regions.  A grid of xcd_blocks(items), of which some have no item.
constexpr uint32_t kXcds = 8;
__host__ __device__ inline uint32_t xcd_blocks(uint32_t items) { return (items + kXcds - 1) / kXcds * kXcds; }
__device__ __forceinline__ uint32_t xcd_order(uint32_t block, uint32_t items) {
  return block % kXcds * ((items + kXcds - 1) / kXcds) + block / kXcds;
}

inline bool float_dtype(int32_t dt) { return dt == SR_DT_F32 || dt == SR_DT_BF16 || dt == SR_DT_F16; }

// Memory that a call reads or writes.
struct Extent {
  const void* p;
  uint64_t bytes;

  bool meets(const Extent& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
    return p && o.p && bytes && o.bytes && a < b + o.bytes && b < a + bytes;
  }
};

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SR_OK : fail(SR_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace sr_step

#endif  // SR_STEP_H
