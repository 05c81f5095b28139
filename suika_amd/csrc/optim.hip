// optim.hip -- the optimizer's part of a training step over a share's
// tensors (C ABI in include/suika_step.h): the sum of the gradients' squares,
// clipping, and the AdamW update.
//
// Every call works on a list of arrays of any length.  The list goes to the
// kernels by value, in tables of up to 4 KB of kernel arguments, so nothing is
// uploaded and nothing is kept between calls; a longer list takes several
// launches.  Arrays are cut into chunks of a fixed number of elements, numbered
// through the table.  A wave finds the array of a chunk by comparing all first
// chunks at once, a few of them a lane: one vector load on the way to the
// addresses, and nothing in memory beside the arguments.
//
// HBM bounds all of it but the smallest calls.  The figures below are of one
// MI355X; where the arrays of a state lie in HBM moves an update by up to 6%
// from one process to the next.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <new>
#include <type_traits>
#include <vector>

#include "suika_step.h"
#include "sr_step.h"

namespace {

using namespace sr_step;

constexpr int kThreads = 256;

// A table of 4 KB, less the 256 bytes of arguments that the compiler adds.
constexpr size_t kTableBytes = 3832;

// Most chunks of one launch: a grid has fewer than 2^32 threads, with 512 of
// them a chunk and chunks rounded up to the dies half of that.
constexpr uint32_t kMostChunks = 1u << 22;

// Where the chunks of a table's entries start.
template <int ENTRIES>
struct Chunks {
  static constexpr int kEach = (ENTRIES + kWave - 1) / kWave;     // entries of a lane
  static_assert(ENTRIES % kEach == 0, "a lane's entries are loaded together");

  uint32_t first[ENTRIES];       // rises strictly: empty arrays are left out
  uint32_t count;                // entries
  uint32_t chunks;

  void clear() {
    count = chunks = 0;
    for (uint32_t& f : first) f = 0xffffffffu;
  }
  bool room(uint64_t n, uint32_t chunk) const {
    return count < ENTRIES && (count == 0 || chunks + (n + chunk - 1) / chunk <= kMostChunks);
  }
  // Takes an array of n elements; returns its entry.
  uint32_t add(uint64_t n, uint32_t chunk) {
    first[count] = chunks;
    chunks += uint32_t((n + chunk - 1) / chunk);
    return count++;
  }

  // The entry of chunk c, and where it and the next one start.
  struct Found {
    uint32_t entry, from, to;
  };

  __device__ __forceinline__ Found find(uint32_t c) const {
    const int lane = threadIdx.x % kWave;
    const bool in = lane < ENTRIES / kEach;
    uint32_t f[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) f[k] = first[(in ? lane : 0) * kEach + k];
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) n += uint32_t(__popcll(__ballot(in && f[k] <= c)));
    Found r;
    r.entry = __builtin_amdgcn_readfirstlane(n) - 1;
    r.from = at(f, r.entry);
    r.to = r.entry + 1 < ENTRIES ? at(f, r.entry + 1) : 0xffffffffu;
    r.to = r.to < chunks ? r.to : chunks;
    return r;
  }

 private:
  __device__ __forceinline__ static uint32_t at(const uint32_t (&f)[kEach], uint32_t i) {
    uint32_t x = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t y = __builtin_amdgcn_readlane(f[k], i / kEach);
      x = i % kEach == k ? y : x;
    }
    return x;
  }
};

// ------------------------------------------------------------ sum of squares

// sum += x^2 over all elements, in 64 bits: squares of f32 values neither
// overflow nor vanish there, and each product of two 24-bit numbers is exact.
// The sums of workgroups are added by a second launch in a fixed order.  1.88 GB
// of bf16 take 270 us, 7.0 TB/s: eight 16-byte loads a lane are on their way at
// once, and a workgroup takes consecutive chunks (chunks dealt out to 2048
// workgroups that stay: 341 us).
constexpr int kSumEntries = 189;
constexpr uint32_t kSumChunk = 32768;      // elements
constexpr uint32_t kSumBlocks = 16384;     // workgroups of one launch at most

// Loads stream past the caches (2.56 GB of bf16 372 us, cached 422; 320 MB of
// f32 51.5, cached 58), unless the arrays are read again soon and are not much
// more than the 256 MB memory-side cache: then the next reader finds part of
// them there (clipping 320 MB of f32 into other tensors, norm included, 151 us
// with cached loads, 159 with streamed ones; 640 MB 307 and 310; 1.28 GB 627
// and 618).
constexpr uint64_t kSumCached = uint64_t(1) << 30;

struct SumTable {
  struct Entry { uint64_t data, n; } entry[kSumEntries];
  Chunks<kSumEntries> at;
};
static_assert(sizeof(SumTable) <= kTableBytes, "kernel arguments");
static_assert(SR_STEP_MAX_ELEMENTS / kSumChunk <= kMostChunks, "an array fits into a launch");

constexpr int kFinishThreads = 1024;

template <int THREADS>
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[THREADS / kWave];
  x = wave_sum(x);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int i = 0; i < THREADS / kWave; ++i) s += part[i];
  return s;
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(kThreads) void square_sum_kernel(uint32_t run, uint32_t chunks, double* partial,
                                                             SumTable t) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kBatch = 8;
  double sum[4] = {0, 0, 0, 0};
  const uint32_t end = min((blockIdx.x + 1) * run, chunks);
  for (uint32_t c = blockIdx.x * run; c < end; ++c) {
    const auto found = t.at.find(c);
    const uint32_t i = found.entry;
    const uint64_t at = uint64_t(c - found.from) * kSumChunk;
    const uint64_t left = t.entry[i].n - at;
    const uint32_t n = left < kSumChunk ? uint32_t(left) : kSumChunk;
    const T* p = global<const T>(t.entry[i].data) + at;
    uint32_t e = threadIdx.x * N;
    for (; e + (kBatch - 1) * kThreads * N + N <= n; e += kBatch * kThreads * N) {
      Vec<T, N> x[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const Vec<T, N>* v = reinterpret_cast<const Vec<T, N>*>(p + e + b * kThreads * N);
        x[b] = STREAM ? __builtin_nontemporal_load(v) : *v;
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const double d = double(float(x[b][k]));
          sum[k & 3] = fma(d, d, sum[k & 3]);
        }
    }
    for (; e + N <= n; e += kThreads * N) {
      float x[N];
      load<T, N>(p + e, x);
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k & 3] = fma(double(x[k]), double(x[k]), sum[k & 3]);
    }
    const uint32_t rest = n - n % N;     // the elements behind the last whole vector, one a lane
    if (threadIdx.x < n % N) {
      const double x = double(float(p[rest + threadIdx.x]));
      sum[0] = fma(x, x, sum[0]);
    }
  }
  const double s = block_sum<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kFinishThreads) void finish_sum_kernel(const double* partial, uint32_t count, double* sum,
                                                                    float* norm) {
  constexpr uint32_t kAhead = 4;
  double x = 0;
  uint32_t i = threadIdx.x;
  for (; i + (kAhead - 1) * kFinishThreads < count; i += kAhead * kFinishThreads) {
    double p[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) p[a] = partial[i + a * kFinishThreads];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) x += p[a];
  }
  for (; i < count; i += kFinishThreads) x += partial[i];
  x = block_sum<kFinishThreads>(x);
  if (threadIdx.x == 0) {
    *sum = x;
    if (norm) *norm = float(sqrt(x));
  }
}

// The whole sum of few elements in one workgroup and one launch: its waves take
// the arrays in turn.  24 arrays of 300 f32 elements: 6.8 us a call, 9.1 with
// two launches; at 96000 elements two launches are as fast (9.0).
constexpr uint64_t kSmallElements = 32768;

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void small_sum_kernel(double* sum, float* norm, SumTable t) {
  constexpr int N = 16 / sizeof(T);
  double x = 0;
  for (uint32_t i = threadIdx.x / kWave; i < t.at.count; i += kFinishThreads / kWave) {
    const T* p = global<const T>(t.entry[i].data);
    const uint32_t n = uint32_t(t.entry[i].n);
    for (uint32_t e = threadIdx.x % kWave * N; e < n; e += kWave * N) {
      if (e + N <= n) {
        float v[N];
        load<T, N>(p + e, v);
#pragma unroll
        for (int k = 0; k < N; ++k) x = fma(double(v[k]), double(v[k]), x);
      } else {
        for (uint32_t k = e; k < n; ++k) x = fma(double(float(p[k])), double(float(p[k])), x);
      }
    }
  }
  x = block_sum<kFinishThreads>(x);
  if (threadIdx.x == 0) {
    *sum = x;
    if (norm) *norm = float(sqrt(x));
  }
}

// ------------------------------------------------------------------ clipping

// A copy with a factor that every workgroup forms from the sum: 325 MB of bf16
// into 650 MB of f32 in 146 us (6.6 TB/s), the norm before it 50.
constexpr int kClipEntries = 128;
constexpr uint32_t kClipChunk = 4096;

struct ClipTable {
  struct Entry { uint64_t src, dst, n; } entry[kClipEntries];
  Chunks<kClipEntries> at;
  float max_norm;
  const double* square_sum;
  float* norm;
};
static_assert(sizeof(ClipTable) <= kTableBytes, "kernel arguments");
static_assert(SR_STEP_MAX_ELEMENTS / kClipChunk <= kMostChunks, "an array fits into a launch");
static_assert(uint64_t(kMostChunks) * kThreads < uint64_t(1) << 32, "a grid's threads");

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN.
__device__ __forceinline__ float clip_factor(double square_sum, float max_norm) {
  const double f = double(max_norm) / (sqrt(square_sum) + 1e-6);
  return f > 1.0 ? 1.0f : float(f);
}

template <typename S, typename D>
__global__ __launch_bounds__(kThreads) void clip_kernel(ClipTable t) {
  constexpr int N = 4;
  constexpr int kBatch = kClipChunk / (kThreads * N);
  const double q = *t.square_sum;
  if (t.norm && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = float(sqrt(q));
  if (t.at.count == 0) return;
  const uint32_t c = blockIdx.x;
  const auto found = t.at.find(c);
  const uint32_t i = found.entry;
  const float f = clip_factor(q, t.max_norm);
  if (f == 1.0f && t.entry[i].dst == t.entry[i].src) return;
  const uint64_t at = uint64_t(c - found.from) * kClipChunk;
  const uint64_t left = t.entry[i].n - at;
  const uint32_t n = left < kClipChunk ? uint32_t(left) : kClipChunk;
  const S* src = global<const S>(t.entry[i].src) + at;
  D* dst = global<D>(t.entry[i].dst) + at;
  float x[kBatch][N];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const uint32_t e = (b * kThreads + threadIdx.x) * N;
    if (e + N <= n) load_stream<S, N>(src + e, x[b]);
  }
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const uint32_t e = (b * kThreads + threadIdx.x) * N;
    if (e + N <= n) {
#pragma unroll
      for (int k = 0; k < N; ++k) x[b][k] *= f;
      store_stream<D, N>(dst + e, x[b]);
    } else {
      for (uint32_t k = e; k < n; ++k) dst[k] = D(float(src[k]) * f);
    }
  }
}

// --------------------------------------------------------------------- AdamW

constexpr int kAdamThreads = 512;
constexpr uint32_t kAdamChunk = 2048;
constexpr uint64_t kAdamPart = uint64_t(kMostChunks) * kAdamChunk;     // elements of one entry: longer arrays have several
static_assert(uint64_t(kMostChunks + kXcds) * kAdamThreads < uint64_t(1) << 32, "a grid's threads");

// What a table holds of one parameter; without a copy of the weight, one
// address less.
template <bool COPY> struct AdamEntry { uint64_t weight, exp_avg, exp_avg_sq, grad, param; };
template <> struct AdamEntry<false> { uint64_t weight, exp_avg, exp_avg_sq, grad; };

template <bool COPY>
struct AdamTable {
  static constexpr int kEntries = COPY ? 80 : 96;
  AdamEntry<COPY> entry[kEntries];
  Chunks<kEntries> at;
  uint16_t tail[kEntries];        // elements of the last chunk
  const double* square_sum;
  float max_norm;
  float decay;                    // 1 - lr * weight_decay
  float beta1, rest1, beta2, rest2;
  float step_size;                // lr / (1 - beta1^step)
  float root_scale;               // 1 / sqrt(1 - beta2^step)
  float eps;
};
static_assert(sizeof(AdamTable<true>) <= kTableBytes && sizeof(AdamTable<false>) <= kTableBytes, "kernel arguments");

struct NoCopy {};

// One chunk a workgroup, one vector of every field a lane, all loads before the
// first store.  Chunks go to the dies by eighths (xcd_order).  That pays for the
// largest states and costs the smaller ones: TB/s of the 28 bytes an element
// that are read and written, by eighths / in plain order, of 40, 200, 400 and 936 M
// elements in 100 tensors: f32 5.5 / 6.1, 5.8 / 5.7, 5.8 / 5.6, 5.8 / 5.7; mixed
// 5.6 / 6.0, 5.5 / 5.7, 5.6 / 5.6, 5.7 / 5.4.  Loads and stores stream: with stores that
// write through the L2 the update itself is as fast or 3% faster, but the next
// kernel's reads wait for what they left in the memory-side cache (GPT-125M's
// share with clipping 238 us a step, streamed 212).
// W: type of the weight, M: of the moments, G: of the gradient, P: of the
// weight's copy, or NoCopy.
template <typename W, typename M, typename G, typename P>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(uint32_t chunks,
                                                             AdamTable<!__is_same(P, NoCopy)> t) {
  constexpr int N = kAdamChunk / kAdamThreads;
  const uint32_t c = xcd_order(blockIdx.x, chunks);
  if (c >= chunks) return;
  const auto found = t.at.find(c);
  const uint32_t i = found.entry;
  const uint32_t n = c + 1 == found.to ? t.tail[i] : kAdamChunk;
  const uint64_t at = uint64_t(c - found.from) * kAdamChunk;
  W* weight = global<W>(t.entry[i].weight) + at;
  M* exp_avg = global<M>(t.entry[i].exp_avg) + at;
  M* exp_avg_sq = global<M>(t.entry[i].exp_avg_sq) + at;
  const G* grad = global<const G>(t.entry[i].grad) + at;

  const uint32_t e = threadIdx.x * N;
  const bool whole = e + N <= n;
  float g[N], w[N], m[N], v[N];
  if (whole) {
    load_stream<G, N>(grad + e, g);
    load_stream<W, N>(weight + e, w);
    load_stream<M, N>(exp_avg + e, m);
    load_stream<M, N>(exp_avg_sq + e, v);
  }
  const float factor = t.square_sum ? clip_factor(*t.square_sum, t.max_norm) : 1.0f;
  auto update = [&](float gi, float& wi, float& mi, float& vi) {
    gi *= factor;
    mi = fmaf(mi, t.beta1, gi * t.rest1);
    vi = fmaf(vi, t.beta2, gi * gi * t.rest2);
    const float root = fmaf(sqrtf(vi), t.root_scale, t.eps);
    wi = fmaf(wi, t.decay, -(t.step_size * mi) / root);
  };
  if (whole) {
#pragma unroll
    for (int k = 0; k < N; ++k) update(g[k], w[k], m[k], v[k]);
    store_stream<W, N>(weight + e, w);
    store_stream<M, N>(exp_avg + e, m);
    store_stream<M, N>(exp_avg_sq + e, v);
    if constexpr (!__is_same(P, NoCopy)) store_stream<P, N>(global<P>(t.entry[i].param) + at + e, w);
  } else {
    for (uint32_t k = e; k < n; ++k) {
      float wi = float(weight[k]), mi = float(exp_avg[k]), vi = float(exp_avg_sq[k]);
      update(float(grad[k]), wi, mi, vi);
      weight[k] = W(wi);
      exp_avg[k] = M(mi);
      exp_avg_sq[k] = M(vi);
      if constexpr (!__is_same(P, NoCopy)) (global<P>(t.entry[i].param) + at)[k] = P(wi);
    }
  }
}

// ---------------------------------------------------------------------- host

int check_arrays(const char* who, const sr_array* a, int32_t count) {
  if (count < 0 || (count > 0 && a == nullptr)) return fail(SR_EINVAL, "%s: no arrays", who);
  for (int32_t i = 0; i < count; ++i) {
    if (a[i].reserved != 0) return fail(SR_EINVAL, "%s: arrays[%d].reserved is not 0", who, i);
    if (!float_dtype(a[i].dtype)) return fail(SR_EDTYPE, "%s: arrays[%d]: dtype %d", who, i, a[i].dtype);
    if (a[i].n > SR_STEP_MAX_ELEMENTS)
      return fail(SR_EBOUNDS, "%s: arrays[%d] has %llu elements", who, i, (unsigned long long)a[i].n);
    if (a[i].n && a[i].data == nullptr) return fail(SR_EINVAL, "%s: arrays[%d] is null", who, i);
    if (reinterpret_cast<uintptr_t>(a[i].data) % sr_internal::dtype_size(a[i].dtype))
      return fail(SR_EALIGN, "%s: arrays[%d] is not aligned to its elements", who, i);
  }
  return SR_OK;
}

uint64_t bytes_of(const sr_array& a) { return a.n * sr_internal::dtype_size(a.dtype); }

// Memory that a call reads or writes.
struct Span {
  uintptr_t from, to;
  bool written;
};

void add_span(std::vector<Span>& spans, const void* p, uint64_t bytes, bool written) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  if (p && bytes) spans.push_back({a, a + bytes, written});
}

// By address.  A state's fields mostly lie in the order of its tensors, field by
// field, so the spans come in a few ascending runs, which are merged: the checks
// stand before the first launch, where the GPU waits for them (147 tensors of
// four fields 6 us in all on this host, sorted 21).
void sort_spans(std::vector<Span>& spans) {
  auto before = [](const Span& a, const Span& b) { return a.from < b.from; };
  auto next_run = [&](auto from) { return std::is_sorted_until(from, spans.end(), before); };
  for (int passes = 0;; ++passes) {
    auto from = spans.begin(), mid = next_run(from);
    if (mid == spans.end()) return;
    if (passes == 4) return std::sort(from, spans.end(), before);
    while (mid != spans.end()) {
      const auto to = next_run(mid);
      std::inplace_merge(from, mid, to, before);
      from = to;
      mid = next_run(from);
    }
  }
}

// Whether anything written overlaps anything else.
bool clash(std::vector<Span>& spans) {
  sort_spans(spans);
  uintptr_t any = 0, written = 0;    // ends of what came before
  for (const Span& s : spans) {
    if (s.from < (s.written ? any : written)) return true;
    any = std::max(any, s.to);
    if (s.written) written = std::max(written, s.to);
  }
  return false;
}

constexpr int32_t kFloatTypes[3] = {SR_DT_F32, SR_DT_BF16, SR_DT_F16};

// Launches of a list: the arrays of one type at a time, as many as a table takes.
template <typename F>
int sum_launches(const sr_array* a, int32_t count, F&& launch) {
  for (int32_t dt : kFloatTypes) {
    SumTable t;
    t.at.clear();
    auto flush = [&]() -> int {
      if (t.at.count == 0) return SR_OK;
      const int rc = launch(dt, t);
      t.at.clear();
      return rc;
    };
    for (int32_t i = 0; i < count; ++i) {
      if (a[i].dtype != dt || a[i].n == 0) continue;
      if (!t.at.room(a[i].n, kSumChunk)) {
        if (int rc = flush()) return rc;
      }
      t.entry[t.at.add(a[i].n, kSumChunk)] = {reinterpret_cast<uint64_t>(a[i].data), a[i].n};
    }
    if (int rc = flush()) return rc;
  }
  return SR_OK;
}

// Consecutive chunks of one workgroup, and the workgroups.
uint32_t sum_run(const SumTable& t) { return (t.at.chunks + kSumBlocks - 1) / kSumBlocks; }
uint32_t sum_blocks(const SumTable& t) { return (t.at.chunks + sum_run(t) - 1) / sum_run(t); }

template <typename T>
void launch_sum(const SumTable& t, uint32_t run, uint32_t blocks, bool stream_loads, double* partial,
                hipStream_t stream) {
  if (stream_loads) square_sum_kernel<T, true><<<blocks, kThreads, 0, stream>>>(run, t.at.chunks, partial, t);
  else square_sum_kernel<T, false><<<blocks, kThreads, 0, stream>>>(run, t.at.chunks, partial, t);
}

template <typename S, typename D>
void launch_clip(const ClipTable& t, hipStream_t stream) {
  clip_kernel<S, D><<<t.at.chunks, kThreads, 0, stream>>>(t);
}

template <typename S>
void launch_clip_to(int32_t dst, const ClipTable& t, hipStream_t stream) {
  if (dst == SR_DT_F32) launch_clip<S, float>(t, stream);
  else if (dst == SR_DT_BF16) launch_clip<S, bf16>(t, stream);
  else launch_clip<S, f16>(t, stream);
}

template <typename W, typename M, typename G, bool COPY>
void launch_adamw_of(const AdamTable<COPY>& t, hipStream_t stream) {
  typedef typename std::conditional<COPY, bf16, NoCopy>::type P;
  adamw_kernel<W, M, G, P><<<xcd_blocks(t.at.chunks), kAdamThreads, 0, stream>>>(t.at.chunks, t);
}

// The tensors whose fields have the types W, M and G, and a copy or none.
template <typename W, typename M, typename G, bool COPY>
int adamw_launches(const sr_adamw_tensor* tensors, int32_t count, AdamTable<COPY> t, hipStream_t stream) {
  auto code = [](bool wide) { return wide ? SR_DT_F32 : SR_DT_BF16; };
  const int32_t weight = code(__is_same(W, float)), moment = code(__is_same(M, float)), grad = code(__is_same(G, float));
  t.at.clear();
  auto flush = [&]() -> int {
    if (t.at.count == 0) return SR_OK;
    launch_adamw_of<W, M, G, COPY>(t, stream);
    t.at.clear();
    return launched("sr_adamw");
  };
  for (int32_t i = 0; i < count; ++i) {
    const sr_adamw_tensor& x = tensors[i];
    if (x.n == 0 || x.weight_dtype != weight || x.moment_dtype != moment || x.grad_dtype != grad ||
        (x.param != nullptr) != COPY)
      continue;
    for (uint64_t from = 0; from < x.n; from += kAdamPart) {
      const uint64_t n = std::min(x.n - from, kAdamPart);
      if (!t.at.room(n, kAdamChunk)) {
        if (int rc = flush()) return rc;
      }
      const uint32_t k = t.at.add(n, kAdamChunk);
      auto& e = t.entry[k];
      e.weight = reinterpret_cast<uint64_t>(x.weight) + from * sizeof(W);
      e.exp_avg = reinterpret_cast<uint64_t>(x.exp_avg) + from * sizeof(M);
      e.exp_avg_sq = reinterpret_cast<uint64_t>(x.exp_avg_sq) + from * sizeof(M);
      e.grad = reinterpret_cast<uint64_t>(x.grad) + from * sizeof(G);
      if constexpr (COPY) e.param = reinterpret_cast<uint64_t>(x.param) + from * sizeof(bf16);
      t.tail[k] = uint16_t(n - (n - 1) / kAdamChunk * kAdamChunk);
    }
  }
  return flush();
}

// Without launches for the types that no tensor has.
template <typename W, bool COPY>
int adamw_types(const sr_adamw_tensor* tensors, int32_t count, const AdamTable<COPY>& t, hipStream_t stream) {
  if (int rc = adamw_launches<W, float, float, COPY>(tensors, count, t, stream)) return rc;
  if (int rc = adamw_launches<W, float, bf16, COPY>(tensors, count, t, stream)) return rc;
  if (int rc = adamw_launches<W, bf16, float, COPY>(tensors, count, t, stream)) return rc;
  return adamw_launches<W, bf16, bf16, COPY>(tensors, count, t, stream);
}

template <bool COPY>
void adamw_scalars(AdamTable<COPY>& t, const sr_adamw_options& o, int64_t step, const double* square_sum) {
  t.square_sum = square_sum;
  t.max_norm = square_sum ? float(o.max_norm) : 0.0f;
  t.decay = float(1 - o.lr * o.weight_decay);
  t.beta1 = float(o.beta1);
  t.rest1 = float(1 - o.beta1);
  t.beta2 = float(o.beta2);
  t.rest2 = float(1 - o.beta2);
  t.step_size = float(o.lr / (1 - std::pow(o.beta1, double(step))));
  t.root_scale = float(1 / std::sqrt(1 - std::pow(o.beta2, double(step))));
  t.eps = float(o.eps);
}

// ------------------------------------------------------- checks, then launches

// The bytes of a workspace for the sum of checked arrays.
uint64_t sum_workspace(const sr_array* arrays, int32_t count) {
  uint64_t blocks = 0;
  sum_launches(arrays, count, [&](int32_t, const SumTable& t) {
    blocks += sum_blocks(t);
    return SR_OK;
  });
  return blocks * sizeof(double);
}

int check_sum(const char* who, const sr_array* arrays, int32_t count, const void* workspace, uint64_t workspace_bytes,
              const double* sum, const float* norm, uint64_t* bytes = nullptr) {
  if (int rc = check_arrays(who, arrays, count)) return rc;
  const uint64_t need = sum_workspace(arrays, count);
  if (bytes) *bytes = need;
  if (sum == nullptr) return fail(SR_EINVAL, "%s: sum is null", who);
  if (workspace_bytes < need || (need && workspace == nullptr))
    return fail(SR_EINVAL, "%s: a workspace of %llu bytes, %llu are needed", who, (unsigned long long)workspace_bytes,
                (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 || reinterpret_cast<uintptr_t>(sum) % 8 ||
      reinterpret_cast<uintptr_t>(norm) % 4)
    return fail(SR_EALIGN, "%s: the workspace or a result is not aligned", who);
  return SR_OK;
}

int launch_square_sum(const sr_array* arrays, int32_t count, bool read_again, void* workspace, double* sum, float* norm,
                      hipStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  uint32_t used = 0;
  uint64_t bytes = 0;
  for (int32_t i = 0; i < count; ++i) bytes += bytes_of(arrays[i]);
  uint64_t elements = 0;
  int32_t tables = 0;
  for (int32_t i = 0; i < count; ++i) elements += arrays[i].n;
  const bool stream_loads = !read_again || bytes > kSumCached;
  if (elements <= kSmallElements) {
    sum_launches(arrays, count, [&](int32_t, const SumTable&) {
      ++tables;
      return SR_OK;
    });
  }
  const bool small = tables == 1;
  const int rc = sum_launches(arrays, count, [&](int32_t dt, const SumTable& t) {
    if (small) {
      if (dt == SR_DT_F32) small_sum_kernel<float><<<1, kFinishThreads, 0, stream>>>(sum, norm, t);
      else if (dt == SR_DT_BF16) small_sum_kernel<bf16><<<1, kFinishThreads, 0, stream>>>(sum, norm, t);
      else small_sum_kernel<f16><<<1, kFinishThreads, 0, stream>>>(sum, norm, t);
      return launched("sr_square_sum");
    }
    const uint32_t blocks = sum_blocks(t), run = sum_run(t);
    if (dt == SR_DT_F32) launch_sum<float>(t, run, blocks, stream_loads, partial + used, stream);
    else if (dt == SR_DT_BF16) launch_sum<bf16>(t, run, blocks, stream_loads, partial + used, stream);
    else launch_sum<f16>(t, run, blocks, stream_loads, partial + used, stream);
    used += blocks;
    return launched("sr_square_sum");
  });
  if (rc || small) return rc;
  finish_sum_kernel<<<1, kFinishThreads, 0, stream>>>(partial, used, sum, norm);
  return launched("sr_square_sum");
}

// What a norm takes: the sum that is given, or the place and the workspace for
// that of the gradients.  Adds its memory to `spans`.
int check_norm(const char* who, const sr_norm& n, const sr_array* grads, int32_t count, std::vector<Span>& spans) {
  add_span(spans, n.norm, sizeof(float), true);
  if (n.square_sum == nullptr) {
    uint64_t need = 0;
    if (int rc = check_sum(who, grads, count, n.workspace, n.workspace_bytes, n.sum, n.norm, &need)) return rc;
    add_span(spans, n.sum, sizeof(double), true);
    add_span(spans, n.workspace, need, true);
    return SR_OK;
  }
  if (reinterpret_cast<uintptr_t>(n.square_sum) % 8 || reinterpret_cast<uintptr_t>(n.norm) % 4)
    return fail(SR_EALIGN, "%s: square_sum or norm is not aligned", who);
  add_span(spans, n.square_sum, sizeof(double), false);
  return SR_OK;
}

// *norm = sqrt(*square_sum), with nothing to clip.
int launch_norm(const char* who, const double* square_sum, float* norm, hipStream_t stream) {
  ClipTable t;
  t.at.clear();
  t.at.chunks = 1;
  t.max_norm = 0;
  t.square_sum = square_sum;
  t.norm = norm;
  launch_clip<float, float>(t, stream);
  return launched(who);
}

int clip(const char* who, const sr_array* src, const sr_array* dst, int32_t count, float max_norm, const sr_norm& n,
         hipStream_t stream) try {
  if (int rc = check_arrays(who, src, count)) return rc;
  if (dst != nullptr) {
    if (int rc = check_arrays(who, dst, count)) return rc;
  }
  std::vector<Span> spans;
  spans.reserve(2 * size_t(count) + 4);
  if (int rc = check_norm(who, n, src, count, spans)) return rc;
  if (!(max_norm >= 0)) return fail(SR_EINVAL, "%s: max_norm %g", who, double(max_norm));
  if (dst == nullptr) dst = src;
  for (int32_t i = 0; i < count; ++i) {
    if (src[i].n != dst[i].n)
      return fail(SR_EINVAL, "%s: src[%d] has %llu elements, dst[%d] %llu", who, i, (unsigned long long)src[i].n, i,
                  (unsigned long long)dst[i].n);
    add_span(spans, dst[i].data, bytes_of(dst[i]), true);
  }
  for (int32_t i = 0; i < count; ++i)
    if (src[i].data != dst[i].data || src[i].dtype != dst[i].dtype)
      add_span(spans, src[i].data, bytes_of(src[i]), false);
  if (clash(spans)) return fail(SR_EOVERLAP, "%s: an array or a value that is written overlaps another", who);
  const double* square_sum = n.square_sum;
  if (square_sum == nullptr) {
    if (int rc = launch_square_sum(src, count, true, n.workspace, n.sum, nullptr, stream)) return rc;
    square_sum = n.sum;
  }
  bool any = false;
  for (int32_t s : kFloatTypes) {
    for (int32_t d : kFloatTypes) {
      ClipTable t;
      t.at.clear();
      t.max_norm = max_norm;
      t.square_sum = square_sum;
      auto flush = [&]() -> int {
        if (t.at.count == 0) return SR_OK;
        t.norm = any ? nullptr : n.norm;
        any = true;
        if (s == SR_DT_F32) launch_clip_to<float>(d, t, stream);
        else if (s == SR_DT_BF16) launch_clip_to<bf16>(d, t, stream);
        else launch_clip_to<f16>(d, t, stream);
        t.at.clear();
        return launched(who);
      };
      for (int32_t i = 0; i < count; ++i) {
        if (src[i].dtype != s || dst[i].dtype != d || src[i].n == 0) continue;
        if (!t.at.room(src[i].n, kClipChunk)) {
          if (int rc = flush()) return rc;
        }
        t.entry[t.at.add(src[i].n, kClipChunk)] = {reinterpret_cast<uint64_t>(src[i].data),
                                                   reinterpret_cast<uint64_t>(dst[i].data), src[i].n};
      }
      if (int rc = flush()) return rc;
    }
  }
  return any || n.norm == nullptr ? int(SR_OK) : launch_norm(who, square_sum, n.norm, stream);
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "%s: out of host memory", who);
}

// One update of checked tensors, all of the same step.
int launch_adamw(const sr_adamw_tensor* tensors, int32_t count, const sr_adamw_options& o, int64_t step,
                 const double* square_sum, hipStream_t stream) {
  AdamTable<true> with_copy;
  AdamTable<false> alone;
  adamw_scalars(with_copy, o, step, square_sum);
  adamw_scalars(alone, o, step, square_sum);
  if (int rc = adamw_types<float, true>(tensors, count, with_copy, stream)) return rc;
  if (int rc = adamw_types<float, false>(tensors, count, alone, stream)) return rc;
  return adamw_types<bf16, false>(tensors, count, alone, stream);
}

int adamw(const char* who, const sr_adamw_tensor* tensors, const int64_t* steps, int32_t count,
          const sr_adamw_options* o, const sr_norm* n, hipStream_t stream) try {
  if (count < 0 || (count > 0 && tensors == nullptr) || o == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (!(o->lr >= 0) || !std::isfinite(o->lr) || !(o->eps >= 0) || !(o->weight_decay >= 0) || !(o->beta1 >= 0) ||
      !(o->beta1 < 1) || !(o->beta2 >= 0) || !(o->beta2 < 1) || (steps == nullptr && o->step < 1))
    return fail(SR_EINVAL, "%s: lr %g, betas %g and %g, eps %g, weight_decay %g, step %lld", who, o->lr, o->beta1,
                o->beta2, o->eps, o->weight_decay, (long long)o->step);
  if (n != nullptr && !(o->max_norm >= 0)) return fail(SR_EINVAL, "%s: max_norm %g", who, o->max_norm);
  std::vector<Span> spans;
  std::vector<sr_array> grads;      // where their sum of squares is formed here
  const bool own_sum = n != nullptr && n->square_sum == nullptr;
  spans.reserve(5 * size_t(count) + 4);
  if (own_sum) grads.reserve(size_t(count));
  for (int32_t i = 0; i < count; ++i) {
    const sr_adamw_tensor& x = tensors[i];
    if (x.reserved != 0) return fail(SR_EINVAL, "%s: tensors[%d].reserved is not 0", who, i);
    if (steps != nullptr && steps[i] < 1) return fail(SR_EINVAL, "%s: steps[%d] is %lld", who, i, (long long)steps[i]);
    for (int32_t dt : {x.weight_dtype, x.moment_dtype, x.grad_dtype})
      if (dt != SR_DT_F32 && dt != SR_DT_BF16) return fail(SR_EDTYPE, "%s: tensors[%d]: dtype %d", who, i, dt);
    if (x.param != nullptr && x.weight_dtype != SR_DT_F32)
      return fail(SR_EDTYPE, "%s: tensors[%d]: a copy of a weight that is not f32", who, i);
    if (x.n > SR_STEP_MAX_ELEMENTS)
      return fail(SR_EBOUNDS, "%s: tensors[%d] has %llu elements", who, i, (unsigned long long)x.n);
    if (x.n && (!x.weight || !x.exp_avg || !x.exp_avg_sq || !x.grad))
      return fail(SR_EINVAL, "%s: tensors[%d]: a field is null", who, i);
    const int ws = sr_internal::dtype_size(x.weight_dtype), ms = sr_internal::dtype_size(x.moment_dtype),
              gs = sr_internal::dtype_size(x.grad_dtype);
    const struct { const void* p; int size; } field[5] = {
        {x.weight, ws}, {x.exp_avg, ms}, {x.exp_avg_sq, ms}, {x.param, 2}, {x.grad, gs}};
    for (const auto& f : field)
      if (reinterpret_cast<uintptr_t>(f.p) % f.size)
        return fail(SR_EALIGN, "%s: tensors[%d]: a field is not aligned to its elements", who, i);
    if (own_sum) grads.push_back({const_cast<void*>(x.grad), x.n, x.grad_dtype, 0});
  }
  if (n != nullptr) {
    if (int rc = check_norm(who, *n, grads.data(), int32_t(grads.size()), spans)) return rc;
  }
  auto size = [](int32_t dt) { return dt == SR_DT_F32 ? 4 : 2; };
  for (int32_t i = 0; i < count; ++i) add_span(spans, tensors[i].weight, tensors[i].n * size(tensors[i].weight_dtype), true);
  for (int32_t i = 0; i < count; ++i) add_span(spans, tensors[i].exp_avg, tensors[i].n * size(tensors[i].moment_dtype), true);
  for (int32_t i = 0; i < count; ++i)
    add_span(spans, tensors[i].exp_avg_sq, tensors[i].n * size(tensors[i].moment_dtype), true);
  for (int32_t i = 0; i < count; ++i) add_span(spans, tensors[i].param, tensors[i].n * 2, true);
  for (int32_t i = 0; i < count; ++i) add_span(spans, tensors[i].grad, tensors[i].n * size(tensors[i].grad_dtype), false);
  if (clash(spans)) return fail(SR_EOVERLAP, "%s: a field or a value that is written overlaps another", who);
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  SR_STEP_TRY(hipStreamIsCapturing(stream, &capturing));
  if (capturing != hipStreamCaptureStatusNone)
    return fail(SR_EINVAL, "%s: the step number is a host value: the call cannot be captured", who);
  const double* square_sum = nullptr;
  if (own_sum) {
    square_sum = n->sum;
    if (int rc = launch_square_sum(grads.data(), int32_t(grads.size()), true, n->workspace, n->sum, n->norm, stream))
      return rc;
  } else if (n != nullptr) {
    square_sum = n->square_sum;
    if (n->norm != nullptr) {
      if (int rc = launch_norm(who, square_sum, n->norm, stream)) return rc;
    }
  }
  if (steps == nullptr) return launch_adamw(tensors, count, *o, o->step, square_sum, stream);
  if (std::adjacent_find(steps, steps + count, std::not_equal_to<int64_t>()) == steps + count)
    return count ? launch_adamw(tensors, count, *o, steps[0], square_sum, stream) : int(SR_OK);
  // the tensors of one step after those of another, each in launches of its own
  std::vector<int32_t> order(size_t(count), 0);
  for (int32_t i = 0; i < count; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int32_t a, int32_t b) { return steps[a] < steps[b]; });
  std::vector<sr_adamw_tensor> sorted;
  for (int32_t i : order) sorted.push_back(tensors[i]);
  for (int32_t from = 0, to; from < count; from = to) {
    for (to = from; to < count && steps[order[to]] == steps[order[from]];) ++to;
    if (int rc = launch_adamw(&sorted[from], to - from, *o, steps[order[from]], square_sum, stream)) return rc;
  }
  return SR_OK;
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "%s: out of host memory", who);
}

}  // namespace

extern "C" {

int sr_square_sum_workspace(const sr_array* arrays, int32_t count, uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_square_sum_workspace: null argument");
  if (int rc = check_arrays("sr_square_sum_workspace", arrays, count)) return rc;
  *bytes = sum_workspace(arrays, count);
  return SR_OK;
}

int sr_square_sum(const sr_array* arrays, int32_t count, int32_t read_again, void* workspace, uint64_t workspace_bytes,
                  double* sum, float* norm, hipStream_t stream) {
  uint64_t need = 0;
  if (int rc = check_sum("sr_square_sum", arrays, count, workspace, workspace_bytes, sum, norm, &need)) return rc;
  const Extent written[3] = {{sum, sizeof(double)}, {norm, sizeof(float)}, {workspace, need}};
  bool meets = written[0].meets(written[1]) || written[0].meets(written[2]) || written[1].meets(written[2]);
  for (int32_t i = 0; i < count; ++i) {
    const Extent array{arrays[i].data, bytes_of(arrays[i])};
    for (const Extent& w : written) meets = meets || w.meets(array);
  }
  if (meets) return fail(SR_EOVERLAP, "sr_square_sum: a result or the workspace overlaps other memory of the call");
  return launch_square_sum(arrays, count, read_again != 0, workspace, sum, norm, stream);
}

int sr_clip(const sr_array* src, const sr_array* dst, int32_t count, const double* square_sum, float max_norm,
            float* norm, hipStream_t stream) {
  if (square_sum == nullptr) return fail(SR_EINVAL, "sr_clip: square_sum is null");
  const sr_norm given{square_sum, nullptr, nullptr, 0, norm};
  return clip("sr_clip", src, dst, count, max_norm, given, stream);
}

int sr_clip_norm(const sr_array* src, const sr_array* dst, int32_t count, float max_norm, const sr_norm* norm,
                 hipStream_t stream) {
  if (norm == nullptr) return fail(SR_EINVAL, "sr_clip_norm: norm is null");
  return clip("sr_clip_norm", src, dst, count, max_norm, *norm, stream);
}

int sr_adamw(const sr_adamw_tensor* tensors, int32_t count, const sr_adamw_options* o, const double* square_sum,
             hipStream_t stream) {
  const sr_norm given{square_sum, nullptr, nullptr, 0, nullptr};
  return adamw("sr_adamw", tensors, nullptr, count, o, square_sum ? &given : nullptr, stream);
}

int sr_adamw_norm(const sr_adamw_tensor* tensors, const int64_t* steps, int32_t count, const sr_adamw_options* o,
                  const sr_norm* norm, hipStream_t stream) {
  return adamw("sr_adamw_norm", tensors, steps, count, o, norm, stream);
}

}  // extern "C"
