// logprob.hip -- log probabilities of given tokens, entropy and the best
// alternatives from a head's logits, and the gradient of the logits (C ABI in
// include/suika_step.h).
//
// With d = (x - M) log2 e for a running maximum M, one pass over a row keeps
//   s = sum 2^d   and   w = sum d 2^d,
// so that lse = M + ln s and entropy = ln s - ln 2 w / s.  When M grows by D
// (in units of log2), s <- s 2^-D and w <- 2^-D (w - D s).  Every lane keeps
// its own M, s and w; they are joined once per row.
//
// A workgroup takes a row, with four 16-byte loads a lane on their way while
// four are taken in.  HBM bounds rows of f32 (2047 x 50304 in 62 us, 6.65 TB/s);
// rows of bf16 (8192 x 32000 in 91 us, 5.8 TB/s) come near what the vector units
// give: about ten instruction slots a logit, four of them its exponential.
//
// The alternatives come from a second look at few of the logits: the k-th
// largest of 64 lane groups' maxima is a bound that at least k logits reach,
// and only the groups whose maximum reaches it are read again, their vectors
// dealt out to all lanes.  The logits that reach it are ranked against each
// other; equal ones by column.  With 5 alternatives the bf16 rows take 102 to
// 112 us, with 20 128 to 132 (each lane reading its own group's vectors again: 217
// and 231).
// A chain of loads and barriers a row, and the second reads, are what they cost.
//
// Rows that this arithmetic does not cover (NaN or +inf, a largest logit beyond
// 1e7 or so, nothing but -inf) are noticed by their sums and go through plain
// loops over the row instead, and so do alternatives that there is no room to
// list.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "suika_step.h"
#include "sr_step.h"

namespace {

using namespace sr_step;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kShare = kThreads / kWave;   // lanes of one of the 64 groups that share a maximum
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();
constexpr float kLeast = -1e38f;       // start of a running maximum, in log2 units
constexpr int kMaxTop = SR_LOGPROB_MAX_TOP;
constexpr uint32_t kCandidates = 1024;

struct Stats {
  float m;     // largest logit, as it is
  float M;     // the maximum that s and w go by: max(kLeast, m log2 e)
  float s, w;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  r.M = fmaxf(a.M, b.M);
  const float da = a.M - r.M, db = b.M - r.M;
  const float ea = exp2_fast(da), eb = exp2_fast(db);
  r.s = a.s * ea + b.s * eb;
  // a part without weight has none here either, however far its maximum is off
  r.w = (a.s > 0 || a.s != a.s ? ea * fmaf(fmaxf(da, -1000.0f), a.s, a.w) : 0) +
        (b.s > 0 || b.s != b.s ? eb * fmaf(fmaxf(db, -1000.0f), b.s, b.w) : 0);
  return r;
}

// Takes N logits into a lane's statistics.
template <int N>
__device__ __forceinline__ void take(Stats& t, const float (&x)[N]) {
  float top = x[0];
#pragma unroll
  for (int k = 1; k < N; ++k) top = fmaxf(top, x[k]);
  if (top > t.m) {
    t.m = top;
    const float M = fmaxf(top * kLog2e, kLeast);
    const float down = t.M - M;
    const float f = exp2_fast(down);
    t.w = f * fmaf(fmaxf(down, -1000.0f), t.s, t.w);
    t.s *= f;
    t.M = M;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float d = fmaf(x[k], kLog2e, -t.M);
    const float e = exp2_fast(d);              // NaN stays NaN
    t.s += e;
    t.w = fmaf(fmaxf(d, -160.0f), e, t.w);     // 2^-160 is 0, and so is its part
  }
}

// The wave's statistics, in every lane: the maximum first, then the sums in its
// units.
__device__ __forceinline__ Stats wave_join(Stats t) {
  float m = t.m, M = t.M;
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) {
    m = fmaxf(m, __shfl_xor(m, d));
    M = fmaxf(M, __shfl_xor(M, d));
  }
  const Stats none{m, M, 0, 0};
  t = join(t, none);
  return {m, M, wave_sum(t.s), wave_sum(t.w)};
}

// Whether the sums say what they should: the largest logit's own part is 1.
__device__ __forceinline__ bool sound(const Stats& t) {
  return t.s >= 0.5f && t.s < kInf && t.w > -kInf && t.w < kInf && t.m < kInf;
}

// Order of logits: NaN above +inf, -0 as 0.  Larger keys come first.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A logit and its column, as one number that falls in the order of the
// alternatives: by value, then by column.
__device__ __forceinline__ uint64_t candidate(float x, uint32_t column) {
  return uint64_t(key_of(x)) << 32 | (0xffffffffu - column);
}
__device__ __forceinline__ uint32_t column_of(uint64_t c) { return 0xffffffffu - uint32_t(c); }

struct Shared {
  Stats stats[kWaves];
  float maxima[kWave];
  uint32_t group[kWave], place[kWave];
  uint32_t count;
  uint64_t list[kCandidates];
  uint64_t best[kWaves];
  uint64_t chosen[kMaxTop];
};

__device__ __forceinline__ Stats block_join(Shared& sh, Stats t) {
  t = wave_join(t);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.stats[threadIdx.x / kWave] = t;
  __syncthreads();
  Stats all = sh.stats[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = join(all, sh.stats[w]);
  return all;
}

__device__ __forceinline__ float block_max(Shared& sh, float x) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.maxima[threadIdx.x / kWave] = x;
  __syncthreads();
  float r = sh.maxima[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = fmaxf(r, sh.maxima[w]);
  return r;
}

__device__ __forceinline__ float block_add(Shared& sh, float x) {
  x = wave_sum(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.maxima[threadIdx.x / kWave] = x;
  __syncthreads();
  float r = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) r += sh.maxima[w];
  return r;
}

__device__ __forceinline__ uint64_t block_best(Shared& sh, uint64_t x) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)x, d);
    x = o > x ? o : x;
  }
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.best[threadIdx.x / kWave] = x;
  __syncthreads();
  uint64_t r = sh.best[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = sh.best[w] > r ? sh.best[w] : r;
  return r;
}

// ------------------------------------------------------------------ one row

// N logits from column c on, -inf from column `to` on.
template <typename T, int N>
__device__ __forceinline__ void load_or_fill(const T* row, uint32_t c, uint32_t to, float (&x)[N]) {
  if (c + N <= to) {
    load<T, N>(row + c, x);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = c + k < to ? float(row[c + k]) : -kInf;
  }
}

template <typename T, int N, int B>
__device__ __forceinline__ void load_batch(const T* p, Vec<T, N> (&x)[B]) {
#pragma unroll
  for (int b = 0; b < B; ++b) x[b] = __builtin_nontemporal_load(reinterpret_cast<const Vec<T, N>*>(p + b * kThreads * N));
}

// A lane's statistics of columns from..to.  The next batch is on its way while
// one is taken in.
template <typename T>
__device__ __forceinline__ Stats row_stats(const T* row, uint32_t from, uint32_t to) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kBatch = 4;
  constexpr uint32_t kStep = kBatch * kThreads * N;
  Stats t{-kInf, kLeast, 0, 0};
  uint32_t c = from + threadIdx.x * N;
  auto whole = [&](uint32_t at) { return at + (kBatch - 1) * kThreads * N + N <= to; };
  Vec<T, N> ahead[kBatch];
  if (whole(c)) load_batch<T, N, kBatch>(row + c, ahead);
  while (whole(c)) {
    float x[kBatch * N];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int k = 0; k < N; ++k) x[b * N + k] = float(ahead[b][k]);
    c += kStep;
    if (whole(c)) load_batch<T, N, kBatch>(row + c, ahead);
    take<kBatch * N>(t, x);
  }
  for (; c < to; c += kThreads * N) {
    float x[N];
    load_or_fill<T, N>(row, c, to, x);
    take<N>(t, x);
  }
  return t;
}

struct Summary {
  float lse, entropy;
  float shift;      // logprob = (x - shift) - rest
  float rest;
};

// Statistics of a row that the running sums do not cover.
template <typename T>
__device__ __forceinline__ Summary plain_summary(Shared& sh, const T* row, uint32_t vocab) {
  float m = -kInf, bad = 0;
  for (uint32_t c = threadIdx.x; c < vocab; c += kThreads) {
    const float x = float(row[c]);
    if (!(x < kInf)) bad = 1;      // NaN, +inf
    m = fmaxf(m, x);
  }
  m = block_max(sh, m);
  bad = block_max(sh, bad);
  const float nan = __builtin_nanf("");
  if (bad > 0) return {nan, nan, nan, nan};
  if (m == -kInf) return {-kInf, 0, 0, 0};
  float s = 0, w = 0;
  for (uint32_t c = threadIdx.x; c < vocab; c += kThreads) {
    const float d = fmaxf(float(row[c]) - m, -200.0f);
    const float e = expf(d);
    s += e;
    w = fmaf(d, e, w);
  }
  s = block_add(sh, s);
  w = block_add(sh, w);
  return {m + logf(s), fmaxf(logf(s) - w / s, 0.0f), m, logf(s)};
}

__device__ __forceinline__ Summary summary_of(const Stats& t) {
  const float ls = logf(t.s);
  // the sums go by M, which is m log2 e but for a rounding that 2^M took part in
  const float slip = fmaf(t.m, kLog2e, -t.M) * kLn2;
  const float rest = ls - slip;
  return {t.m + rest, fmaxf(fmaf(-kLn2, t.w / t.s, ls), 0.0f), t.m, rest};
}

// The k best candidates of the lanes, one after the other: a look at the whole
// row for each.
template <typename T>
__device__ __forceinline__ void plain_top(Shared& sh, const T* row, uint32_t from, uint32_t to, int k) {
  uint64_t last = ~uint64_t(0);
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (uint32_t c = from + threadIdx.x; c < to; c += kThreads) {
      const uint64_t x = candidate(float(row[c]), c);
      if ((i == 0 || x < last) && x > best) best = x;
    }
    last = block_best(sh, best);
    if (threadIdx.x == 0) sh.chosen[i] = last;
  }
  __syncthreads();
}

// sh.chosen[0..k) = the k largest of n <= kCandidates different numbers in
// sh.list, in falling order (n >= k).
__device__ __forceinline__ void rank_list(Shared& sh, uint32_t n, int k) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = sh.list[i];
    int before = 0;
    for (uint32_t j = 0; j < n; ++j) before += sh.list[j] > mine;
    if (before < k) sh.chosen[before] = mine;
  }
  __syncthreads();
}

// Adds the logits of the groups in `groups` that reach `bound`, or are above
// it, to the list (its count was set, and the groups' list is free, before a
// barrier).  The groups' vectors are dealt out to all lanes, neighbours
// of a group to neighbouring lanes, and several loads of a lane are on their
// way at once.
template <typename T>
__device__ __forceinline__ void list_reaching(Shared& sh, const T* row, uint32_t from, uint32_t to, uint64_t groups,
                                              float bound, bool above) {
  constexpr uint32_t N = 16 / sizeof(T), kAhead = 4;
  const uint32_t lane = threadIdx.x % kWave;
  if (threadIdx.x < kWave && (groups >> lane & 1)) sh.group[__popcll(groups & ((uint64_t(1) << lane) - 1))] = lane;
  __syncthreads();
  // Quads of lanes take (group, round) pairs, 64 of them at a time.
  const uint32_t rounds = (to - from + kThreads * N - 1) / (kThreads * N);
  const uint32_t all = uint32_t(__popcll(groups)), step = kThreads / kShare;
  const uint32_t g_step = step / rounds, r_step = step % rounds;
  uint32_t g = threadIdx.x / kShare / rounds, r = threadIdx.x / kShare % rounds;
  auto reaches = [&](float x) { return above ? x > bound : x >= bound; };
  auto add = [&](float x, uint32_t c) {
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < kCandidates) sh.list[at] = candidate(x, c);
  };
  while (__ballot(g < all)) {
    Vec<T, N> x[kAhead];
    uint32_t c[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      c[a] = g < all ? from + (sh.group[g] * kShare + threadIdx.x % kShare + r * kThreads) * N : to;
      if (c[a] + N <= to) x[a] = *reinterpret_cast<const Vec<T, N>*>(row + c[a]);
      g += g_step;
      r += r_step;
      if (r >= rounds) {
        r -= rounds;
        ++g;
      }
    }
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      if (c[a] + N <= to) {
        float top = float(x[a][0]);
#pragma unroll
        for (uint32_t k = 1; k < N; ++k) top = fmaxf(top, float(x[a][k]));
        if (!reaches(top)) continue;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
          if (reaches(float(x[a][k]))) add(float(x[a][k]), c[a] + k);
      } else {
        for (uint32_t k = c[a]; k < to; ++k)
          if (reaches(float(row[k]))) add(float(row[k]), k);
      }
    }
  }
}

// Adds the first `need` columns whose logit equals `bound` to the list, in
// their order.
template <typename T>
__device__ __forceinline__ void list_equal(Shared& sh, const T* row, uint32_t from, uint32_t to, float bound, uint32_t need) {
  uint32_t* part = reinterpret_cast<uint32_t*>(sh.maxima);
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t start = sh.count;
  uint32_t found = 0;
  for (uint32_t at = from; at < to && found < need; at += kThreads) {
    const uint32_t c = at + threadIdx.x;
    const float x = c < to ? float(row[c]) : 0.0f;
    const bool equal = c < to && x == bound;
    const uint64_t mask = __ballot(equal);
    __syncthreads();
    if (lane == 0) part[wave] = uint32_t(__popcll(mask));
    __syncthreads();
    uint32_t place = found + uint32_t(__popcll(mask & ((uint64_t(1) << lane) - 1)));
    for (uint32_t w = 0; w < kWaves; ++w) {
      if (w < wave) place += part[w];
      found += part[w];
    }
    if (equal && place < need) sh.list[start + place] = candidate(x, c);
  }
  __syncthreads();
}

// sh.chosen = the k best of columns from..to (at least k columns, k <= 64); `m`
// is the largest logit of this lane's part, `finite` that there is no NaN.
template <typename T>
__device__ __forceinline__ void row_top(Shared& sh, const T* row, uint32_t from, uint32_t to, int k, float m, bool finite) {
  static_assert(kMaxTop <= kWave, "as many groups as alternatives");
  if (!finite) {
    plain_top(sh, row, from, to, k);
    return;
  }
  // Lanes are taken in 64 groups.  The k-th largest of the groups' maxima is
  // the bound: k groups have a logit that reaches it.
#pragma unroll
  for (int d = 1; d < kShare; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  __syncthreads();
  if (threadIdx.x % kShare == 0) sh.maxima[threadIdx.x / kShare] = m;
  if (threadIdx.x < kWave) sh.place[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  // Every wave compares with a quarter of the groups, so that the counts add up
  // to a group's place.
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const float mine = sh.maxima[lane];
  uint32_t before = 0;
#pragma unroll
  for (uint32_t j = 0; j < kWave / kWaves; ++j) {
    const uint32_t other = wave * (kWave / kWaves) + j;
    const float o = sh.maxima[other];
    before += o > mine || (o == mine && other < lane);
  }
  atomicAdd(&sh.place[lane], before);
  __syncthreads();
  const int at = __ffsll((unsigned long long)__ballot(sh.place[lane] == uint32_t(k - 1))) - 1;
  const float bound = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), at));
  list_reaching(sh, row, from, to, __ballot(mine >= bound), bound, false);
  __syncthreads();
  uint32_t n = sh.count;
  if (n > kCandidates) {
    // many logits equal the bound (a mask's -inf, say): those above it, and the first of the equal ones
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    list_reaching(sh, row, from, to, __ballot(mine > bound), bound, true);
    __syncthreads();
    n = sh.count;
    if (n > kCandidates - kMaxTop) {
      plain_top(sh, row, from, to, k);
      return;
    }
    if (n < uint32_t(k)) {
      list_equal(sh, row, from, to, bound, uint32_t(k) - n);
      n = uint32_t(k);
    }
  }
  rank_list(sh, n, k);
}

template <typename I>
__device__ __forceinline__ int64_t target_at(const I* targets, uint64_t row) { return int64_t(targets[row]); }

// A row's target and its logit, read ahead of the row.
struct Target {
  bool scored, inside;
  float x;
};

template <typename T, typename I>
__device__ __forceinline__ Target target_of(const T* row, const I* targets, uint64_t i, uint32_t vocab) {
  const int64_t t = target_at(targets, i);
  const bool inside = t >= 0 && uint64_t(t) < vocab;
  return {t >= 0, inside, inside ? float(row[t]) : 0.0f};
}

struct Outputs {
  float* logprob;
  float* entropy;
  float* lse;
  float* lse_low;       // or null
  float* top_logprob;
  int64_t* top_index;
};

__device__ __forceinline__ float logprob_of(float x, const Summary& r) { return (x - r.shift) - r.rest; }

// What the rounding of lse = shift + rest lost, exactly (the two-sum of Knuth):
// of logits that are large together, lse alone knows the probabilities to
// |lse| 2^-24 of themselves only.
__device__ __forceinline__ float low_of(const Summary& r) {
  const float b = r.lse - r.shift;
  const float low = (r.shift - (r.lse - b)) + (r.rest - b);
  return fabsf(r.lse) < kInf ? low : 0.0f;
}

// Writes a row's results; sh.chosen holds the alternatives.
__device__ __forceinline__ void put(Shared& sh, const Target& t, uint64_t i, int k, const Summary& r,
                                    const Outputs& out) {
  if (threadIdx.x == 0) {
    float lp = 0;
    if (t.scored) lp = t.inside ? logprob_of(t.x, r) : r.lse != r.lse ? r.lse : -kInf;
    out.logprob[i] = lp;
    out.entropy[i] = r.entropy;
    out.lse[i] = r.lse;
    if (out.lse_low) out.lse_low[i] = low_of(r);
  }
  if (int(threadIdx.x) < k) {
    const uint64_t c = sh.chosen[threadIdx.x];
    out.top_logprob[i * k + threadIdx.x] = logprob_of(value_of(uint32_t(c >> 32)), r);
    out.top_index[i * k + threadIdx.x] = column_of(c);
  }
}

template <bool TOP, typename T, typename I>
__global__ __launch_bounds__(kThreads) void row_kernel(const T* logits, const I* targets, uint64_t stride,
                                                       uint32_t vocab, int k, Outputs out) {
  __shared__ Shared sh;
  const uint64_t i = blockIdx.x;
  const T* row = logits + i * stride;
  const Target target = target_of(row, targets, i, vocab);
  const Stats mine = row_stats(row, 0, vocab);
  const Stats all = block_join(sh, mine);
  const Summary r = sound(all) ? summary_of(all) : plain_summary(sh, row, vocab);
  if constexpr (TOP) row_top(sh, row, 0, vocab, k, mine.m, r.lse == r.lse);
  put(sh, target, i, TOP ? k : 0, r, out);
}

// ---------------------------------------------------------------- split rows

// Few rows do not fill the GPU with a workgroup each, so each is cut into parts
// of `length` columns that leave their statistics and their best k candidates
// in the workspace; a second launch joins them.  4 rows of 152064 bf16 logits
// with 20 alternatives: 13.1 us, uncut 72; the two launches are chains of a few
// loads each, 7.3 and 6.6 us.
struct Parts {
  uint32_t parts, length;
  Stats* stats;         // [rows][parts]
  uint64_t* best;       // [rows][parts][k], falling; 0 where a part has fewer
};

template <bool TOP, typename T>
__global__ __launch_bounds__(kThreads) void part_kernel(const T* logits, uint64_t stride, uint32_t vocab, int k,
                                                        Parts out) {
  __shared__ Shared sh;
  const uint32_t part = blockIdx.x;
  const uint64_t i = blockIdx.y;
  const T* row = logits + i * stride;
  const uint32_t from = part * out.length, to = min(from + out.length, vocab);
  const Stats mine = row_stats(row, from, to);
  const Stats all = block_join(sh, mine);
  const uint64_t at = i * out.parts + part;
  if (threadIdx.x == 0) out.stats[at] = all;
  if constexpr (TOP) {
    const int own = min(k, int(to - from));
    row_top(sh, row, from, to, own, mine.m, all.s == all.s);
    if (int(threadIdx.x) < k) out.best[at * k + threadIdx.x] = int(threadIdx.x) < own ? sh.chosen[threadIdx.x] : 0;
  }
}

// sh.chosen = the k best of n candidates, of which `most` is the best of this
// lane's (every kThreads-th).  As in a row: the k-th largest of the lane groups'
// maxima bounds them from below.
__device__ __forceinline__ void parts_top(Shared& sh, const uint64_t* best, uint32_t n, uint64_t most, int k) {
#pragma unroll
  for (int d = 1; d < kShare; d <<= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)most, d);
    most = o > most ? o : most;
  }
  __syncthreads();
  if (threadIdx.x % kShare == 0) sh.list[threadIdx.x / kShare] = most;
  if (threadIdx.x < kWave) sh.place[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint64_t mine = sh.list[lane];
  uint32_t before = 0;
#pragma unroll
  for (uint32_t j = 0; j < kWave / kWaves; ++j) {
    const uint32_t other = wave * (kWave / kWaves) + j;
    const uint64_t o = sh.list[other];
    before += o > mine || (o == mine && other < lane);
  }
  atomicAdd(&sh.place[lane], before);
  __syncthreads();
  const int at = __ffsll((unsigned long long)__ballot(sh.place[lane] == uint32_t(k - 1))) - 1;
  const uint64_t bound = __shfl((unsigned long long)mine, at);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t x = best[i];
    if (x >= bound && x != 0) {
      const uint32_t to = atomicAdd(&sh.count, 1u);
      if (to < kCandidates) sh.list[to] = x;
    }
  }
  __syncthreads();
  const uint32_t listed = sh.count;
  if (listed <= kCandidates) {
    rank_list(sh, listed, k);
    return;
  }
  uint64_t last = ~uint64_t(0);
  for (int i = 0; i < k; ++i) {
    uint64_t top = 0;
    for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
      const uint64_t x = best[j];
      if ((i == 0 || x < last) && x > top) top = x;
    }
    last = block_best(sh, top);
    if (threadIdx.x == 0) sh.chosen[i] = last;
  }
  __syncthreads();
}

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void parts_kernel(const T* logits, const I* targets, uint64_t stride,
                                                         uint32_t vocab, int k, Parts in, Outputs out) {
  __shared__ Shared sh;
  const uint64_t i = blockIdx.x;
  const T* row = logits + i * stride;
  const Target target = target_of(row, targets, i, vocab);
  const Stats mine = threadIdx.x < in.parts ? in.stats[i * in.parts + threadIdx.x] : Stats{-kInf, kLeast, 0, 0};
  const uint32_t n = in.parts * uint32_t(k);
  const uint64_t* best = in.best + i * n;
  uint64_t most = 0;
  for (uint32_t j = threadIdx.x; j < n; j += kThreads) most = best[j] > most ? best[j] : most;
  const Stats all = block_join(sh, mine);
  const Summary r = sound(all) ? summary_of(all) : plain_summary(sh, row, vocab);
  if (k) parts_top(sh, best, n, most, k);
  put(sh, target, i, k, r, out);
}

// ----------------------------------------------------------------- gradient

// One vector a lane, in the order of memory, stores through the L2: 8192 x 32000
// bf16 in 168 us (6.2 TB/s), 2047 x 50304 f32 in 123 (6.7), HBM bound (workgroups
// in the order of rows, four vectors a lane: 176 and 124; stores streamed: 185
// and 148).
// PAIR: with lse_low, one more value of the row behind an address in memory
// (8192 x 32000 bf16 under the profiler 176 us, without 174; decided at run time,
// the single lse takes 176 as well).
template <bool PAIR, typename T, typename I>
__global__ __launch_bounds__(kThreads) void grad_kernel(const T* logits, const I* targets, uint64_t stride,
                                                        uint32_t vocab, uint32_t columns, uint32_t spans,
                                                        const float* lse, const float* entropy,
                                                        const float* g_logprob, const float* g_entropy, T* grad,
                                                        uint64_t grad_stride, const float* lse_low) {
  constexpr int N = 16 / sizeof(T);
  const uint32_t i = blockIdx.x / spans;
  const uint32_t c = ((blockIdx.x - i * spans) * kThreads + threadIdx.x) * N;
  const T* row = logits + i * stride;
  T* to = grad + i * grad_stride;
  const bool whole = c + N <= columns;
  Vec<T, N> x;
  if (whole) x = __builtin_nontemporal_load(reinterpret_cast<const Vec<T, N>*>(row + c));
  const int64_t target = target_at(targets, i);
  const float l = lse[i], low = PAIR ? lse_low[i] : 0.0f, h = entropy[i];
  const float gl = g_logprob && target >= 0 ? g_logprob[i] : 0.0f;
  const float gh = g_entropy ? g_entropy[i] : 0.0f;
  // grad = [target] gl - p (gl + gh (ln p + h)) with ln p = d - low; d = x - l is exact where x is within a factor
  // of two of l
  const float base = PAIR ? fmaf(-gh, low, fmaf(gh, h, gl)) : fmaf(gh, h, gl), low2 = low * kLog2e;
  const bool empty = l == -kInf;
  auto value = [&](float x, uint32_t c) {
    const float d = x - l;
    const float p = exp2_fast(PAIR ? fmaf(d, kLog2e, -low2) : d * kLog2e);             // NaN stays NaN
    float g = -p * fmaf(gh, fmaxf(d, -200.0f), base);
    if (int64_t(c) == target) g += gl;
    return empty || c >= vocab ? 0.0f : g;
  };
  if (whole) {
    float g[N];
#pragma unroll
    for (int k = 0; k < N; ++k) g[k] = value(float(x[k]), c + k);
    store_region<kThrough, T, N>(region(to, uint32_t(columns * sizeof(T))), uint32_t(c * sizeof(T)), g);
  } else {
    for (uint32_t k = c; k < columns; ++k) to[k] = T(value(float(row[k]), k));
  }
}

// ---------------------------------------------------------------------- host

int check_shape(const char* who, const sr_logprob_shape* s) {
  if (s == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (s->target_dtype != SR_DT_I32 && s->target_dtype != SR_DT_I64)
    return fail(SR_EDTYPE, "%s: targets of dtype %d", who, s->target_dtype);
  if (!float_dtype(s->dtype)) return fail(SR_EDTYPE, "%s: logits of dtype %d", who, s->dtype);
  if (s->rows > SR_STEP_MAX_ROWS || s->columns > SR_STEP_MAX_ROWS)
    return fail(SR_EBOUNDS, "%s: %llu rows of %llu columns", who, (unsigned long long)s->rows,
                (unsigned long long)s->columns);
  if (s->vocab < 1 || s->vocab > s->columns)
    return fail(SR_EINVAL, "%s: a vocabulary of %llu in %llu columns", who, (unsigned long long)s->vocab,
                (unsigned long long)s->columns);
  if (s->stride < s->columns || s->stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "%s: rows %llu apart for %llu columns", who, (unsigned long long)s->stride,
                (unsigned long long)s->columns);
  if (s->rows && (s->logits == nullptr || s->targets == nullptr)) return fail(SR_EINVAL, "%s: null argument", who);
  if (reinterpret_cast<uintptr_t>(s->logits) % sr_internal::dtype_size(s->dtype) ||
      reinterpret_cast<uintptr_t>(s->targets) % sr_internal::dtype_size(s->target_dtype))
    return fail(SR_EALIGN, "%s: not aligned to the elements", who);
  return SR_OK;
}

int check_top(const char* who, const sr_logprob_shape& s, int32_t top) {
  if (top < 0 || top > kMaxTop || uint64_t(top) > s.vocab)
    return fail(SR_EINVAL, "%s: the best %d of %llu (at most %d)", who, top, (unsigned long long)s.vocab, kMaxTop);
  return SR_OK;
}

// How rows are cut: into as many parts as give every compute unit eight
// workgroups, of 2048 columns or more.
struct Cut {
  uint32_t parts, length;
  uint64_t best, bytes;
};

Cut parts_of(const sr_logprob_shape& s, int32_t top) {
  constexpr uint64_t kFill = 2048, kLeastColumns = 2048, kMostParts = 128;
  Cut c{1, uint32_t(s.vocab), 0, 0};
  if (s.rows == 0) return c;
  const uint64_t parts = std::min({kFill / s.rows, s.vocab / kLeastColumns, kMostParts});
  if (parts < 2) return c;
  c.length = uint32_t((s.vocab + parts - 1) / parts + 7) / 8 * 8;      // whole vectors
  c.parts = uint32_t((s.vocab + c.length - 1) / c.length);
  c.best = (s.rows * c.parts * sizeof(Stats) + 255) / 256 * 256;
  c.bytes = c.best + s.rows * c.parts * uint64_t(top) * sizeof(uint64_t);
  return c;
}

// f(logits, targets) with their types.
template <typename T, typename F>
void with_targets(const sr_logprob_shape& s, F&& f) {
  if (s.target_dtype == SR_DT_I64) f(static_cast<const T*>(s.logits), static_cast<const int64_t*>(s.targets));
  else f(static_cast<const T*>(s.logits), static_cast<const int32_t*>(s.targets));
}

template <typename F>
void with_types(const sr_logprob_shape& s, F&& f) {
  if (s.dtype == SR_DT_F32) with_targets<float>(s, f);
  else if (s.dtype == SR_DT_BF16) with_targets<bf16>(s, f);
  else with_targets<f16>(s, f);
}

int logprobs(const char* who, const sr_logprob_shape* shape, int32_t top, const Outputs& out, bool pair, void* workspace,
             uint64_t workspace_bytes, hipStream_t stream) {
  if (int rc = check_shape(who, shape)) return rc;
  if (int rc = check_top(who, *shape, top)) return rc;
  const uint64_t need = parts_of(*shape, top).bytes;
  const sr_logprob_shape& s = *shape;
  if (s.rows == 0) return SR_OK;
  if (!out.logprob || !out.entropy || !out.lse || (pair && !out.lse_low) ||
      (top && (!out.top_logprob || !out.top_index)))
    return fail(SR_EINVAL, "%s: an output is null", who);
  for (const float* p : {out.logprob, out.entropy, out.lse, out.lse_low, out.top_logprob})
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(SR_EALIGN, "%s: an output is not aligned", who);
  if (reinterpret_cast<uintptr_t>(out.top_index) % 8) return fail(SR_EALIGN, "%s: an output is not aligned", who);
  if (workspace_bytes < need || (need && workspace == nullptr))
    return fail(SR_EINVAL, "%s: a workspace of %llu bytes, %llu are needed", who, (unsigned long long)workspace_bytes,
                (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(SR_EALIGN, "%s: workspace not aligned", who);
  const Extent written[] = {{out.logprob, s.rows * 4}, {out.entropy, s.rows * 4}, {out.lse, s.rows * 4},
                            {out.lse_low, s.rows * 4}, {out.top_logprob, top ? s.rows * top * 4 : 0},
                            {out.top_index, top ? s.rows * top * 8 : 0}, {workspace, need}};
  const Extent read[] = {{s.logits, ((s.rows - 1) * s.stride + s.columns) * sr_internal::dtype_size(s.dtype)},
                         {s.targets, s.rows * sr_internal::dtype_size(s.target_dtype)}};
  for (const Extent& w : written) {
    for (const Extent& o : written)
      if (&o != &w && w.meets(o)) return fail(SR_EOVERLAP, "%s: two outputs overlap", who);
    for (const Extent& o : read)
      if (w.meets(o)) return fail(SR_EOVERLAP, "%s: an output overlaps an input", who);
  }
  const Cut cut = parts_of(s, top);
  char* base = static_cast<char*>(workspace);
  const Parts parts{cut.parts, cut.length, reinterpret_cast<Stats*>(base), reinterpret_cast<uint64_t*>(base + cut.best)};
  with_types(s, [&](auto* logits, auto* targets) {
    const uint32_t rows = uint32_t(s.rows), vocab = uint32_t(s.vocab);
    if (cut.parts == 1) {
      if (top) row_kernel<true><<<rows, kThreads, 0, stream>>>(logits, targets, s.stride, vocab, int(top), out);
      else row_kernel<false><<<rows, kThreads, 0, stream>>>(logits, targets, s.stride, vocab, 0, out);
      return;
    }
    const dim3 grid(cut.parts, rows);
    if (top) part_kernel<true><<<grid, kThreads, 0, stream>>>(logits, s.stride, vocab, int(top), parts);
    else part_kernel<false><<<grid, kThreads, 0, stream>>>(logits, s.stride, vocab, 0, parts);
    parts_kernel<<<rows, kThreads, 0, stream>>>(logits, targets, s.stride, vocab, int(top), parts, out);
  });
  return launched(who);
}

int logprobs_grad(const char* who, const sr_logprob_shape* shape, const float* lse, const float* lse_low, bool pair,
                  const float* entropy, const float* g_logprob, const float* g_entropy, void* grad,
                  uint64_t grad_stride, hipStream_t stream) {
  if (int rc = check_shape(who, shape)) return rc;
  const sr_logprob_shape& s = *shape;
  if (s.rows == 0) return SR_OK;
  if (!lse || (pair && !lse_low) || !entropy || !grad) return fail(SR_EINVAL, "%s: null argument", who);
  if (grad_stride < s.columns || grad_stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "%s: rows %llu apart for %llu columns", who, (unsigned long long)grad_stride,
                (unsigned long long)s.columns);
  for (const float* p : {lse, lse_low, entropy, g_logprob, g_entropy})
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(SR_EALIGN, "%s: not aligned to the elements", who);
  const uint64_t size = sr_internal::dtype_size(s.dtype);
  if (reinterpret_cast<uintptr_t>(grad) % size) return fail(SR_EALIGN, "%s: not aligned to the elements", who);
  const Extent to{grad, ((s.rows - 1) * grad_stride + s.columns) * size};
  const Extent logits{s.logits, ((s.rows - 1) * s.stride + s.columns) * size};
  const bool in_place = grad == s.logits && grad_stride == s.stride;
  if ((!in_place && to.meets(logits)) ||
      to.meets({s.targets, s.rows * sr_internal::dtype_size(s.target_dtype)}) || to.meets({lse, s.rows * 4}) ||
      to.meets({lse_low, s.rows * 4}) || to.meets({entropy, s.rows * 4}) || to.meets({g_logprob, s.rows * 4}) ||
      to.meets({g_entropy, s.rows * 4}))
    return fail(SR_EOVERLAP, "%s: the gradient overlaps an input", who);
  const uint64_t step = kThreads * 16 / size, spans = (s.columns + step - 1) / step, blocks = s.rows * spans;
  if (blocks >= uint64_t(1) << 24)     // the grid's threads stay below 2^32
    return fail(SR_EBOUNDS, "%s: %llu rows of %llu columns", who, (unsigned long long)s.rows,
                (unsigned long long)s.columns);
  with_types(s, [&](const auto* logits, const auto* targets) {
    typedef typename std::remove_cv<typename std::remove_reference<decltype(*logits)>::type>::type T;
    auto launch = [&](auto* kernel) {
      kernel<<<uint32_t(blocks), kThreads, 0, stream>>>(
          logits, targets, s.stride, uint32_t(s.vocab), uint32_t(s.columns), uint32_t(spans), lse, entropy, g_logprob,
          g_entropy, static_cast<T*>(grad), grad_stride, lse_low);
    };
    typedef typename std::remove_cv<typename std::remove_reference<decltype(*targets)>::type>::type I;
    if (pair) launch(grad_kernel<true, T, I>);
    else launch(grad_kernel<false, T, I>);
  });
  return launched(who);
}

}  // namespace

extern "C" {

int sr_logprob_workspace(const sr_logprob_shape* shape, int32_t top, uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_logprob_workspace: null argument");
  if (int rc = check_shape("sr_logprob_workspace", shape)) return rc;
  if (int rc = check_top("sr_logprob_workspace", *shape, top)) return rc;
  *bytes = parts_of(*shape, top).bytes;
  return SR_OK;
}

int sr_logprob(const sr_logprob_shape* shape, int32_t top, float* logprob, float* entropy, float* lse,
               float* top_logprob, int64_t* top_index, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return logprobs("sr_logprob", shape, top, {logprob, entropy, lse, nullptr, top_logprob, top_index}, false, workspace,
                  workspace_bytes, stream);
}

int sr_logprob_pair(const sr_logprob_shape* shape, int32_t top, float* logprob, float* entropy, float* lse,
                    float* lse_low, float* top_logprob, int64_t* top_index, void* workspace, uint64_t workspace_bytes,
                    hipStream_t stream) {
  return logprobs("sr_logprob_pair", shape, top, {logprob, entropy, lse, lse_low, top_logprob, top_index}, true,
                  workspace, workspace_bytes, stream);
}

int sr_logprob_grad(const sr_logprob_shape* shape, const float* lse, const float* entropy, const float* g_logprob,
                    const float* g_entropy, void* grad, uint64_t grad_stride, hipStream_t stream) {
  return logprobs_grad("sr_logprob_grad", shape, lse, nullptr, false, entropy, g_logprob, g_entropy, grad, grad_stride,
                       stream);
}

int sr_logprob_pair_grad(const sr_logprob_shape* shape, const float* lse, const float* lse_low, const float* entropy,
                         const float* g_logprob, const float* g_entropy, void* grad, uint64_t grad_stride,
                         hipStream_t stream) {
  return logprobs_grad("sr_logprob_pair_grad", shape, lse, lse_low, true, entropy, g_logprob, g_entropy, grad,
                       grad_stride, stream);
}

}  // extern "C"
