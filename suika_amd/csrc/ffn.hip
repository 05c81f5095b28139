// ffn.hip -- the gated feed-forward block of a tensor-parallel share and its
// gradients (C ABI in include/suika_step.h).
//
//   a = x G^T   b = x U^T   h = act(a) b   y = h D^T
//
// Gate G and up U are this rank's rows, down D this rank's columns, so the
// ranks' y add up.  Forward, both projections, the activation and the product
// are one kernel: a tile has the rows of G and of U in turn, so a wave has a
// and b of the same columns.  Backward, the product dy D ends in the gradients
// of a and b; dx is one product over both pairs, and the three matrices'
// gradients are one launch.
//
// h, da and db are rounded to the operands' type, as the next product takes
// them; sums are in 32 bits.  a and b are kept for the gradients as floats: kept
// in bf16 they would be two roundings more on the way to each gradient, whose
// distance from the exact one grew from 1.4 to 2.1 roundings of its own; writing
// and reading them costs 4 bytes more a value, 2% of a training step's time.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "suika_step.h"
#include "sr_step.h"
#include "sr_tile.h"

namespace {

using namespace sr_step;
using sr_tile::Block;
using sr_tile::COL;
using sr_tile::f32x4;
using sr_tile::Grid;
using sr_tile::Operand;
using sr_tile::Product;
using sr_tile::ROW;
using sr_tile::Shared;
using sr_tile::Side;

// -------------------------------------------------------------- activations

struct Act {
  float value, slope;
};

// exp(x) for results of T.  The fast one rounds x log2(e), which leaves x 2^-24 of the
// result's size: 1e-5 where the weight below is 1e-38.  16 bits round that off, floats
// would show it (a gate of -60 3e-6 off).
template <typename T>
__device__ __forceinline__ float exp_for(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  else return __expf(x);
}

// All three are a times a weight between 0 and 1.  exp overflows to infinity
// for far negative a, where the weight is then 0.
template <typename T>
__device__ __forceinline__ float weight_of(float z) { return 1.0f / (1.0f + exp_for<T>(-z)); }

constexpr float kTanhScale = 1.5957691216057308f;     // 2 sqrt(2 / pi)
constexpr float kTanhCube = 0.044715f;

template <typename T, bool SLOPE>
__device__ __forceinline__ Act act(float a, int32_t kind) {
  Act r{0, 0};
  if (kind == SR_ACT_GELU) {
    const float p = 0.5f * erfcf(a * -0.70710678118654752f);
    r.value = a * p;
    if (SLOPE) r.slope = fmaf(a * 0.39894228040143268f, exp_for<T>(-0.5f * a * a), p);
    return r;
  }
  float z = a, dz = 1.0f;
  if (kind == SR_ACT_GELU_TANH) {
    const float q = fminf(a * a, 1e30f);      // finite, so that a weight of 0 makes the slope's term 0
    z = kTanhScale * fmaf(kTanhCube * q, a, a);
    dz = kTanhScale * fmaf(3 * kTanhCube, q, 1.0f);
  }
  const float p = weight_of<T>(z);
  r.value = a * p;
  // the rest of the weight, 1 - p, from the other side: nothing cancels
  if (SLOPE) r.slope = fmaf(r.value * weight_of<T>(-z), dz, p);
  return r;
}

// ------------------------------------------------------------------ products

// Which tiles of a launch have their steps dealt out to several workgroups: those from
// `whole` on, to `splits` of them with `steps` steps each.  A workgroup then leaves the
// sums of its steps as floats, a tile a part, and a launch behind it joins the parts of a
// tile in order.
struct Cut {
  uint32_t whole;
  uint32_t splits, steps;
  uint64_t parts;
};

// A workgroup's tile, and its steps of all.
struct Turn {
  uint32_t tile, from, to;
  uint32_t part;              // where its sums go, if `split`
  bool split;
};

__device__ __forceinline__ Turn turn_of(const Cut& c, uint32_t item) {
  const bool split = item >= c.whole;
  if (!split) return {item, 0, 0xffffffffu, 0, false};
  const uint32_t part = item - c.whole, from = part % c.splits * c.steps;
  return {c.whole + part / c.splits, from, from + c.steps, part, true};
}

// Eight sums of a part: of row r, from column n on.
template <int SIZE>
__device__ __forceinline__ void store_part(const Cut& c, uint32_t part, uint32_t r, uint32_t n, const float (&v)[8]) {
  store_row(global<float>(c.parts) + (uint64_t(part) * SIZE + r) * SIZE + n, v, 8);
}

// The joined sums of the tile that is the `tile`th of the split ones.
template <int SIZE>
__device__ __forceinline__ void join_parts(const Cut& c, uint32_t tile, uint32_t r, uint32_t n, float (&sum)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0;
  const float* p = global<const float>(c.parts) + (uint64_t(tile) * c.splits * SIZE + r) * SIZE + n;
  for (uint32_t s = 0; s < c.splits; ++s) {
    float x[8];
    load_row(p + s * (SIZE * SIZE), x, 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += x[e];
  }
}

constexpr int kPlainThreads = 256;

// Both projections.  Bound by the matrix cores, and by the results' bytes where a and
// b are kept: 8192 tokens, 4096 columns, 5504 rows of both (bf16, 739 GFLOP) 776 to
// 850 us with 0.45 GB written.  Few tiles with long sums are split (kActivatedGain).
struct ForwardArgs {
  Product p;
  Grid grid;
  Cut cut;
  uint64_t h, a, b;           // a and b: kept for the gradients, or 0
  uint64_t h_stride;          // elements
  uint32_t tokens, ffn, padded;     // columns of h: those behind ffn are zeros
  int32_t activation;
};

template <typename T>
__device__ __forceinline__ void store_forward(const ForwardArgs& t, uint32_t r, uint32_t n, const float (&a)[8],
                                              const float (&b)[8]) {
  if (r >= t.tokens || n >= t.padded) return;
  float h[8];
  // (the columns behind ffn are zeros also where a row of x has an infinity)
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = n + e < t.ffn ? act<T, false>(a[e], t.activation).value * b[e] : 0.0f;
  store_row(global<T>(t.h) + r * t.h_stride + n, h, t.padded - n);
  if (t.a && n < t.ffn) {
    store_row(global<float>(t.a) + uint64_t(r) * t.ffn + n, a, t.ffn - n);
    store_row(global<float>(t.b) + uint64_t(r) * t.ffn + n, b, t.ffn - n);
  }
}

template <typename T, int SIZE>
__global__ __launch_bounds__(sr_tile::threads<T>(SIZE), SIZE == 64 ? 3 : 2) void forward_kernel(ForwardArgs t) {
  typedef sr_tile::Tile<T, false, SIZE, ROW, ROW, true> Tile;
  SR_TILE_MEMORY(Tile);
  const uint32_t item = sr_tile::item_of(blockIdx.x, t.grid.items, SIZE);
  if (item >= t.grid.items) return;
  const Turn turn = turn_of(t.cut, item);
  uint32_t row, column;
  sr_tile::banded(turn.tile, t.grid.rows, t.grid.columns, row, column);
  row *= SIZE;
  column *= Tile::kColumns;
  Tile tile;
  sr_tile::run(tile, t.p, row, column, turn.from, min(turn.to, (t.p.k + Tile::kK - 1) / Tile::kK), (Shared)a0, (Shared)a1,
               (Shared)b0, (Shared)b1);
  __syncthreads();
  tile.template results<false, false>(SR_TILE_SLAB(Tile), sr_tile::nothing, [&](uint32_t r, uint32_t n, const float (&a)[8],
                                                                         const float (&b)[8], sr_tile::Nothing) {
    if (turn.split) {
      if (row + r >= t.tokens) return;
      store_part<SIZE>(t.cut, turn.part, r, n, a);
      store_part<SIZE>(t.cut, turn.part, r, Tile::kColumns + n, b);
    } else {
      store_forward<T>(t, row + r, column + n, a, b);
    }
  });
}

// Both projections' sums joined: eight columns a lane.
template <typename T, int SIZE>
__global__ __launch_bounds__(kPlainThreads) void forward_join_kernel(ForwardArgs t) {
  constexpr uint32_t kColumns = SIZE / 2, kBlocks = SIZE * kColumns / 8 / kPlainThreads;      // of a tile
  const uint32_t tile = blockIdx.x / kBlocks, at = (blockIdx.x % kBlocks * kPlainThreads + threadIdx.x) * 8;
  const uint32_t r = at / kColumns, n = at % kColumns;
  uint32_t row, column;
  sr_tile::banded(t.cut.whole + tile, t.grid.rows, t.grid.columns, row, column);
  row = row * SIZE + r;
  column = column * kColumns + n;
  if (row >= t.tokens || column >= t.padded) return;
  float a[8], b[8];
  join_parts<SIZE>(t.cut, tile, r, n, a);
  join_parts<SIZE>(t.cut, tile, r, kColumns + n, b);
  store_forward<T>(t, row, column, a, b);
}

// dh = dy D, and from it da, db and h again: the same h as forward's, which is
// not kept (writing and reading it would be as many bytes).  The shape above: 369 GFLOP
// in 496 to 515 us, 0.63 GB read and written behind the products.
struct BackwardArgs {
  Product p;
  Grid grid;
  Cut cut;
  uint64_t a, b;              // kept
  uint64_t da, db, h;         // 0: not wanted
  uint64_t stride;            // of da, db and h
  uint32_t tokens, ffn, padded;
  int32_t activation;
};

struct Kept {
  float a[8], b[8];
};

__device__ __forceinline__ Kept load_kept(const BackwardArgs& t, uint32_t r, uint32_t n) {
  Kept k{};
  if (r >= t.tokens || n >= t.ffn) return k;
  load_row(global<const float>(t.a) + uint64_t(r) * t.ffn + n, k.a, t.ffn - n);
  load_row(global<const float>(t.b) + uint64_t(r) * t.ffn + n, k.b, t.ffn - n);
  return k;
}

template <typename T>
__device__ __forceinline__ void store_backward(const BackwardArgs& t, uint32_t r, uint32_t n, const float (&dh)[8],
                                               const Kept& k) {
  if (r >= t.tokens || n >= t.padded) return;
  float da[8], db[8], h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const Act f = act<T, true>(k.a[e], t.activation);
    const float d = n + e < t.ffn ? dh[e] : 0.0f;      // (0 also where a row of dy has an infinity)
    h[e] = f.value * k.b[e];
    db[e] = d * f.value;
    da[e] = d * k.b[e] * f.slope;
  }
  const uint64_t at = r * t.stride + n;
  if (t.da) {
    store_row(global<T>(t.da) + at, da, t.padded - n);
    store_row(global<T>(t.db) + at, db, t.padded - n);
  }
  if (t.h) store_row(global<T>(t.h) + at, h, t.padded - n);
}

template <typename T, int SIZE>
__global__ __launch_bounds__(sr_tile::threads<T>(SIZE), SIZE == 64 ? 3 : 2) void backward_kernel(BackwardArgs t) {
  typedef sr_tile::Tile<T, false, SIZE, ROW, COL> Tile;
  SR_TILE_MEMORY(Tile);
  const uint32_t item = sr_tile::item_of(blockIdx.x, t.grid.items, SIZE);
  if (item >= t.grid.items) return;
  const Turn turn = turn_of(t.cut, item);
  uint32_t row, column;
  sr_tile::banded(turn.tile, t.grid.rows, t.grid.columns, row, column);
  row *= SIZE;
  column *= SIZE;
  Tile tile;
  sr_tile::run(tile, t.p, row, column, turn.from, min(turn.to, (t.p.k + Tile::kK - 1) / Tile::kK), (Shared)a0, (Shared)a1,
               (Shared)b0, (Shared)b1);
  __syncthreads();
  if (turn.split) {
    tile.template results<false, true>(SR_TILE_SLAB(Tile), sr_tile::nothing, [&](uint32_t r, uint32_t n, const float (&v)[8],
                                                                            sr_tile::Nothing) {
      if (row + r < t.tokens) store_part<SIZE>(t.cut, turn.part, r, n, v);
    });
    return;
  }
  tile.template results<false, true>(
      SR_TILE_SLAB(Tile), [&](uint32_t r, uint32_t n) { return load_kept(t, row + r, column + n); },
      [&](uint32_t r, uint32_t n, const float (&dh)[8], const Kept& k) { store_backward<T>(t, row + r, column + n, dh, k); });
}

// dh joined: eight columns a lane.
template <typename T, int SIZE>
__global__ __launch_bounds__(kPlainThreads) void backward_join_kernel(BackwardArgs t) {
  constexpr uint32_t kBlocks = SIZE * SIZE / 8 / kPlainThreads;      // of a tile
  const uint32_t tile = blockIdx.x / kBlocks, at = (blockIdx.x % kBlocks * kPlainThreads + threadIdx.x) * 8;
  const uint32_t r = at / SIZE, n = at % SIZE;
  uint32_t row, column;
  sr_tile::banded(t.cut.whole + tile, t.grid.rows, t.grid.columns, row, column);
  row = row * SIZE + r;
  column = column * SIZE + n;
  if (row >= t.tokens || column >= t.padded) return;
  const Kept k = load_kept(t, row, column);
  float dh[8];
  join_parts<SIZE>(t.cut, tile, r, n, dh);
  store_backward<T>(t, row, column, dh, k);
}

// Plain products, up to three in a launch.  The steps of all their tiles, or of those
// behind the last whole round of the compute units, may be split.  The shape
// above: y 369 GFLOP in 334 to 350 us, dx 739 in 642 to 677, the matrices' gradients
// 1108 in 1005 (both operands' rows side by side).  Steps split, and joined: y and
// dx of 1021 tokens, 3584 columns and 4736 rows 60 and 98 us, of one workgroup a tile 74 and
// 119; of 509, 768 and 2050 in floats 29 and 46, 47 and 120.
struct Job {
  Product p;
  uint32_t rows, columns;     // of C
  uint32_t tile_rows, tile_columns, first;     // its first tile
  uint64_t out;               // dense
};

constexpr int kMostJobs = 3;

struct ProductArgs {
  Job job[kMostJobs];
  uint32_t items;
  Cut cut;
};

// The job of a tile, and the tile's place in its C.
template <int SIZE>
__device__ __forceinline__ const Job& job_of(const ProductArgs& t, uint32_t tile, uint32_t& row, uint32_t& column) {
  int j = 0;
#pragma unroll
  for (int i = 1; i < kMostJobs; ++i) j = tile >= t.job[i].first ? i : j;
  const Job& job = t.job[j];
  sr_tile::banded(tile - job.first, job.tile_rows, job.tile_columns, row, column);
  row *= SIZE;
  column *= SIZE;
  return job;
}

template <typename T, int SIZE, Side A, Side B>
__global__ __launch_bounds__(sr_tile::threads<T>(SIZE), SIZE == 64 ? 3 : 2) void product_kernel(ProductArgs t) {
  typedef sr_tile::Tile<T, false, SIZE, A, B> Tile;
  SR_TILE_MEMORY(Tile);
  const uint32_t item = sr_tile::item_of(blockIdx.x, t.items, SIZE);
  if (item >= t.items) return;
  const Turn turn = turn_of(t.cut, item);
  uint32_t row, column;
  const Job& job = job_of<SIZE>(t, turn.tile, row, column);
  const uint32_t steps = (job.p.k + Tile::kK - 1) / Tile::kK * (job.p.a2.data ? 2 : 1);
  Tile tile;
  sr_tile::run(tile, job.p, row, column, turn.from, min(turn.to, steps), (Shared)a0, (Shared)a1, (Shared)b0, (Shared)b1);
  __syncthreads();
  tile.template results<false, false>(SR_TILE_SLAB(Tile), sr_tile::nothing, [&](uint32_t r, uint32_t n, const float (&v)[8],
                                                                         sr_tile::Nothing) {
    const uint32_t i = row + r, j = column + n;
    if (i >= job.rows || j >= job.columns) return;
    if (turn.split) store_part<SIZE>(t.cut, turn.part, r, n, v);
    else store_row(global<T>(job.out) + uint64_t(i) * job.columns + j, v, job.columns - j);
  });
}

// The products' sums joined: eight values a lane.
template <typename T, int SIZE>
__global__ __launch_bounds__(kPlainThreads) void join_kernel(ProductArgs t) {
  constexpr uint32_t kBlocks = SIZE * SIZE / 8 / kPlainThreads;      // of a tile
  const uint32_t tile = blockIdx.x / kBlocks, at = (blockIdx.x % kBlocks * kPlainThreads + threadIdx.x) * 8;
  uint32_t row, column;
  const Job& job = job_of<SIZE>(t, t.cut.whole + tile, row, column);
  const uint32_t r = at / SIZE, n = at % SIZE;
  row += r;
  column += n;
  if (row >= job.rows || column >= job.columns) return;
  float sum[8];
  join_parts<SIZE>(t.cut, tile, r, n, sum);
  store_row(global<T>(job.out) + uint64_t(row) * job.columns + column, sum, job.columns - column);
}

// A copy of rows that tiles can be loaded from: each starts at a multiple of 16
// bytes and ends in zeros.
template <typename T>
__global__ __launch_bounds__(kPlainThreads) void align_kernel(const T* from, uint64_t stride, uint32_t columns, T* to,
                                                              uint32_t padded) {
  const uint32_t n = (blockIdx.y * kPlainThreads + threadIdx.x) * 8;
  if (n >= padded) return;
  float v[8];
  load_row(from + blockIdx.x * stride + n, v, n < columns ? columns - n : 0);
  store_row(to + uint64_t(blockIdx.x) * padded + n, v, padded - n);
}

// ---------------------------------------------------------------- few tokens

// Up to 64 tokens: the matrices' bytes bound it, so their rows go from memory
// straight to the matrix cores.  A workgroup has some rows (of G and of U) for all
// tokens; its waves share out the k, and their sums are joined in shared memory.
// The tokens come from the L2 for every workgroup, and a wave's loads and products take
// turns, which is what keeps more than a few tokens from the matrices' 6 TB/s: workgroups
// have as many rows as leave no compute unit without work.
//
// Measured (bf16, us of both launches): 1 token, 3584 columns and 4736 rows 14.8 + 7.8
// (15.3 at a copy's rate), 24 tokens, 4096 and 5504 22.1 + 16.2 (20.4), 64 tokens, 3584
// and 4736 26.8 + 24 (15.4).
template <typename T> struct Thin;
template <> struct Thin<bf16> {
  typedef __bf16 Frag __attribute__((ext_vector_type(8)));
  __device__ static void add(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Thin<f16> {
  typedef _Float16 Frag __attribute__((ext_vector_type(8)));
  __device__ static void add(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Thin<float> {
  typedef f32x4 Frag;
  __device__ static void add(const Frag& a, const Frag& b, f32x4& c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  }
};

struct ThinArgs {
  uint64_t x, m, m2, out;     // m2: up, or 0
  uint64_t x_stride, m_stride, m2_stride;     // elements
  uint32_t tokens, rows, k, out_stride;
  uint32_t each;              // rows of a workgroup, of each matrix
  int32_t activation;
};

// With both projections kept for the gradients.
struct ThinKept : ThinArgs {
  uint64_t a, b;
};

// GROUPS: of 16 tokens; BLOCKS: of 16 rows, GATED: half of them of G, then the same of
// U; WAVES: of a workgroup; Args: ThinKept where the projections are kept (a kernel of its
// own: 16 more bytes of arguments take a launch 0.25 us, 6% of the smallest calls).
template <typename T, int GROUPS, int BLOCKS, int WAVES, bool GATED, typename Args>
__global__ __launch_bounds__(WAVES * kWave) void thin_kernel(Args t) {
  typedef Thin<T> K;
  typedef typename K::Frag Frag;
  constexpr int kEach = 16 / sizeof(T);       // k of a lane
  constexpr int kSpan = 4 * kEach;            // of a wave's 16 x 16 block
  constexpr int kAhead = 4;                   // of them on their way at once
  constexpr uint32_t kRows = 16 * BLOCKS / (GATED ? 2 : 1);      // of each matrix
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  // (a lane without a row of its own loads its neighbour's)
  const uint32_t first_row = blockIdx.x * t.each, end = min(first_row + t.each, t.rows);
  const uint32_t mine = lane / 16 * kEach;
  const T* m[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) {
    const uint32_t place = i * 16 + lane % 16, row = min(first_row + place % kRows, end - 1);
    m[i] = place < kRows ? global<const T>(t.m) + row * t.m_stride : global<const T>(t.m2) + row * t.m2_stride;
  }
  const T* x[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
    x[g] = global<const T>(t.x) + min(uint32_t(16 * g) + lane % 16, t.tokens - 1) * t.x_stride;
  f32x4 c[BLOCKS][GROUPS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) c[i][g] = f32x4(0.0f);
  auto read = [&](const T* p) { return *reinterpret_cast<const Vec<T, kEach>*>(p); };
  const uint32_t blocks = t.k / (kSpan * kAhead);
  for (uint32_t b = wave; b < blocks; b += WAVES) {
    const uint32_t k = b * (kSpan * kAhead) + mine;
    Frag w[BLOCKS][kAhead], v[GROUPS][kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) w[i][a] = read(m[i] + k + a * kSpan);
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) v[g][a] = read(x[g] + k + a * kSpan);
    // all loads on their way: left to itself the compiler has three to six of them
    // there at a time (24 tokens, 5504 rows of 4096 columns 31 us instead of 22)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) K::add(w[i][a], v[g][a], c[i][g]);
  }
  // what is left of k, a block at a time
  const uint32_t rest = blocks * kSpan * kAhead;
  for (uint32_t k0 = rest + wave * kSpan; k0 < t.k; k0 += WAVES * kSpan) {
    const uint32_t k = k0 + mine;
    auto tail = [&](const T* p) {
      if (k + kEach <= t.k) return Frag(read(p + k));
      Frag f;
#pragma unroll
      for (int e = 0; e < kEach; ++e) f[e] = k + e < t.k ? p[k + e] : T(0);
      return f;
    };
    Frag w[BLOCKS];
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) w[i] = tail(m[i]);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const Frag v = tail(x[g]);
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) K::add(w[i], v, c[i][g]);
    }
  }
  // four rows of a token a lane; the waves' sums in order
  __shared__ f32x4 part[WAVES][BLOCKS][GROUPS][kWave];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) part[wave][i][g][lane] = c[i][g];
  __syncthreads();
  for (uint32_t p = wave; p < (kRows + 15) / 16 * GROUPS; p += WAVES) {
    const uint32_t i = p / GROUPS, g = p % GROUPS, place = i * 16 + lane / 16 * 4, other = place + kRows;
    if (place >= kRows) continue;
    const uint32_t i2 = other / 16, lane2 = other % 16 / 4 * 16 + lane % 16;      // U's sums
    const uint32_t token = g * 16 + lane % 16, first = first_row + place;
    f32x4 sum = part[0][i][g][lane], up{};
    if (GATED) up = part[0][i2][g][lane2];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      sum += part[w][i][g][lane];
      if (GATED) up += part[w][i2][g][lane2];
    }
    if (token >= t.tokens) continue;
    T* out = global<T>(t.out) + uint64_t(token) * t.out_stride;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (first + r >= end) continue;
      out[first + r] = static_cast<T>(GATED ? act<T, false>(sum[r], t.activation).value * up[r] : sum[r]);
      if constexpr (std::is_same_v<Args, ThinKept>) {
        const uint64_t at = uint64_t(token) * t.rows + first + r;
        global<float>(t.a)[at] = sum[r];
        global<float>(t.b)[at] = up[r];
      }
    }
  }
}

// ---------------------------------------------------------------------- host

// Calls of so few tokens take the thin kernels: 64, or 32 where the projections are
// kept, and then where tiles would have to copy rows first, or ffn is no more than four
// times hidden: y's few rows of long sums are split only in tiles.  Trained: 5 tokens, 4986
// columns and 1886 rows in floats, which tiles copy, 176 us instead of 254; 24 tokens, 4096
// and 5504 in bf16 117 instead of 123, but 48 tokens 139 instead of 127; 32 tokens, 700 and
// 11008 in floats would be 181 instead of 166.
constexpr uint64_t kFewTokens = 64, kFewKept = 32, kNarrow = 4;
constexpr uint64_t kMostSide = uint64_t(1) << 20;     // hidden, ffn: an aligned row is within kMostStride

uint64_t padded(uint64_t n) { return (n + 7) / 8 * 8; }
uint64_t ceil_div(uint64_t n, uint64_t d) { return (n + d - 1) / d; }

// Parts of a workspace, each at a multiple of 256 bytes.
struct Space {
  char* base;
  uint64_t used = 0;

  uint64_t take(uint64_t bytes) {
    const uint64_t at = used;
    used += (bytes + 255) / 256 * 256;
    return reinterpret_cast<uint64_t>(base) + at;
  }
};

// A user's matrix: rows of `columns` dense elements.
struct Matrix {
  const void* data;
  uint64_t rows, columns, stride;
};

// Whether tiles can be loaded from it as it is.
bool loadable(const Matrix& m, int size) {
  return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && m.stride * size % 16 == 0 && m.columns * size % 16 == 0 &&
         m.stride * size <= sr_tile::kMostStride;
}

// (a row a block: at most SR_STEP_MAX_ROWS of them, and kMostSide / 2048 for its columns)
template <typename T>
void launch_align(const Matrix& m, uint64_t to, hipStream_t stream) {
  const uint32_t wide = uint32_t(padded(m.columns));
  const dim3 grid(uint32_t(m.rows), uint32_t(ceil_div(wide, 8 * kPlainThreads)));
  align_kernel<T><<<grid, kPlainThreads, 0, stream>>>(static_cast<const T*>(m.data), m.stride, uint32_t(m.columns),
                                                      reinterpret_cast<T*>(to), wide);
}

// A matrix as an operand with its rows (ROW) or columns (COL) as C's; copied
// to the workspace first where tiles cannot be loaded from it.  `launch` false:
// only the workspace is counted.
template <typename T>
struct Loader {
  Space& space;
  bool launch;
  hipStream_t stream;

  // The address and the distance of rows in bytes.
  Matrix ready(const Matrix& m) {
    if (loadable(m, sizeof(T)) || m.rows == 0 || m.columns == 0) return m;
    const uint64_t wide = padded(m.columns), to = space.take(m.rows * wide * sizeof(T));
    if (launch) launch_align<T>(m, to, stream);
    return {reinterpret_cast<const void*>(to), m.rows, m.columns, wide};
  }
};

template <typename T>
Operand operand(const Matrix& m, Side side) {
  return {reinterpret_cast<uint64_t>(m.data), m.stride * sizeof(T),
          uint32_t(side == ROW ? m.rows : m.columns)};
}

// Steps of a product over k values.
template <typename T> uint64_t steps_of(uint64_t k) { return ceil_div(k, 128 / sizeof(T)); }

// How products go: their tiles' size, how many of them are not split, and the
// workgroups that the steps of each other one are dealt out to.
struct Way {
  int size;
  uint64_t whole, splits;
  double time;
};

constexpr uint64_t kMostSplits = 24;

// The fastest way for `count` products of rows x columns over `steps` steps each;
// with kMostSplits splits at most, of four steps or more, whose parts are written, read
// and added up by another launch.  Of 256 x 256 tiles, of which a compute unit has one
// at a time, also those alone that would keep few units busy for a round (8192 tokens,
// 4096 columns and 5504 rows, the matrices' gradients have 4 x 256 + 32 tiles: a training
// step takes 3000 us instead of 3110).
//
// Splitting has to take `gain` of the time or less by the model.  Products 0.95 (1021
// tokens, 3584 columns, 4736 rows: the matrices' gradients 0.97 by it and 25 us of 430
// slower, y 0.94 and 60 us instead of 75).  The projections and dh, whose join has the
// activation's reads and writes to itself, 0.75: trained in bf16, dh of that shape is 0.77
// by it and 7 us of 446 slower; 512 tokens of 4096 and 5504, projections 0.88 and 6 us of
// 98 slower; 64 tokens of these 0.74 and 0.53, together 133 us instead of 172; 82 tokens of
// 4976 columns and 168 rows in floats 0.12, the forward pass 35 us instead of 113.
constexpr double kProductGain = 0.95, kActivatedGain = 0.75;

template <typename T>
Way way_of(const uint64_t (*sides)[2], int count, uint64_t steps, double gain) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr double kUnit = 0.4e-6, kLaunch = 10, kRate = 8e12;
  Way best{128, 0, 1, 1e30}, split = best;
  for (int size : {256, 128, 64}) {
    if (kF32 && size == 256) continue;
    uint64_t tiles = 0;
    for (int i = 0; i < count; ++i) tiles += ceil_div(sides[i][0], size) * ceil_div(sides[i][1], size);
    auto time = [&](uint64_t n, uint64_t each) {
      sr_tile::Cost cost(size, kF32);
      cost.add(n, each);
      return cost.time();
    };
    auto consider = [&](uint64_t whole, uint64_t splits) {
      const double join = splits == 1 ? 0 : kLaunch + double(tiles - whole) * size * size * 8 * splits / (kRate * kUnit);
      const double all = time(whole, steps) + time((tiles - whole) * splits, ceil_div(steps, splits)) + join;
      Way& least = splits == 1 ? best : split;
      if (all < least.time) least = {size, whole, splits, all};
    };
    consider(tiles, 1);
    for (uint64_t splits = 2; splits <= std::min(kMostSplits, steps / 4); ++splits) {
      consider(0, splits);
      if (size == 256 && tiles > 256 && tiles % 256) consider(tiles / 256 * 256, splits);
    }
  }
  return split.time < gain * best.time ? split : best;
}

// The cut of a launch's tiles, with the parts' memory, and its items.
int cut_of(const char* who, const Way& way, uint64_t tiles, uint64_t steps, Space& space, Cut& cut, uint32_t& items) {
  cut.whole = uint32_t(way.splits == 1 ? tiles : way.whole);
  cut.steps = uint32_t(ceil_div(steps, way.splits));
  cut.splits = uint32_t(way.splits == 1 ? 1 : ceil_div(steps, cut.steps));
  const uint64_t parted = tiles - cut.whole, all = cut.whole + parted * cut.splits;
  if (all > sr_tile::kMostItems) return fail(SR_EBOUNDS, "%s: %llu parts", who, (unsigned long long)all);
  cut.parts = parted ? space.take(parted * cut.splits * way.size * way.size * sizeof(float)) : 0;
  items = uint32_t(all);
  return SR_OK;
}

// The tiles of a projections' launch (tokens x ffn, `wide` of them a tile), their cut and items.
int grid_of(const char* who, const Way& way, const sr_ffn_shape& s, uint64_t wide, uint64_t steps, Space& space, Grid& grid,
            Cut& cut) {
  const uint64_t rows = ceil_div(s.tokens, way.size), columns = ceil_div(padded(s.ffn), wide);
  if (rows * columns > sr_tile::kMostItems)
    return fail(SR_EBOUNDS, "%s: %llu tokens of %llu columns", who, (unsigned long long)s.tokens, (unsigned long long)s.ffn);
  grid.rows = uint32_t(rows);
  grid.columns = uint32_t(columns);
  return cut_of(who, way, rows * columns, steps, space, cut, grid.items);
}

// Workgroups of a launch that joins parts, of `values` values a tile.
uint32_t join_blocks(const Grid& grid, const Cut& cut, int values) {
  return uint32_t((uint64_t(grid.rows) * grid.columns - cut.whole) * (values / 8 / kPlainThreads));
}

// f(size) with the size as a constant.
template <typename T, typename F>
void with_size(int size, F&& f) {
  if (size == 64) f(std::integral_constant<int, 64>());
  else if (sizeof(T) == 4 || size == 128) f(std::integral_constant<int, 128>());
  else if constexpr (sizeof(T) == 2) f(std::integral_constant<int, 256>());
}

struct Wanted {
  Product p;
  uint64_t rows, columns;
  void* out;
};

// Products with the same sides of operands and as many steps.
template <typename T, Side A, Side B>
int products(const char* who, const Wanted* w, int count, Space& space, bool launch, hipStream_t stream) {
  uint64_t sides[kMostJobs][2] = {};
  uint64_t steps = 0;
  for (int i = 0; i < count; ++i) {
    sides[i][0] = w[i].rows;
    sides[i][1] = w[i].columns;
    steps = steps_of<T>(w[i].p.k) * (w[i].p.a2.data ? 2 : 1);      // alike
  }
  const Way way = way_of<T>(sides, count, steps, kProductGain);
  const int size = way.size;
  ProductArgs t{};
  uint64_t tiles = 0;
  int n = 0;
  for (int i = 0; i < count; ++i) {
    if (w[i].rows == 0 || w[i].columns == 0) continue;
    Job& j = t.job[n++];
    j.p = w[i].p;
    j.rows = uint32_t(w[i].rows);
    j.columns = uint32_t(w[i].columns);
    j.tile_rows = uint32_t(ceil_div(w[i].rows, size));
    j.tile_columns = uint32_t(ceil_div(w[i].columns, size));
    j.first = uint32_t(tiles);
    j.out = reinterpret_cast<uint64_t>(w[i].out);
    tiles += uint64_t(j.tile_rows) * j.tile_columns;
    if (tiles > sr_tile::kMostItems) return fail(SR_EBOUNDS, "%s: a product of %llu x %llu", who,
                                                 (unsigned long long)w[i].rows, (unsigned long long)w[i].columns);
  }
  if (n == 0) return SR_OK;
  for (int i = n; i < kMostJobs; ++i) t.job[i].first = 0xffffffffu;
  if (int rc = cut_of(who, way, tiles, steps, space, t.cut, t.items)) return rc;
  const uint64_t parted = tiles - t.cut.whole;
  if (!launch) return SR_OK;
  with_size<T>(size, [&](auto z) {
    product_kernel<T, z(), A, B><<<sr_tile::blocks_of(t.items, z()), sr_tile::threads<T>(z()), 0, stream>>>(t);
    if (parted) join_kernel<T, z()><<<uint32_t(parted * (z() * z() / 8 / kPlainThreads)), kPlainThreads, 0, stream>>>(t);
  });
  return launched(who);
}

// Rows of a workgroup (of each matrix) so that the compute unit with the most of them
// has few: of the launch's rounds over 256 units, each its rows, and half of a token's
// row for every token.  Measured for G and U of 4096 columns, at 1, 2 and 3 rounds:
// 24 tokens, 5504 rows 22.1, 27.6 and 31.8 us with 22, 11 and 8 rows; 4096 rows 17.6 and
// 22.5 with 16 and 8; 64 tokens, 4736 rows of 3584 columns 26.8, 39.8 and 50.7 with 19,
// 10 and 8.  Up to 16 tokens two workgroups on a unit hide each other's start: 18.4 us
// with 11 rows and 20.8 with 22 (one token, 5504 rows).
uint32_t rows_each(uint32_t rows, bool gated, int groups) {
  const uint32_t most = !gated ? 32 : groups == 1 ? 12 : 24;
  uint32_t best = most;
  uint64_t least = ~uint64_t(0);
  for (uint32_t r = most; r >= 5; --r) {
    const uint64_t time = ceil_div(ceil_div(rows, r), 256) * ((gated ? 2 : 1) * r + 8 * groups);
    if (time < least) best = r, least = time;
  }
  return best;
}

template <typename T, int GROUPS, int BLOCKS, bool GATED, typename Args>
void launch_blocks(const Args& t, hipStream_t stream) {
  // (24 tokens, 5504 rows of both 22.1 us with 4 waves, 23.5 with 8; 48 tokens 33.9 and 31.8)
  constexpr int kWaves = GROUPS == 2 ? 4 : 8;
  thin_kernel<T, GROUPS, BLOCKS, kWaves, GATED, Args><<<uint32_t(ceil_div(t.rows, t.each)), kWaves * kWave, 0, stream>>>(t);
}

template <typename T, int GROUPS, bool GATED, typename Args>
void launch_thin(Args t, hipStream_t stream) {
  t.each = rows_each(t.rows, GATED, GROUPS);
  const uint32_t blocks = ceil_div(t.each, GATED ? 8 : 16);
  if (blocks == 1) launch_blocks<T, GROUPS, 1, GATED>(t, stream);
  else if (blocks == 2) launch_blocks<T, GROUPS, 2, GATED>(t, stream);
  else if constexpr (GATED && GROUPS > 1) launch_blocks<T, GROUPS, 3, GATED>(t, stream);
}

template <typename T, bool GATED, typename Args>
void thin(const Args& t, hipStream_t stream) {
  constexpr bool kKeep = std::is_same_v<Args, ThinKept>;
  if (t.rows == 0) return;
  if (t.tokens <= 16) launch_thin<T, 1, GATED>(t, stream);
  else if (kKeep || t.tokens <= 32) launch_thin<T, 2, GATED>(t, stream);
  else if constexpr (!kKeep) launch_thin<T, 4, GATED>(t, stream);
}

Matrix matrix_x(const sr_ffn_shape& s) { return {s.x, s.tokens, s.hidden, s.x_stride}; }
Matrix matrix_gate(const sr_ffn_shape& s) { return {s.gate, s.ffn, s.hidden, s.gate_stride}; }
Matrix matrix_up(const sr_ffn_shape& s) { return {s.up, s.ffn, s.hidden, s.up_stride}; }
Matrix matrix_down(const sr_ffn_shape& s) { return {s.down, s.hidden, s.ffn, s.down_stride}; }

// The block, or (launch false) only its workspace.
template <typename T>
int forward(const sr_ffn_shape& s, void* out, void* a, void* b, Space& space, bool launch, hipStream_t stream) {
  if (s.tokens == 0) return SR_OK;
  const uint64_t wide = padded(s.ffn);
  const uint64_t h = space.take(s.tokens * wide * sizeof(T));
  const Matrix given[4] = {matrix_x(s), matrix_gate(s), matrix_up(s), matrix_down(s)};
  auto copies = [&] { return !std::all_of(given, given + 4, [](const Matrix& m) { return loadable(m, sizeof(T)); }); };
  if (s.tokens <= kFewTokens && (!a || (s.tokens <= kFewKept && (s.ffn <= kNarrow * s.hidden || copies())))) {
    if (!launch) return SR_OK;
    ThinArgs g{reinterpret_cast<uint64_t>(s.x), reinterpret_cast<uint64_t>(s.gate), reinterpret_cast<uint64_t>(s.up), h,
               s.x_stride, s.gate_stride, s.up_stride, uint32_t(s.tokens), uint32_t(s.ffn), uint32_t(s.hidden),
               uint32_t(wide), 0, s.activation};
    if (a) thin<T, true>(ThinKept{g, reinterpret_cast<uint64_t>(a), reinterpret_cast<uint64_t>(b)}, stream);
    else thin<T, true>(g, stream);
    ThinArgs d{h, reinterpret_cast<uint64_t>(s.down), 0, reinterpret_cast<uint64_t>(out), wide, s.down_stride, 0,
               uint32_t(s.tokens), uint32_t(s.hidden), uint32_t(s.ffn), uint32_t(s.hidden), 0, 0};
    thin<T, false>(d, stream);
    return launched("sr_ffn");
  }
  Loader<T> loader{space, launch, stream};
  const Matrix x = loader.ready(given[0]), gate = loader.ready(given[1]), up = loader.ready(given[2]),
               down = loader.ready(given[3]);
  if (s.ffn) {
    ForwardArgs t{};
    t.p = {operand<T>(x, ROW), operand<T>(gate, ROW), {}, operand<T>(up, ROW), uint32_t(s.hidden)};
    const uint64_t sides[1][2] = {{s.tokens, 2 * s.ffn}}, steps = steps_of<T>(s.hidden);
    const Way way = way_of<T>(sides, 1, steps, kActivatedGain);
    if (int rc = grid_of("sr_ffn", way, s, way.size / 2, steps, space, t.grid, t.cut)) return rc;
    t.h = h;
    t.a = reinterpret_cast<uint64_t>(a);
    t.b = reinterpret_cast<uint64_t>(b);
    t.h_stride = wide;
    t.tokens = uint32_t(s.tokens);
    t.ffn = uint32_t(s.ffn);
    t.padded = uint32_t(wide);
    t.activation = s.activation;
    if (launch) {
      const uint32_t blocks = sr_tile::blocks_of(t.grid.items, way.size);
      with_size<T>(way.size, [&](auto z) {
        forward_kernel<T, z()><<<blocks, sr_tile::threads<T>(z()), 0, stream>>>(t);
        const uint32_t joins = join_blocks(t.grid, t.cut, z() * z() / 2);
        if (joins) forward_join_kernel<T, z()><<<joins, kPlainThreads, 0, stream>>>(t);
      });
      if (int rc = launched("sr_ffn")) return rc;
    }
  }
  const Matrix hm{reinterpret_cast<const void*>(h), s.tokens, s.ffn, wide};
  const Wanted w{{operand<T>(hm, ROW), operand<T>(down, ROW), {}, {}, uint32_t(s.ffn)}, s.tokens, s.hidden, out};
  return products<T, ROW, ROW>("sr_ffn", &w, 1, space, launch, stream);
}

template <typename T>
int backward(const sr_ffn_shape& s, const void* a, const void* b, const void* dy, uint64_t dy_stride,
             const sr_ffn_grads& g, Space& space, bool launch, hipStream_t stream) {
  const char* who = "sr_ffn_grad";
  const uint64_t wide = padded(s.ffn), bytes = s.tokens * wide * sizeof(T);
  Loader<T> loader{space, launch, stream};
  const Matrix dym = loader.ready({dy, s.tokens, s.hidden, dy_stride});
  const bool inner = g.x || g.gate || g.up;
  const uint64_t da = inner ? space.take(bytes) : 0, db = inner ? space.take(bytes) : 0, h = g.down ? space.take(bytes) : 0;
  if (s.tokens && s.ffn && (inner || g.down)) {
    const Matrix down = loader.ready(matrix_down(s));
    BackwardArgs t{};
    t.p = {operand<T>(dym, ROW), operand<T>(down, COL), {}, {}, uint32_t(s.hidden)};
    const uint64_t sides[1][2] = {{s.tokens, s.ffn}}, steps = steps_of<T>(s.hidden);
    const Way way = way_of<T>(sides, 1, steps, kActivatedGain);
    if (int rc = grid_of(who, way, s, way.size, steps, space, t.grid, t.cut)) return rc;
    t.a = reinterpret_cast<uint64_t>(a);
    t.b = reinterpret_cast<uint64_t>(b);
    t.da = da;
    t.db = db;
    t.h = h;
    t.stride = wide;
    t.tokens = uint32_t(s.tokens);
    t.ffn = uint32_t(s.ffn);
    t.padded = uint32_t(wide);
    t.activation = s.activation;
    if (launch) {
      const uint32_t blocks = sr_tile::blocks_of(t.grid.items, way.size);
      with_size<T>(way.size, [&](auto z) {
        backward_kernel<T, z()><<<blocks, sr_tile::threads<T>(z()), 0, stream>>>(t);
        const uint32_t joins = join_blocks(t.grid, t.cut, z() * z());
        if (joins) backward_join_kernel<T, z()><<<joins, kPlainThreads, 0, stream>>>(t);
      });
      if (int rc = launched(who)) return rc;
    }
  }
  auto rows_of = [&](uint64_t p) { return Matrix{reinterpret_cast<const void*>(p), s.tokens, s.ffn, wide}; };
  if (g.x) {
    // dx = da G + db U, one sum over both
    const Matrix gate = loader.ready(matrix_gate(s)), up = loader.ready(matrix_up(s));
    const Wanted w{{operand<T>(rows_of(da), ROW), operand<T>(gate, COL), operand<T>(rows_of(db), ROW), operand<T>(up, COL),
                    uint32_t(s.ffn)},
                   s.tokens, s.hidden, g.x};
    if (int rc = products<T, ROW, COL>(who, &w, 1, space, launch, stream)) return rc;
  }
  Wanted w[kMostJobs];
  int n = 0;
  if (g.gate || g.up) {
    const Operand x = operand<T>(loader.ready(matrix_x(s)), COL);
    if (g.gate) w[n++] = {{operand<T>(rows_of(da), COL), x, {}, {}, uint32_t(s.tokens)}, s.ffn, s.hidden, g.gate};
    if (g.up) w[n++] = {{operand<T>(rows_of(db), COL), x, {}, {}, uint32_t(s.tokens)}, s.ffn, s.hidden, g.up};
  }
  if (g.down)
    w[n++] = {{operand<T>(dym, COL), operand<T>(rows_of(h), COL), {}, {}, uint32_t(s.tokens)}, s.hidden, s.ffn, g.down};
  return products<T, COL, COL>(who, w, n, space, launch, stream);
}


uint64_t extent(const Matrix& m, int size) {
  return m.rows && m.columns ? ((m.rows - 1) * m.stride + m.columns) * size : 0;
}

int check_matrix(const char* who, const char* what, const Matrix& m, int size) {
  if (m.stride < m.columns || m.stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "%s: rows of %s %llu elements apart, %llu columns", who, what, (unsigned long long)m.stride,
                (unsigned long long)m.columns);
  if (m.rows && m.columns && m.data == nullptr) return fail(SR_EINVAL, "%s: %s is null", who, what);
  if (reinterpret_cast<uintptr_t>(m.data) % size) return fail(SR_EALIGN, "%s: %s is not aligned to its elements", who, what);
  return SR_OK;
}

int check_shape(const char* who, const sr_ffn_shape* s) {
  if (s == nullptr) return fail(SR_EINVAL, "%s: no shape", who);
  if (!float_dtype(s->dtype)) return fail(SR_EDTYPE, "%s: dtype %d", who, s->dtype);
  if (s->activation != SR_ACT_SILU && s->activation != SR_ACT_GELU && s->activation != SR_ACT_GELU_TANH)
    return fail(SR_EINVAL, "%s: activation %d", who, s->activation);
  if (s->tokens > SR_STEP_MAX_ROWS || s->hidden > kMostSide || s->ffn > kMostSide)
    return fail(SR_EBOUNDS, "%s: %llu tokens, hidden %llu, ffn %llu", who, (unsigned long long)s->tokens,
                (unsigned long long)s->hidden, (unsigned long long)s->ffn);
  const int size = sr_internal::dtype_size(s->dtype);
  if (int rc = check_matrix(who, "x", matrix_x(*s), size)) return rc;
  if (int rc = check_matrix(who, "gate", matrix_gate(*s), size)) return rc;
  if (int rc = check_matrix(who, "up", matrix_up(*s), size)) return rc;
  return check_matrix(who, "down", matrix_down(*s), size);
}

// The memory of a call: what it writes overlaps nothing else.
struct Memory {
  std::vector<Extent> read, written;

  bool clash() const {
    for (size_t i = 0; i < written.size(); ++i) {
      for (const Extent& r : read)
        if (written[i].meets(r)) return true;
      for (size_t j = 0; j < i; ++j)
        if (written[i].meets(written[j])) return true;
    }
    return false;
  }
};

Memory inputs_of(const sr_ffn_shape& s, int size) {
  Memory m;
  for (const Matrix& x : {matrix_x(s), matrix_gate(s), matrix_up(s), matrix_down(s)}) m.read.push_back({x.data, extent(x, size)});
  return m;
}

int check_workspace(const char* who, const void* workspace, uint64_t bytes, uint64_t need) {
  if (bytes < need || (need && workspace == nullptr))
    return fail(SR_EINVAL, "%s: a workspace of %llu bytes, %llu are needed", who, (unsigned long long)bytes,
                (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(SR_EALIGN, "%s: the workspace is not aligned", who);
  return SR_OK;
}

int check_out(const char* who, const char* what, const void* p, uint64_t n, int size) {
  if (n && p == nullptr) return fail(SR_EINVAL, "%s: %s is null", who, what);
  if (reinterpret_cast<uintptr_t>(p) % size) return fail(SR_EALIGN, "%s: %s is not aligned to its elements", who, what);
  return SR_OK;
}

template <typename F>
int typed(int32_t dtype, F&& f) {
  if (dtype == SR_DT_F32) return f(float());
  if (dtype == SR_DT_BF16) return f(bf16());
  return f(f16());
}

int forward_of(const sr_ffn_shape& s, void* out, void* a, void* b, Space& space, bool launch, hipStream_t stream) {
  return typed(s.dtype, [&](auto t) { return forward<decltype(t)>(s, out, a, b, space, launch, stream); });
}

int backward_of(const sr_ffn_shape& s, const void* a, const void* b, const void* dy, uint64_t dy_stride,
                const sr_ffn_grads& g, Space& space, bool launch, hipStream_t stream) {
  return typed(s.dtype, [&](auto t) { return backward<decltype(t)>(s, a, b, dy, dy_stride, g, space, launch, stream); });
}

}  // namespace

extern "C" {

int sr_ffn_workspace(const sr_ffn_shape* s, int32_t keep, uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_ffn_workspace: null argument");
  if (int rc = check_shape("sr_ffn_workspace", s)) return rc;
  Space space{nullptr};
  void* kept = keep ? reinterpret_cast<void*>(16) : nullptr;
  if (int rc = forward_of(*s, nullptr, kept, kept, space, false, nullptr)) return rc;
  *bytes = space.used;
  return SR_OK;
}

int sr_ffn(const sr_ffn_shape* s, void* out, float* gate_out, float* up_out, void* workspace, uint64_t workspace_bytes,
           hipStream_t stream) try {
  const char* who = "sr_ffn";
  if (int rc = check_shape(who, s)) return rc;
  const int size = sr_internal::dtype_size(s->dtype);
  if ((gate_out == nullptr) != (up_out == nullptr)) return fail(SR_EINVAL, "%s: gate_out and up_out go together", who);
  if (int rc = check_out(who, "out", out, s->tokens * s->hidden, size)) return rc;
  if (int rc = check_out(who, "gate_out", gate_out, 0, 4)) return rc;
  if (int rc = check_out(who, "up_out", up_out, 0, 4)) return rc;
  Space space{nullptr};
  if (int rc = forward_of(*s, out, gate_out, up_out, space, false, nullptr)) return rc;
  if (int rc = check_workspace(who, workspace, workspace_bytes, space.used)) return rc;
  Memory m = inputs_of(*s, size);
  m.written = {{out, s->tokens * s->hidden * size},
               {gate_out, s->tokens * s->ffn * 4},
               {up_out, s->tokens * s->ffn * 4},
               {workspace, space.used}};
  if (m.clash()) return fail(SR_EOVERLAP, "%s: an output or the workspace overlaps other memory of the call", who);
  space = {static_cast<char*>(workspace)};
  return forward_of(*s, out, gate_out, up_out, space, true, stream);
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "sr_ffn: out of host memory");
}

int sr_ffn_grad_workspace(const sr_ffn_shape* s, const void* grad_out, uint64_t grad_out_stride, const sr_ffn_grads* grads,
                          uint64_t* bytes) {
  const char* who = "sr_ffn_grad_workspace";
  if (bytes == nullptr || grads == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (int rc = check_shape(who, s)) return rc;
  if (int rc = check_matrix(who, "grad_out", {grad_out, s->tokens, s->hidden, grad_out_stride},
                            sr_internal::dtype_size(s->dtype)))
    return rc;
  Space space{nullptr};
  if (int rc = backward_of(*s, nullptr, nullptr, grad_out, grad_out_stride, *grads, space, false, nullptr)) return rc;
  *bytes = space.used;
  return SR_OK;
}

int sr_ffn_grad(const sr_ffn_shape* s, const float* gate_out, const float* up_out, const void* grad_out,
                uint64_t grad_out_stride, const sr_ffn_grads* grads, void* workspace, uint64_t workspace_bytes,
                hipStream_t stream) try {
  const char* who = "sr_ffn_grad";
  if (grads == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (int rc = check_shape(who, s)) return rc;
  const int size = sr_internal::dtype_size(s->dtype);
  const Matrix dy{grad_out, s->tokens, s->hidden, grad_out_stride}, kept{nullptr, s->tokens, s->ffn, s->ffn};
  if (int rc = check_matrix(who, "grad_out", dy, size)) return rc;
  for (const float* p : {gate_out, up_out})
    if (int rc = check_matrix(who, p == gate_out ? "gate_out" : "up_out", {p, kept.rows, kept.columns, kept.stride}, 4))
      return rc;
  const uint64_t inner = s->hidden * s->ffn;
  for (const void* p : {grads->x, grads->gate, grads->up, grads->down})
    if (int rc = check_out(who, "a gradient", p, 0, size)) return rc;
  Space space{nullptr};
  if (int rc = backward_of(*s, gate_out, up_out, grad_out, grad_out_stride, *grads, space, false, nullptr)) return rc;
  if (int rc = check_workspace(who, workspace, workspace_bytes, space.used)) return rc;
  Memory m = inputs_of(*s, size);
  m.read.push_back({grad_out, extent(dy, size)});
  m.read.push_back({gate_out, extent(kept, 4)});
  m.read.push_back({up_out, extent(kept, 4)});
  m.written = {{grads->x, s->tokens * s->hidden * size},
               {grads->gate, inner * size},
               {grads->up, inner * size},
               {grads->down, inner * size},
               {workspace, space.used}};
  if (m.clash()) return fail(SR_EOVERLAP, "%s: a gradient or the workspace overlaps other memory of the call", who);
  space = {static_cast<char*>(workspace)};
  return backward_of(*s, gate_out, up_out, grad_out, grad_out_stride, *grads, space, true, stream);
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "sr_ffn_grad: out of host memory");
}

}  // extern "C"
