// muon.hip -- matrices made orthogonal by Newton-Schulz products, and the Muon
// update of a share's matrices (C ABI in include/suika_step.h).
//
//   X = G / max(|G|, eps), then `steps` times
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// on the shorter side: a matrix with more rows than columns is taken as its
// transpose, or the side that is whole where ranks hold parts of the other one,
// whose Gram matrices A then add up.  All matrices of a list go through a step
// together, in one launch a product.
//
// Precision.  A singular value s becomes s (a + b s^2 + c s^4), so small ones,
// and with them all that is rounded in X, grow by up to a factor of a = 3.4 a
// step, 485 in five: what 16 bits round off would be percents of the result.
// X, A and B are therefore held in 22 bits, as two f16 (sr_tile.h), scaled by
// powers of two with which they fit f16, whose largest value is 65504: singular
// values of X are held to 1.9 (check_steps), so X and A, 3.61 at most, are stored times
// 2^14, up to 59200, and B, 30 at most, times 2^11, up to 61440.  A product is three
// of f16 on the matrix cores, a third of their rate and five times that of
// 32-bit floats, and its result is nearer to the exact one than a product of
// 32-bit floats in 32-bit sums: 4e-7 to 2e-6 of the result's size after five
// steps, where plain products in 32 bits are 2e-6 to 2e-5 off.
//
// A and A A are symmetric: their tiles on and above the diagonal are formed and
// stored twice, so a step takes m^2 n + m^3 + 2 m^2 n operations of 4 m^2 n + 2 m^3.
//
// Bound by the matrix cores.  The seven matrices of a Llama2-7B block at TP2 (bf16):
// A 0.97 ms a step, B 0.71, X 1.82 to 1.85, the last X into its place 1.85 to 2.0; the
// norms 50 us and the scaled X 111 us once, at 5 to 6 TB/s.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "suika_step.h"
#include "sr_step.h"
#include "sr_tile.h"

namespace {

using namespace sr_step;
using sr_tile::COL;
using sr_tile::Operand;
using sr_tile::Product;
using sr_tile::ROW;
using sr_tile::Shared;

constexpr float kX = 16384.0f, kB = 2048.0f;     // what X and A, and B, are stored times
constexpr uint64_t kMostSide = uint64_t(1) << 19;

// ------------------------------------------------------------------- tables

// A matrix on its way: m rows of the Gram side, n columns.
struct Entry {
  uint64_t x, y;           // X, and the next one
  uint64_t a, b;
  uint64_t gram;           // floats, where ranks add them up, or 0
  uint32_t m, n;
  uint32_t from;           // its first work item
};

constexpr int kEntries = 48;

template <typename E>
struct Table {
  E entry[kEntries];
  uint32_t count, items;

  // The entry of a work item: entries are compared all at once.
  __device__ __forceinline__ uint32_t find(uint32_t item) const {
    const uint32_t lane = threadIdx.x % kWave;
    const bool in = lane < count && entry[lane < count ? lane : 0].from <= item;
    return __builtin_amdgcn_readfirstlane(uint32_t(__popcll(__ballot(in)))) - 1;
  }
};

__host__ __device__ inline uint32_t whole(uint32_t n) { return (n + 31) / 32 * 32; }

// Where value (row, column) of a matrix of two f16 lies, and its rows' length.
__device__ __forceinline__ uint64_t place(uint32_t row, uint32_t column, uint32_t columns) {
  return uint64_t(row) * (2 * whole(columns)) + column / 32 * 64 + column % 32;
}

__device__ __forceinline__ void store_two(f16* p, const float (&v)[8]) {
  Vec<f16, 8> hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = static_cast<f16>(v[e]);
    lo[e] = static_cast<f16>(v[e] - static_cast<float>(hi[e]));
  }
  *reinterpret_cast<Vec<f16, 8>*>(p) = hi;
  *reinterpret_cast<Vec<f16, 8>*>(p + 32) = lo;
}

struct Two {
  VecAt<f16, 8>::packed hi, lo;

  __device__ __forceinline__ float operator[](int e) const { return static_cast<float>(hi[e]) + static_cast<float>(lo[e]); }
};

__device__ __forceinline__ Two load_two(const f16* p) {
  return {*reinterpret_cast<const Vec<f16, 8>*>(p), *reinterpret_cast<const Vec<f16, 8>*>(p + 32)};
}

// ------------------------------------------------------ momentum, norm and X

// Squares of 64 x 64 values a workgroup, the same for the sums and for X.
constexpr uint32_t kSheet = 64;
constexpr int kSheetThreads = 256;

struct SourceEntry {
  uint64_t source;         // gradient, or the matrix itself
  uint64_t momentum;       // or 0
  uint64_t stride;         // of the source's rows
  uint64_t x;
  uint32_t rows, columns;
  uint32_t from, at;
  int32_t source_type, momentum_type;
  uint32_t flip;           // X is the transpose
  uint32_t sheets;         // before its first one, in all tables
};

struct Mix {
  float keep, add;         // momentum = keep momentum + add gradient
  uint32_t nesterov;
  float max_norm;
  const double* square_sum;
};

__device__ __forceinline__ void load_typed(uint64_t p, uint64_t at, int32_t type, float (&v)[8], uint32_t n) {
  if (type == SR_DT_F32) load_row(global<const float>(p) + at, v, n);
  else if (type == SR_DT_BF16) load_row(global<const bf16>(p) + at, v, n);
  else load_row(global<const f16>(p) + at, v, n);
}

__device__ __forceinline__ void store_typed(uint64_t p, uint64_t at, int32_t type, const float (&v)[8], uint32_t n) {
  if (type == SR_DT_F32) store_row(global<float>(p) + at, v, n);
  else if (type == SR_DT_BF16) store_row(global<bf16>(p) + at, v, n);
  else store_row(global<f16>(p) + at, v, n);
}

// Eight values that are made orthogonal.  UPDATE: the momentum is updated (and
// counts as it is stored), otherwise it has been.
template <bool UPDATE>
__device__ __forceinline__ void source_row(const SourceEntry& e, const Mix& mix, float factor, uint32_t row,
                                           uint32_t column, float (&v)[8], uint32_t n) {
  load_typed(e.source, row * e.stride + column, e.source_type, v, n);
  if (!e.momentum) return;
  const uint64_t at = uint64_t(row) * e.columns + column;
  float m[8];
  load_typed(e.momentum, at, e.momentum_type, m, n);
  if (UPDATE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = fmaf(m[i], mix.keep, factor * v[i] * mix.add);
      if (e.momentum_type == SR_DT_BF16) m[i] = static_cast<float>(static_cast<bf16>(m[i]));
    }
    store_typed(e.momentum, at, e.momentum_type, m, n);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = mix.nesterov ? fmaf(m[i], mix.keep, factor * v[i] * mix.add) : m[i];
}

// The sum of the squares of every sheet, in 64 bits, with the momentum's update.
__global__ __launch_bounds__(kSheetThreads) void sums_kernel(Table<SourceEntry> t, Mix mix, double* parts) {
  const SourceEntry& e = t.entry[t.find(blockIdx.x)];
  const uint32_t sheet = blockIdx.x - e.from, across = (e.columns + kSheet - 1) / kSheet;
  const uint32_t row0 = sheet / across * kSheet, column = sheet % across * kSheet + threadIdx.x % 8 * 8;
  const float factor = mix.square_sum ? clip_factor(*mix.square_sum, mix.max_norm) : 1.0f;
  double sum = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t row = row0 + i * 32 + threadIdx.x / 8;
    if (row >= e.rows || column >= e.columns) continue;
    float v[8];
    source_row<true>(e, mix, factor, row, column, v, e.columns - column);
    // what lies behind the row's end was loaded as 0, and its momentum is 0
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fma(double(v[k]), double(v[k]), sum);
  }
  __shared__ double part[kSheetThreads / kWave];
  sum = wave_sum(sum);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) parts[e.sheets + sheet] = (part[0] + part[1]) + (part[2] + part[3]);
}

// The sums of matrices, a workgroup each, in order.
__global__ __launch_bounds__(kSheetThreads) void join_sums_kernel(Table<SourceEntry> t, const double* parts, double* sums) {
  const SourceEntry& e = t.entry[blockIdx.x];
  const uint32_t n = ((e.columns + kSheet - 1) / kSheet) * ((e.rows + kSheet - 1) / kSheet);
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kSheetThreads) sum += parts[e.sheets + i];
  __shared__ double part[kSheetThreads / kWave];
  sum = wave_sum(sum);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) sums[e.at] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X of a norm of 1 at most, as two f16, padded with zeros to whole steps.
__global__ __launch_bounds__(kSheetThreads) void scale_kernel(Table<SourceEntry> t, Mix mix, const double* sums, double eps) {
  const SourceEntry& e = t.entry[t.find(blockIdx.x)];
  const uint32_t sheet = blockIdx.x - e.from, across = (e.columns + kSheet - 1) / kSheet;
  const uint32_t row0 = sheet / across * kSheet, column0 = sheet % across * kSheet;
  const double norm = sqrt(sums[e.at]);
  const double scale = norm == 0 ? 0.0 : double(kX) / (norm < eps ? eps : norm);      // a NaN stays one
  const float factor = mix.square_sum ? clip_factor(*mix.square_sum, mix.max_norm) : 1.0f;
  __shared__ float turned[kSheet][kSheet + 1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = i * 32 + threadIdx.x / 8, c = threadIdx.x % 8 * 8, row = row0 + r, column = column0 + c;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row < e.rows && column < e.columns) {
      source_row<false>(e, mix, factor, row, column, v, e.columns - column);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = static_cast<float>(double(v[k]) * scale);
    }
    if (e.flip) {
#pragma unroll
      for (int k = 0; k < 8; ++k) turned[c + k][r] = v[k];
    } else if (row < e.rows && column < whole(e.columns)) {
      store_two(global<f16>(e.x) + place(row, column, e.columns), v);
    }
  }
  if (!e.flip) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = i * 32 + threadIdx.x / 8, c = threadIdx.x % 8 * 8, row = column0 + r, column = row0 + c;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = turned[r][c + k];
    if (row < e.columns && column < whole(e.rows)) store_two(global<f16>(e.x) + place(row, column, e.rows), v);
  }
}

// ------------------------------------------------------------------ products

// The tile on or above the diagonal of `side` x `side` tiles, in bands of 8
// columns and row by row in a band: neighbours share rows and columns (56% of the
// reads hit the L2 where tiles come column by column).
__device__ __forceinline__ void triangle(uint32_t item, uint32_t side, uint32_t& row, uint32_t& column) {
  constexpr uint32_t kBand = 8;
  // bands before b have 32 b b + 4 b tiles
  uint32_t b = uint32_t((sqrtf(16.0f + 128.0f * float(item)) - 4.0f) / 64.0f);
  while (b && 32 * b * b + 4 * b > item) --b;
  while (32 * (b + 1) * (b + 1) + 4 * (b + 1) <= item) ++b;
  item -= 32 * b * b + 4 * b;
  const uint32_t first = b * kBand, wide = side - first < kBand ? side - first : kBand;
  if (item < first * wide) {
    row = item / wide;
    column = first + item % wide;
    return;
  }
  item -= first * wide;
  uint32_t in = 0;
  while (item >= wide - in) item -= wide - in++;
  row = first + in;
  column = row + item;
}

__host__ __device__ inline uint32_t tiles(uint32_t n, int size) { return (n + size - 1) / size; }

struct Polynomial {
  float a, b, c;
};

// A matrix of two f16 with m rows of k values, or with rows of a product side by
// side, as an operand.
__device__ __forceinline__ Operand rows_of(uint64_t data, uint32_t m, uint32_t k) { return {data, 4ull * whole(k), m}; }
__device__ __forceinline__ Operand columns_of(uint64_t data, uint32_t n) { return {data, 4ull * whole(n), 2 * whole(n)}; }

// SQUARE false: A = X X^T, or its floats where ranks add them up.  SQUARE true:
// B = b A + c A A.
template <int SIZE, bool SQUARE>
__global__ __launch_bounds__(sr_tile::threads<f16>(SIZE), 2) void symmetric_kernel(Table<Entry> t, Polynomial p) {
  typedef sr_tile::Tile<f16, true, SIZE, ROW, ROW> Tile;
  SR_TILE_MEMORY(Tile);
  uint32_t item = sr_tile::item_of(blockIdx.x, t.items, SIZE);
  if (item >= t.items) return;
  const Entry& e = t.entry[t.find(item)];
  uint32_t row, column;
  triangle(item - e.from, tiles(e.m, SIZE), row, column);
  const bool diagonal = row == column;
  row *= SIZE;
  column *= SIZE;
  const uint32_t k = SQUARE ? e.m : e.n;
  const Operand side = rows_of(SQUARE ? e.a : e.x, e.m, k);
  Tile tile;
  sr_tile::run(tile, Product{side, side, {}, {}, whole(k)}, row, column, 0, whole(k) / Tile::kK, (Shared)a0, (Shared)a1,
               (Shared)b0, (Shared)b1);
  __syncthreads();
  auto load = [&](uint32_t r, uint32_t c) {
    if (!SQUARE || r >= e.m || c >= whole(e.m)) return Two{};
    return load_two(global<const f16>(e.a) + place(r, c, e.m));
  };
  auto store = [&](uint32_t r, uint32_t c, const float (&x)[8], const Two& a) {
    if (r >= e.m || c >= whole(e.m)) return;
    float v[8];
    if (SQUARE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(a[i], p.b * (kB / kX), x[i] * (p.c * (kB / (kX * kX))));
      store_two(global<f16>(e.b) + place(r, c, e.m), v);
    } else if (e.gram) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x[i] * (1 / (kX * kX));
      if (c < e.m) store_row(global<float>(e.gram) + uint64_t(r) * e.m + c, v, e.m - c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x[i] * (1 / kX);
      store_two(global<f16>(e.a) + place(r, c, e.m), v);
    }
  };
  tile.template results<false, false>(
      SR_TILE_SLAB(Tile), [&](uint32_t r, uint32_t c) { return load(row + r, column + c); },
      [&](uint32_t r, uint32_t c, const float (&x)[8], const Two& a) { store(row + r, column + c, x, a); });
  if (diagonal) return;
  tile.template results<true, false>(
      SR_TILE_SLAB(Tile), [&](uint32_t r, uint32_t c) { return load(column + r, row + c); },
      [&](uint32_t r, uint32_t c, const float (&x)[8], const Two& a) { store(column + r, row + c, x, a); });
}

// A from the floats that the ranks added up.
__global__ __launch_bounds__(kSheetThreads) void halves_kernel(Table<Entry> t) {
  const Entry& e = t.entry[t.find(blockIdx.x)];
  const uint32_t across = tiles(e.m, kSheet), sheet = blockIdx.x - e.from;
  const uint32_t column = sheet % across * kSheet + threadIdx.x % 8 * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t row = sheet / across * kSheet + i * 32 + threadIdx.x / 8;
    if (row >= e.m || column >= whole(e.m)) continue;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (column < e.m) load_row(global<const float>(e.gram) + uint64_t(row) * e.m + column, v, e.m - column);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= kX;
    store_two(global<f16>(e.a) + place(row, column, e.m), v);
  }
}

// What B X lacks is a X, added to the whole sum: as a on B's diagonal it would be
// rounded with every step of the sum, which early on is far smaller (3.8e-6 of the
// result's size off instead of 1.7e-6 after five steps of 768 x 768).

// Eight values of X, where there are any.
template <typename E>
__device__ __forceinline__ Two old_x(const E& e, uint32_t row, uint32_t column) {
  if (row >= e.m || column >= whole(e.n)) return Two{};
  return load_two(global<const f16>(e.x) + place(row, column, e.n));
}

// On a wave's values as they lie, for a result that is stored transposed; a times
// what the product is stored times.
template <typename Tile, typename E>
__device__ __forceinline__ void add_scaled(Tile& tile, const E& e, uint32_t row, uint32_t column, float a) {
  tile.values([&](uint32_t r, uint32_t c, float (&v)[4]) {
    r += row;
    c += column;
    if (r >= e.m || c >= whole(e.n)) return;
    const f16* p = global<const f16>(e.x) + place(r, c, e.n);
    const Vec<f16, 4> hi = *reinterpret_cast<const Vec<f16, 4>*>(p), lo = *reinterpret_cast<const Vec<f16, 4>*>(p + 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(static_cast<float>(hi[i]) + static_cast<float>(lo[i]), a, v[i]);
  });
}

// X <- a X + B X.
template <int SIZE>
__global__ __launch_bounds__(sr_tile::threads<f16>(SIZE), 2) void update_kernel(Table<Entry> t, float a) {
  typedef sr_tile::Tile<f16, true, SIZE, ROW, COL> Tile;
  SR_TILE_MEMORY(Tile);
  uint32_t item = sr_tile::item_of(blockIdx.x, t.items, SIZE);
  if (item >= t.items) return;
  const Entry& e = t.entry[t.find(item)];
  uint32_t row, column;
  sr_tile::banded(item - e.from, tiles(e.m, SIZE), tiles(e.n, SIZE), row, column);
  row *= SIZE;
  column *= SIZE;
  Tile tile;
  sr_tile::run(tile, Product{rows_of(e.b, e.m, e.m), columns_of(e.x, e.n), {}, {}, e.m}, row, column, 0,
               whole(e.m) / Tile::kK, (Shared)a0, (Shared)a1, (Shared)b0, (Shared)b1);
  __syncthreads();
  tile.template results<false, false>(
      SR_TILE_SLAB(Tile), [&](uint32_t r, uint32_t c) { return old_x(e, row + r, column + c); },
      [&](uint32_t r, uint32_t c, const float (&x)[8], const Two& old) {
        r += row;
        c += column;
        if (r >= e.m || c >= whole(e.n)) return;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(old[i], a, x[i] * (1 / kB));
        store_two(global<f16>(e.y) + place(r, c, e.n), v);
      });
}

// The last X goes to its destination, or into the weight.
struct LastEntry {
  uint64_t x, b;
  uint64_t to;             // the result, or the weight
  uint64_t param;          // the weight's copy in bf16, or 0
  uint64_t stride;         // of the result's rows
  uint32_t m, n;
  uint32_t from;
  int32_t type;            // of the result or the weight
  uint32_t flip;
  uint32_t weight;         // whether it is a weight
  float decay, step;       // weight = decay weight - step X
};

struct Eight {
  float v[8];
};

template <int SIZE>
__global__ __launch_bounds__(sr_tile::threads<f16>(SIZE), 2) void last_kernel(Table<LastEntry> t, float a) {
  typedef sr_tile::Tile<f16, true, SIZE, ROW, COL> Tile;
  SR_TILE_MEMORY(Tile);
  uint32_t item = sr_tile::item_of(blockIdx.x, t.items, SIZE);
  if (item >= t.items) return;
  const LastEntry& e = t.entry[t.find(item)];
  uint32_t row, column;
  sr_tile::banded(item - e.from, tiles(e.m, SIZE), tiles(e.n, SIZE), row, column);
  row *= SIZE;
  column *= SIZE;
  Tile tile;
  sr_tile::run(tile, Product{rows_of(e.b, e.m, e.m), columns_of(e.x, e.n), {}, {}, e.m}, row, column, 0,
               whole(e.m) / Tile::kK, (Shared)a0, (Shared)a1, (Shared)b0, (Shared)b1);
  if (e.flip) add_scaled(tile, e, row, column, a * kB);
  __syncthreads();
  // the weight that is there
  auto load = [&](uint32_t r, uint32_t c, uint32_t rows, uint32_t columns) {
    Eight w{};
    if (e.weight && r < rows && c < columns) load_typed(e.to, r * e.stride + c, e.type, w.v, columns - c);
    return w;
  };
  auto store = [&](uint32_t r, uint32_t c, uint32_t rows, uint32_t columns, const float (&x)[8], const Eight& w) {
    if (r >= rows || c >= columns) return;
    const uint64_t at = r * e.stride + c;
    const uint32_t n = columns - c;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e.weight ? fmaf(w.v[i], e.decay, -e.step * x[i]) : x[i];
    if (e.param) store_row(global<bf16>(e.param) + at, v, n);
    store_typed(e.to, at, e.type, v, n);
  };
  if (e.flip) {
    tile.template results<true, true>(
        SR_TILE_SLAB(Tile), [&](uint32_t r, uint32_t c) { return load(column + r, row + c, e.n, e.m); },
        [&](uint32_t r, uint32_t c, const float (&x)[8], const Eight& w) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = x[i] * (1 / (kX * kB));
          store(column + r, row + c, e.n, e.m, v, w);
        });
  } else {
    struct Both {
      Eight w;
      Two old;
    };
    tile.template results<false, true>(
        SR_TILE_SLAB(Tile),
        [&](uint32_t r, uint32_t c) { return Both{load(row + r, column + c, e.m, e.n), old_x(e, row + r, column + c)}; },
        [&](uint32_t r, uint32_t c, const float (&x)[8], const Both& b) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(b.old[i], a * (1 / kX), x[i] * (1 / (kX * kB)));
          store(row + r, column + c, e.m, e.n, v, b.w);
        });
  }
}

// ------------------------------------------------------------ small matrices

// A small matrix goes through everything in one workgroup and one launch, its
// values and products in shared memory and 32 bits: 8 matrices of up to 32 x 24
// take 15 us instead of 80 with tiles, whose 17 launches are most of that.
// Up to about 64 x 64 x 64 operations a product a workgroup is as fast as tiles;
// the rule looks at the matrix alone, so its result does not depend on the list.
constexpr uint32_t kSmallSide = 64, kSmallValues = 64 * 196;
constexpr uint64_t kSmallWork = uint64_t(1) << 18;

struct SmallEntry {
  uint64_t source, momentum, to, param;
  uint64_t source_stride, to_stride;
  uint32_t rows, columns;
  int32_t source_type, momentum_type, to_type;
  uint32_t flip, weight;
  float decay, step;
};

constexpr int kSmallEntries = 32;

struct SmallTable {
  SmallEntry entry[kSmallEntries];
  Polynomial step[SR_MAX_NEWTON_SCHULZ];
  Mix mix;
  double eps;
  int32_t steps;
};
static_assert(sizeof(SmallTable) <= 3832, "kernel arguments");

__device__ __forceinline__ float load_one(uint64_t p, uint64_t at, int32_t type) {
  return type == SR_DT_F32 ? global<const float>(p)[at]
                           : type == SR_DT_BF16 ? float(global<const bf16>(p)[at]) : float(global<const f16>(p)[at]);
}

__device__ __forceinline__ void store_one(uint64_t p, uint64_t at, int32_t type, float v) {
  if (type == SR_DT_F32) global<float>(p)[at] = v;
  else if (type == SR_DT_BF16) global<bf16>(p)[at] = bf16(v);
  else global<f16>(p)[at] = f16(v);
}

__host__ __device__ inline uint32_t fours(uint32_t n) { return (n + 3) / 4 * 4; }

// out(i, j, sum over k of P[i][k] Q[k][j], or of Q[j][k] with ROWS), R x R sums a
// lane; sides are multiples of 4.
template <int R, bool ROWS, typename F>
__device__ __forceinline__ void small_squares(const float* p, uint32_t p_wide, const float* q, uint32_t q_wide, uint32_t rows,
                                              uint32_t columns, uint32_t depth, F&& out) {
  using sr_tile::f32x4;
  typedef float Across __attribute__((ext_vector_type(R)));
  const uint32_t across = columns / R;
  for (uint32_t t = threadIdx.x; t < rows / R * across; t += kSheetThreads) {
    const uint32_t i = t / across * R, j = t % across * R;
    float sum[R][R] = {};
    for (uint32_t k = 0; k < depth; k += 4) {
      f32x4 a[R], b[R];
      Across c[4];
#pragma unroll
      for (int r = 0; r < R; ++r) a[r] = *reinterpret_cast<const f32x4*>(p + (i + r) * p_wide + k);
      if (ROWS) {
#pragma unroll
        for (int r = 0; r < R; ++r) b[r] = *reinterpret_cast<const f32x4*>(q + (j + r) * q_wide + k);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] = *reinterpret_cast<const Across*>(q + (k + r) * q_wide + j);
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int x = 0; x < R; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[r][x] = fmaf(a[r][e], ROWS ? b[x][e] : c[e][x], sum[r][x]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = 0; x < R; ++x) out(i + r, j + x, sum[r][x]);
  }
}

// Smaller squares where that gives more lanes work.
template <bool ROWS, typename F>
__device__ __forceinline__ void small_product(const float* p, uint32_t p_wide, const float* q, uint32_t q_wide, uint32_t rows,
                                              uint32_t columns, uint32_t depth, F&& out) {
  if (rows * columns <= 4 * kSheetThreads) small_squares<2, ROWS>(p, p_wide, q, q_wide, rows, columns, depth, out);
  else small_squares<4, ROWS>(p, p_wide, q, q_wide, rows, columns, depth, out);
}

__global__ __launch_bounds__(kSheetThreads) void small_kernel(SmallTable t) {
  constexpr uint32_t kGram = kSmallSide * (kSmallSide + 4);
  __shared__ __attribute__((aligned(16))) float first[kSmallValues + kSmallSide * 4], second[kSmallValues + kSmallSide * 4],
      gram[kGram], factor[kGram];
  __shared__ double part[kSheetThreads / kWave];
  const SmallEntry& e = t.entry[blockIdx.x];
  const uint32_t m = e.flip ? e.columns : e.rows, n = e.flip ? e.rows : e.columns;
  const uint32_t high = fours(m), wide = fours(n) + 4, side = fours(m) + 4;
  for (uint32_t i = threadIdx.x; i < high * wide; i += kSheetThreads) first[i] = second[i] = 0;
  __syncthreads();
  const float clip = t.mix.square_sum ? clip_factor(*t.mix.square_sum, t.mix.max_norm) : 1.0f;
  const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const uint32_t values = e.rows * e.columns;
  constexpr uint32_t kAhead = 4;      // values of a lane that are loaded at once
  double squares = 0;
  for (uint32_t i = threadIdx.x; i < values; i += kAhead * kSheetThreads) {
    float v[kAhead], old[kAhead];
    uint32_t row[kAhead], column[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      const uint32_t at = min(i + a * kSheetThreads, values - 1);
      row[a] = at / e.columns;
      column[a] = at % e.columns;
      v[a] = load_one(e.source, row[a] * e.source_stride + column[a], e.source_type);
      old[a] = e.momentum ? load_one(e.momentum, at, e.momentum_type) : 0.0f;
    }
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      const uint32_t at = i + a * kSheetThreads;
      if (at >= values) continue;
      if (e.momentum) {
        float m = fmaf(old[a], t.mix.keep, clip * v[a] * t.mix.add);
        if (e.momentum_type == SR_DT_BF16) m = float(bf16(m));
        store_one(e.momentum, at, e.momentum_type, m);
        v[a] = t.mix.nesterov ? fmaf(m, t.mix.keep, clip * v[a] * t.mix.add) : m;
      }
      squares = fma(double(v[a]), double(v[a]), squares);
      first[e.flip ? column[a] * wide + row[a] : row[a] * wide + column[a]] = v[a];
    }
  }
  squares = wave_sum(squares);
  if (lane == 0) part[wave] = squares;
  __syncthreads();
  const double norm = sqrt((part[0] + part[1]) + (part[2] + part[3]));
  const double scale = 1.0 / (norm < t.eps ? t.eps : norm);
  for (uint32_t i = threadIdx.x; i < high * wide; i += kSheetThreads) first[i] = norm == 0 ? 0.0f : float(double(first[i]) * scale);
  __syncthreads();
  float *x = first, *y = second;
  for (int32_t k = 0; k < t.steps; ++k) {
    const Polynomial p = t.step[k];
    small_product<true>(x, wide, x, wide, high, high, wide - 4,
                        [&](uint32_t i, uint32_t j, float v) { gram[i * side + j] = v; });
    __syncthreads();
    small_product<false>(gram, side, gram, side, high, high, high, [&](uint32_t i, uint32_t j, float v) {
      factor[i * side + j] = fmaf(gram[i * side + j], p.b, p.c * v);
    });
    __syncthreads();
    small_product<false>(factor, side, x, wide, high, wide - 4, high,
                         [&](uint32_t i, uint32_t j, float v) { y[i * wide + j] = fmaf(x[i * wide + j], p.a, v); });
    __syncthreads();
    float* const z = x;
    x = y;
    y = z;
  }
  for (uint32_t i = threadIdx.x; i < values; i += kAhead * kSheetThreads) {
    float v[kAhead];
    uint64_t to[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      const uint32_t at = min(i + a * kSheetThreads, values - 1), row = at / e.columns, column = at % e.columns;
      to[a] = row * e.to_stride + column;
      v[a] = x[e.flip ? column * wide + row : row * wide + column];
      if (e.weight) v[a] = fmaf(load_one(e.to, to[a], e.to_type), e.decay, -e.step * v[a]);
    }
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
      if (i + a * kSheetThreads >= values) continue;
      if (e.param) global<bf16>(e.param)[to[a]] = bf16(v[a]);
      store_one(e.to, to[a], e.to_type, v[a]);
    }
  }
}

static_assert(sizeof(Table<SourceEntry>) + 32 <= 4064 && sizeof(Table<Entry>) <= 3832 && sizeof(Table<LastEntry>) <= 4064,
              "kernel arguments");

// ---------------------------------------------------------------------- host

// One matrix of a call.
struct Work {
  const void* source;
  void* momentum;
  void* to;
  void* param;
  uint64_t rows, columns, source_stride, to_stride;
  int32_t source_type, momentum_type, to_type;
  int32_t split;
  bool weight;
  float decay, step;

  // The Gram matrix is that of the shorter side, or of the side that is whole.
  bool flip() const { return split < 0 ? rows > columns : split == 0; }
  uint32_t m() const { return uint32_t(flip() ? columns : rows); }
  uint32_t n() const { return uint32_t(flip() ? rows : columns); }
  // Whether it goes through one workgroup: what does not fit shared memory, or is
  // summed up over ranks, does not.
  bool small() const {
    return split < 0 && m() <= kSmallSide && uint64_t(fours(m())) * fours(n()) <= kSmallValues &&
           uint64_t(m()) * m() * n() <= kSmallWork;
  }
  bool empty() const { return split < 0 ? rows == 0 || columns == 0 : m() == 0; }
};

struct Space {
  char* base;
  uint64_t used = 0, most = 0;

  uint64_t take(uint64_t bytes) {
    const uint64_t at = used;
    used += (bytes + 255) / 256 * 256;
    most = std::max(most, used);
    return reinterpret_cast<uint64_t>(base) + at;
  }
};

uint64_t x_bytes(const Work& w) { return uint64_t(w.m()) * whole(w.n()) * 4; }
uint64_t gram_bytes(const Work& w) { return uint64_t(w.m()) * whole(w.m()) * 4; }

// Matrices that go through the steps together.  Ranks that add Gram matrices up
// have the same ones in a group: it goes by what is the same on all of them, the Gram
// matrices, and the memory of X comes on top.
constexpr uint64_t kGroupBytes = uint64_t(8) << 30;

struct Group {
  std::vector<const Work*> work;
  bool split;
};

std::vector<Group> groups_of(const std::vector<Work>& all) {
  std::vector<Group> groups;
  for (bool split : {false, true}) {
    std::vector<const Work*> some;
    for (const Work& w : all)
      if ((w.split >= 0) == split && !w.empty() && !w.small()) some.push_back(&w);
    // long tiles first: what remains at a launch's end is short
    std::stable_sort(some.begin(), some.end(), [&](const Work* a, const Work* b) {
      return a->m() != b->m() ? a->m() > b->m() : !split && a->n() > b->n();
    });
    uint64_t bytes = 0;
    for (const Work* w : some) {
      const uint64_t more = split ? 3 * gram_bytes(*w) : 2 * (x_bytes(*w) + gram_bytes(*w));
      if (groups.empty() || groups.back().split != split || groups.back().work.size() == kEntries ||
          bytes + more > kGroupBytes) {
        groups.push_back({{}, split});
        bytes = 0;
      }
      groups.back().work.push_back(w);
      bytes += more;
    }
  }
  return groups;
}

template <typename E, typename F>
int number(Table<E>& t, uint64_t most, F&& items) {
  uint64_t sum = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.entry[i].from = uint32_t(sum);
    sum += items(t.entry[i]);
    if (sum > most) return fail(SR_EBOUNDS, "more tiles than a launch takes");
  }
  t.items = uint32_t(sum);
  return SR_OK;
}

// The tiles' size by the time that a launch takes with either, and the items of
// the tables that have it.  `tiles_of` counts an entry's tiles, `depth_of` their
// steps.
template <typename E, typename F, typename G>
int number_tiles(Table<E>& t, int& size, F&& tiles_of, G&& depth_of) {
  sr_tile::Cost large(256, false), small(128, false);
  for (uint32_t i = 0; i < t.count; ++i) {
    large.add(tiles_of(t.entry[i], 256), depth_of(t.entry[i]));
    small.add(tiles_of(t.entry[i], 128), depth_of(t.entry[i]));
  }
  size = large.time() <= small.time() ? 256 : 128;
  return number(t, sr_tile::kMostItems, [&](const E& e) { return tiles_of(e, size); });
}

template <typename E> uint64_t triangle_tiles(const E& e, int size) {
  const uint64_t n = tiles(e.m, size);
  return n * (n + 1) / 2;
}
template <typename E> uint64_t all_tiles(const E& e, int size) { return uint64_t(tiles(e.m, size)) * tiles(e.n, size); }

struct Steps {
  const sr_newton_schulz* ns;
  Mix mix;
  const char* who;
};

int reduce(const Steps& s, uint64_t data, uint64_t count, int32_t dtype, hipStream_t stream) {
  const int rc = s.ns->reduce(s.ns->reduce_context, reinterpret_cast<void*>(data), count, dtype, stream);
  return rc == 0 ? int(SR_OK) : fail(SR_EINVAL, "%s: the sum over the ranks failed (%d)", s.who, rc);
}

// A group's matrices as they are given, in sheets; their X come later.
int sources_of(const Group& g, Table<SourceEntry>& source) {
  source.count = uint32_t(g.work.size());
  uint64_t sheets = 0;
  for (size_t i = 0; i < g.work.size(); ++i) {
    const Work& w = *g.work[i];
    source.entry[i] = {reinterpret_cast<uint64_t>(w.source), reinterpret_cast<uint64_t>(w.momentum), w.source_stride, 0,
                       uint32_t(w.rows), uint32_t(w.columns), 0, uint32_t(i), w.source_type, w.momentum_type, w.flip(),
                       uint32_t(sheets)};
    sheets += uint64_t(tiles(uint32_t(w.rows), kSheet)) * tiles(uint32_t(w.columns), kSheet);
  }
  return number(source, (uint64_t(1) << 24) - 1,
                [](const SourceEntry& e) { return uint64_t(tiles(e.rows, kSheet)) * tiles(e.columns, kSheet); });
}

// The momentum's update and the squares' sums of a group.
int run_sums(const Group& g, const Steps& s, uint64_t sums, Space& space, bool launch, hipStream_t stream) {
  Table<SourceEntry> source{};
  if (int rc = sources_of(g, source)) return rc;
  double* const parts = reinterpret_cast<double*>(space.take(source.items * sizeof(double)));
  if (!launch) return SR_OK;
  if (source.items) sums_kernel<<<source.items, kSheetThreads, 0, stream>>>(source, s.mix, parts);
  join_sums_kernel<<<source.count, kSheetThreads, 0, stream>>>(source, parts, reinterpret_cast<double*>(sums));
  return launched(s.who);
}

// The steps of a group.
int run_steps(const Group& g, const Steps& s, uint64_t sums, Space& space, bool launch, hipStream_t stream) {
  Table<SourceEntry> source{};
  if (int rc = sources_of(g, source)) return rc;
  Table<Entry> t{};
  Table<LastEntry> last{};
  t.count = last.count = uint32_t(g.work.size());
  uint64_t gram_floats = 0;
  for (size_t i = 0; i < g.work.size(); ++i) gram_floats += uint64_t(g.work[i]->m()) * g.work[i]->m();
  const uint64_t grams = g.split ? space.take(gram_floats * sizeof(float)) : 0;
  gram_floats = 0;
  for (size_t i = 0; i < g.work.size(); ++i) {
    const Work& w = *g.work[i];
    Entry& e = t.entry[i];
    e.x = space.take(x_bytes(w));
    e.y = space.take(x_bytes(w));
    e.a = space.take(gram_bytes(w));
    e.b = space.take(gram_bytes(w));
    e.m = w.m();
    e.n = w.n();
    if (g.split) {
      e.gram = grams + gram_floats * sizeof(float);
      gram_floats += uint64_t(e.m) * e.m;
    }
    source.entry[i].x = e.x;
    last.entry[i] = {0, e.b, reinterpret_cast<uint64_t>(w.to), reinterpret_cast<uint64_t>(w.param), w.to_stride, e.m, e.n, 0,
                     w.to_type, w.flip(), w.weight, w.decay, w.step};
  }
  int large = 0, wide = 0;
  Table<Entry> gram = t, update = t;
  // A and A A have the same tiles; the steps are counted of both
  if (int rc = number_tiles(gram, large, triangle_tiles<Entry>, [](const Entry& e) { return (whole(e.m) + whole(e.n)) / 64; }))
    return rc;
  if (int rc = number_tiles(update, wide, all_tiles<Entry>, [](const Entry& e) { return whole(e.m) / 32; })) return rc;
  if (int rc = number(last, sr_tile::kMostItems, [&](const LastEntry& e) { return all_tiles(e, wide); })) return rc;
  Table<Entry> halves = t;
  if (int rc = number(halves, (uint64_t(1) << 24) - 1, [](const Entry& e) { return uint64_t(tiles(e.m, kSheet)) * tiles(e.m, kSheet); })) return rc;
  if (!launch) return SR_OK;

  double* const sum = reinterpret_cast<double*>(sums);
  if (g.split) {
    if (int rc = reduce(s, sums, source.count, SR_DT_F64, stream)) return rc;
  }
  if (source.items) scale_kernel<<<source.items, kSheetThreads, 0, stream>>>(source, s.mix, sum, s.ns->eps);
  for (int32_t k = 0; k < s.ns->steps; ++k) {
    const double* c = s.ns->coefficients + 3 * k;
    const Polynomial p{float(c[0]), float(c[1]), float(c[2])};
    const uint32_t blocks = sr_tile::blocks_of(gram.items, large);
    if (large == 256) symmetric_kernel<256, false><<<blocks, sr_tile::threads<f16>(256), 0, stream>>>(gram, p);
    else symmetric_kernel<128, false><<<blocks, sr_tile::threads<f16>(128), 0, stream>>>(gram, p);
    if (g.split) {
      if (int rc = launched(s.who)) return rc;
      if (int rc = reduce(s, grams, gram_floats, SR_DT_F32, stream)) return rc;
      halves_kernel<<<halves.items, kSheetThreads, 0, stream>>>(halves);
    }
    if (large == 256) symmetric_kernel<256, true><<<blocks, sr_tile::threads<f16>(256), 0, stream>>>(gram, p);
    else symmetric_kernel<128, true><<<blocks, sr_tile::threads<f16>(128), 0, stream>>>(gram, p);
    if (update.items == 0) continue;      // nothing of these matrices is here
    if (k + 1 < s.ns->steps) {
      const uint32_t many = sr_tile::blocks_of(update.items, wide);
      if (wide == 256) update_kernel<256><<<many, sr_tile::threads<f16>(256), 0, stream>>>(update, p.a);
      else update_kernel<128><<<many, sr_tile::threads<f16>(128), 0, stream>>>(update, p.a);
      for (uint32_t i = 0; i < t.count; ++i) {
        std::swap(gram.entry[i].x, gram.entry[i].y);
        std::swap(update.entry[i].x, update.entry[i].y);
      }
    } else {
      for (uint32_t i = 0; i < t.count; ++i) last.entry[i].x = update.entry[i].x;
      const uint32_t many = sr_tile::blocks_of(last.items, wide);
      if (wide == 256) last_kernel<256><<<many, sr_tile::threads<f16>(256), 0, stream>>>(last, p.a);
      else last_kernel<128><<<many, sr_tile::threads<f16>(128), 0, stream>>>(last, p.a);
    }
    if (int rc = launched(s.who)) return rc;
  }
  return SR_OK;
}

// The small ones.
int run_small(const std::vector<Work>& all, const Steps& s, hipStream_t stream) {
  SmallTable t;
  t.mix = s.mix;
  t.eps = s.ns->eps;
  t.steps = s.ns->steps;
  for (int32_t k = 0; k < s.ns->steps; ++k) {
    const double* c = s.ns->coefficients + 3 * k;
    t.step[k] = {float(c[0]), float(c[1]), float(c[2])};
  }
  int count = 0;
  auto flush = [&]() -> int {
    if (count == 0) return SR_OK;
    small_kernel<<<count, kSheetThreads, 0, stream>>>(t);
    count = 0;
    return launched(s.who);
  };
  for (const Work& w : all) {
    if (w.empty() || !w.small()) continue;
    t.entry[count++] = {reinterpret_cast<uint64_t>(w.source), reinterpret_cast<uint64_t>(w.momentum),
                        reinterpret_cast<uint64_t>(w.to), reinterpret_cast<uint64_t>(w.param), w.source_stride, w.to_stride,
                        uint32_t(w.rows), uint32_t(w.columns), w.source_type, w.momentum_type, w.to_type, w.flip(), w.weight,
                        w.decay, w.step};
    if (count == kSmallEntries) {
      if (int rc = flush()) return rc;
    }
  }
  return flush();
}

// All groups, one after another in the same memory.  All momentum is updated before
// the ranks' first sum, so that what a failing one leaves does not depend on the groups.
int run_all(const std::vector<Work>& all, const Steps& s, Space& space, bool launch, hipStream_t stream) {
  if (launch) {
    if (int rc = run_small(all, s, stream)) return rc;
  }
  const std::vector<Group> groups = groups_of(all);
  constexpr uint64_t kSums = kEntries * sizeof(double);      // of a group
  const uint64_t sums = space.take(groups.size() * kSums), shared = space.used;
  for (size_t i = 0; i < groups.size(); ++i) {
    space.used = shared;
    if (int rc = run_sums(groups[i], s, sums + i * kSums, space, launch, stream)) return rc;
  }
  for (size_t i = 0; i < groups.size(); ++i) {
    space.used = shared;
    if (int rc = run_steps(groups[i], s, sums + i * kSums, space, launch, stream)) return rc;
  }
  return SR_OK;
}

// -------------------------------------------------------------------- checks

// The iterates' singular values stay below what X and A are stored for, and B's
// below what it is: bounds on [0, high], step by step.
int check_steps(const char* who, const sr_newton_schulz* ns) {
  if (ns == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (ns->reserved != 0) return fail(SR_EINVAL, "%s: reserved is not 0", who);
  if (ns->steps < 1 || ns->steps > SR_MAX_NEWTON_SCHULZ) return fail(SR_EINVAL, "%s: %d steps", who, ns->steps);
  if (ns->coefficients == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (!(ns->eps >= 0) || !std::isfinite(ns->eps)) return fail(SR_EINVAL, "%s: eps %g", who, ns->eps);
  double high = 1.0;
  for (int32_t k = 0; k < ns->steps; ++k) {
    const double a = ns->coefficients[3 * k], b = ns->coefficients[3 * k + 1], c = ns->coefficients[3 * k + 2];
    auto weight = [&](double q) { return std::fabs(a + b * q + c * q * q); };        // of s^2
    auto value = [&](double q) { return std::sqrt(q) * weight(q); };
    const double end = high * high * 1.001;      // and what roundings add
    double most = std::max(value(end), 0.0), heavy = std::max({weight(0), weight(end), std::fabs(a)});
    // where the derivatives vanish
    std::vector<double> at;
    if (c != 0) {
      at.push_back(-b / (2 * c));
      const double root = 9 * b * b - 20 * a * c;
      if (root >= 0) {
        at.push_back((-3 * b + std::sqrt(root)) / (10 * c));
        at.push_back((-3 * b - std::sqrt(root)) / (10 * c));
      }
    } else if (b != 0) {
      at.push_back(-a / (3 * b));
    }
    for (double q : at) {
      if (!(q > 0 && q < end)) continue;
      most = std::max(most, value(q));
      heavy = std::max(heavy, weight(q));
    }
    if (!(most <= 1.9) || !(heavy <= 15.0))
      return fail(SR_EINVAL, "%s: coefficients %g, %g, %g of step %d: the iterates leave the range that they are stored in",
                  who, a, b, c, k);
    high = most;
  }
  return SR_OK;
}

int check_sides(const char* who, int32_t i, uint64_t rows, uint64_t columns, int32_t split, const sr_newton_schulz* ns) {
  if (rows > kMostSide || columns > kMostSide || rows * columns > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EBOUNDS, "%s: matrix %d of %llu x %llu", who, i, (unsigned long long)rows, (unsigned long long)columns);
  if (split < -1 || split > 1) return fail(SR_EINVAL, "%s: matrix %d: split %d", who, i, split);
  if (split >= 0 && ns->reduce == nullptr) return fail(SR_EINVAL, "%s: matrix %d is split, but there is no reduce", who, i);
  return SR_OK;
}

struct Span {
  uintptr_t from, to;
  bool written;
};

void add_span(std::vector<Span>& spans, const void* p, uint64_t bytes, bool written) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  if (p && bytes) spans.push_back({a, a + bytes, written});
}

bool clash(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  uintptr_t any = 0, written = 0;
  for (const Span& s : spans) {
    if (s.from < (s.written ? any : written)) return true;
    any = std::max(any, s.to);
    if (s.written) written = std::max(written, s.to);
  }
  return false;
}

int finish(const char* who, const std::vector<Work>& all, std::vector<Span>& spans, const Steps& s, void* workspace,
           uint64_t workspace_bytes, uint64_t* bytes, hipStream_t stream) {
  Space space{nullptr};
  if (int rc = run_all(all, s, space, false, nullptr)) return rc;
  if (bytes) *bytes = space.most;
  else {
    if (workspace_bytes < space.most || (space.most && workspace == nullptr))
      return fail(SR_EINVAL, "%s: a workspace of %llu bytes, %llu are needed", who, (unsigned long long)workspace_bytes,
                  (unsigned long long)space.most);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(SR_EALIGN, "%s: the workspace is not aligned", who);
    add_span(spans, workspace, space.most, true);
  }
  if (clash(spans)) return fail(SR_EOVERLAP, "%s: memory that is written overlaps other memory of the call", who);
  if (bytes) return SR_OK;
  space = {static_cast<char*>(workspace)};
  return run_all(all, s, space, true, stream);
}

int check_matrix(const char* who, const char* what, int32_t i, const sr_matrix& m) {
  if (!float_dtype(m.dtype)) return fail(SR_EDTYPE, "%s: %s[%d]: dtype %d", who, what, i, m.dtype);
  if (m.stride < m.cols || m.stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "%s: %s[%d]: rows %llu elements apart, %llu columns", who, what, i, (unsigned long long)m.stride,
                (unsigned long long)m.cols);
  if (m.rows && m.cols && m.data == nullptr) return fail(SR_EINVAL, "%s: %s[%d] is null", who, what, i);
  if (reinterpret_cast<uintptr_t>(m.data) % sr_internal::dtype_size(m.dtype))
    return fail(SR_EALIGN, "%s: %s[%d] is not aligned to its elements", who, what, i);
  return SR_OK;
}

uint64_t extent(const sr_matrix& m) {
  return m.rows && m.cols ? ((m.rows - 1) * m.stride + m.cols) * sr_internal::dtype_size(m.dtype) : 0;
}

// bytes: only the checks and the workspace's size.
int orthogonalize(const char* who, const sr_matrix* src, const sr_matrix* dst, int32_t count, const sr_newton_schulz* ns,
                  void* workspace, uint64_t workspace_bytes, uint64_t* bytes, hipStream_t stream) try {
  if (count < 0 || (count > 0 && (src == nullptr || dst == nullptr))) return fail(SR_EINVAL, "%s: no matrices", who);
  if (int rc = check_steps(who, ns)) return rc;
  std::vector<Work> all;
  std::vector<Span> spans;
  for (int32_t i = 0; i < count; ++i) {
    const sr_matrix &f = src[i], &t = dst[i];
    if (int rc = check_sides(who, i, f.rows, f.cols, f.split, ns)) return rc;
    if (int rc = check_matrix(who, "src", i, f)) return rc;
    if (int rc = check_matrix(who, "dst", i, t)) return rc;
    if (f.rows != t.rows || f.cols != t.cols)
      return fail(SR_EINVAL, "%s: src[%d] is %llu x %llu, dst[%d] %llu x %llu", who, i, (unsigned long long)f.rows,
                  (unsigned long long)f.cols, i, (unsigned long long)t.rows, (unsigned long long)t.cols);
    all.push_back({f.data, nullptr, t.data, nullptr, f.rows, f.cols, f.stride, t.stride, f.dtype, 0, t.dtype, f.split, false, 0, 0});
    // a matrix may be its own result: it is read before
    if (f.data != t.data || f.stride != t.stride || f.dtype != t.dtype) add_span(spans, f.data, extent(f), false);
    add_span(spans, t.data, extent(t), true);
  }
  return finish(who, all, spans, {ns, {0, 0, 0, 0, nullptr}, who}, workspace, workspace_bytes, bytes, stream);
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "%s: out of host memory", who);
}

int muon(const char* who, const sr_muon_tensor* tensors, int32_t count, const sr_muon_options* o, const sr_newton_schulz* ns,
         void* workspace, uint64_t workspace_bytes, uint64_t* bytes, hipStream_t stream) try {
  if (count < 0 || (count > 0 && tensors == nullptr) || o == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (int rc = check_steps(who, ns)) return rc;
  if (o->reserved != 0) return fail(SR_EINVAL, "%s: reserved is not 0", who);
  if (!(o->lr >= 0) || !std::isfinite(o->lr) || !(o->weight_decay >= 0) || !std::isfinite(o->weight_decay) ||
      !(o->momentum >= 0) || !(o->momentum < 1))
    return fail(SR_EINVAL, "%s: lr %g, weight_decay %g, momentum %g", who, o->lr, o->weight_decay, o->momentum);
  if (o->square_sum != nullptr && !(o->max_norm >= 0)) return fail(SR_EINVAL, "%s: max_norm %g", who, o->max_norm);
  if (reinterpret_cast<uintptr_t>(o->square_sum) % 8) return fail(SR_EALIGN, "%s: square_sum is not aligned", who);
  std::vector<Work> all;
  std::vector<Span> spans;
  for (int32_t i = 0; i < count; ++i) {
    const sr_muon_tensor& x = tensors[i];
    if (x.reserved != 0) return fail(SR_EINVAL, "%s: tensors[%d].reserved is not 0", who, i);
    if (int rc = check_sides(who, i, x.rows, x.cols, x.split, ns)) return rc;
    for (int32_t dt : {x.weight_dtype, x.moment_dtype, x.grad_dtype})
      if (dt != SR_DT_F32 && dt != SR_DT_BF16) return fail(SR_EDTYPE, "%s: tensors[%d]: dtype %d", who, i, dt);
    if (x.param != nullptr && x.weight_dtype != SR_DT_F32)
      return fail(SR_EDTYPE, "%s: tensors[%d]: a copy of a weight that is not f32", who, i);
    if (!(x.scale >= 0) || !std::isfinite(x.scale)) return fail(SR_EINVAL, "%s: tensors[%d]: scale %g", who, i, x.scale);
    const uint64_t n = x.rows * x.cols;
    if (n && (!x.weight || !x.exp_avg || !x.grad)) return fail(SR_EINVAL, "%s: tensors[%d]: a field is null", who, i);
    const int ws = sr_internal::dtype_size(x.weight_dtype), ms = sr_internal::dtype_size(x.moment_dtype),
              gs = sr_internal::dtype_size(x.grad_dtype);
    const struct { const void* p; int size; bool written; } field[4] = {
        {x.weight, ws, true}, {x.exp_avg, ms, true}, {x.param, 2, true}, {x.grad, gs, false}};
    for (const auto& f : field) {
      if (reinterpret_cast<uintptr_t>(f.p) % f.size)
        return fail(SR_EALIGN, "%s: tensors[%d]: a field is not aligned to its elements", who, i);
      add_span(spans, f.p, n * f.size, f.written);
    }
    all.push_back({x.grad, x.exp_avg, x.weight, x.param, x.rows, x.cols, x.cols, x.cols, x.grad_dtype, x.moment_dtype,
                   x.weight_dtype, x.split, true, float(1 - o->lr * o->weight_decay), float(o->lr * x.scale)});
  }
  add_span(spans, o->square_sum, sizeof(double), false);
  const Mix mix{float(o->momentum), float(1 - o->momentum), uint32_t(o->nesterov != 0), float(o->max_norm), o->square_sum};
  return finish(who, all, spans, {ns, mix, who}, workspace, workspace_bytes, bytes, stream);
} catch (const std::bad_alloc&) {
  return fail(SR_ENOMEM, "%s: out of host memory", who);
}

}  // namespace

extern "C" {

int sr_orthogonalize_workspace(const sr_matrix* src, const sr_matrix* dst, int32_t count, const sr_newton_schulz* ns,
                               uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_orthogonalize_workspace: null argument");
  return orthogonalize("sr_orthogonalize_workspace", src, dst, count, ns, nullptr, 0, bytes, nullptr);
}

int sr_orthogonalize(const sr_matrix* src, const sr_matrix* dst, int32_t count, const sr_newton_schulz* ns, void* workspace,
                     uint64_t workspace_bytes, hipStream_t stream) {
  return orthogonalize("sr_orthogonalize", src, dst, count, ns, workspace, workspace_bytes, nullptr, stream);
}

int sr_muon_workspace(const sr_muon_tensor* tensors, int32_t count, const sr_muon_options* options, const sr_newton_schulz* ns,
                      uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_muon_workspace: null argument");
  return muon("sr_muon_workspace", tensors, count, options, ns, nullptr, 0, bytes, nullptr);
}

int sr_muon(const sr_muon_tensor* tensors, int32_t count, const sr_muon_options* options, const sr_newton_schulz* ns,
            void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return muon("sr_muon", tensors, count, options, ns, workspace, workspace_bytes, nullptr, stream);
}

}  // extern "C"
