// embed.hip -- rows of a vocabulary shard for given tokens, and the gradient
// of those rows (C ABI in include/suika_step.h).
//
// The lookup is a copy with a table of rows: HBM bounds it (16384 tokens of 4096
// bf16 columns, 186 MB with the rows they hit, 29.5 us, 6.3 TB/s).  Outputs are
// streamed, the table's rows are cached: frequent tokens read the same ones.
//
// The gradient of row r is the sum of the outputs' gradients at the tokens
// that are r.  Adding them with atomics would make the result depend on the
// order in which workgroups run, so the tokens are sorted first (a stable
// counting sort, one launch) and every row sums its own in that order:
//
//   sort    Workgroup b of B owns rows b, b + B, ... (frequent tokens are
//           neighbours in a vocabulary) and reads all tokens, which come from
//           the L2: it counts those of the workgroups before it, which is where
//           its own start in the sorted list, and those of each of its rows,
//           and places them in a second pass.  No workgroup waits for another.
//           Its time is a chain of loads, scans and barriers: 11.2 us for 16384
//           tokens, 18 for 30011; 28 where one row has 9800 of 16384, which is
//           one workgroup's.  (Ranges of neighbouring rows: 24 and 43 us, as
//           the range of the frequent tokens is one workgroup's.)
//   sum     A group of lanes per row adds up the row's tokens, each lane one or
//           two 16-byte column blocks.  A row of many tokens (a space, a filler)
//           is cut into pieces that are summed side by side, into 32-bit partial
//           sums.  A chain of tokens bounds it where rows have many, so eight
//           are loaded at once and the indices of the next eight beside them;
//           groups of whole waves keep the rows' addresses in scalar registers,
//           which leaves room for that at full occupancy.  Rows in the order of
//           memory, gradients read and written past the caches: 48.2 us for
//           256 MB (5.3 TB/s; four tokens at once and indices as they are
//           needed 51.8; with cached accesses 73; rows in the sort's order 78).
//   join    The partial sums of such rows, added in order: 6.7 us (30011
//           tokens of 3584 columns 7.9).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "suika_step.h"
#include "sr_step.h"

namespace {

using namespace sr_step;

constexpr int kThreads = 256;

// The lanes of one row: a group of a power of two, each of them taking every
// `lanes`-th 16-byte block of the row's columns, U blocks in all; the row's last
// block may be shorter.  A row of more blocks takes several groups.
struct Lanes {
  uint32_t blocks;      // column blocks of a row
  uint32_t log2;        // lanes of a group
  uint32_t slices;      // groups along a row
};

Lanes lanes_of(uint64_t cols, uint32_t per_block, uint32_t most, uint32_t each) {
  Lanes l;
  l.blocks = uint32_t((cols + per_block - 1) / per_block);
  l.log2 = 0;
  while ((1u << l.log2) * each < l.blocks && (1u << l.log2) < most) ++l.log2;
  l.slices = (l.blocks + (each << l.log2) - 1) / (each << l.log2);
  return l;
}

// The first column of this lane's blocks, and from one of them to the next.
template <int N, int U>
__device__ __forceinline__ uint32_t first_column(const Lanes& l) {
  return ((blockIdx.y * U << l.log2) + (threadIdx.x & ((1u << l.log2) - 1))) * N;
}

// --------------------------------------------------------------------- rows

constexpr int kLookupBlocks = 2;      // of a lane

template <typename T, typename I, int U>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const I* tokens, const T* weight, T* out, uint32_t n_tokens,
                                                             uint64_t rows, uint64_t cols, uint64_t stride,
                                                             uint64_t start, float scale, Lanes l) {
  constexpr int N = 16 / sizeof(T);
  const uint32_t i = (blockIdx.x << (8 - l.log2)) + (threadIdx.x >> l.log2);
  if (i >= n_tokens) return;
  const uint64_t row = uint64_t(int64_t(tokens[i])) - start;
  const uint64_t c = first_column<N, U>(l), step = uint64_t(N) << l.log2;
  const bool inside = row < rows;
  const T* src = weight + (inside ? row * stride : 0) + c;
  T* dst = out + uint64_t(i) * cols + c;
  const float by = inside ? scale : 0.0f;      // rows outside are zeros whatever the scale is
  float x[U][N] = {};
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (inside && c + u * step + N <= cols) load<T, N>(src + u * step, x[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t at = c + u * step;
    if (at + N <= cols) {
#pragma unroll
      for (int k = 0; k < N; ++k) x[u][k] *= by;
      store_stream<T, N>(dst + u * step, x[u]);
    } else {
      for (uint64_t k = at; k < cols; ++k) dst[k - c] = inside ? T(float(src[k - c]) * scale) : T(0.0f);
    }
  }
}

// --------------------------------------------------------------------- sort

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr uint32_t kSortRows = 512;       // most rows of one workgroup

// The order in which rows are sorted: by the workgroup that owns them.
struct Owners {
  uint32_t log2;     // of the number of workgroups
  uint32_t range;    // rows of each
};

// One workgroup a compute unit, or more where that many rows have no room.
Owners owners_of(uint64_t rows) {
  Owners o{8, 0};
  while ((rows + (1u << o.log2) - 1) >> o.log2 > kSortRows) ++o.log2;
  o.range = uint32_t((rows + (1u << o.log2) - 1) >> o.log2);
  return o;
}

// A piece of a row's tokens: sorted positions from..to.  The pieces of a row
// follow one another; the first says how many they are.
struct alignas(16) Piece {
  uint32_t row;      // kNoPiece: none
  uint32_t from, to;
  uint32_t pieces;
};
constexpr uint32_t kNoPiece = 0xffffffffu;

// The tokens of a piece of a row of n: `least` or, of long rows, as many as the
// row then has pieces, so that adding up a piece and joining them take the same
// number of steps (16384 tokens of 4096 bf16 columns: sort and join 11.2 and
// 6.7 us, with `least` for all 12.6 and 9.2).
__device__ __forceinline__ uint32_t piece_of(uint32_t n, uint32_t least) {
  return max(least, (uint32_t(sqrtf(float(n))) + 3) / 4 * 4);
}

// The sorted positions of a row's tokens, and the first two tokens: most rows
// have no more, and these are one load less away.
struct alignas(16) Run {
  uint32_t from, to;
  uint32_t token[2];
};

// What the launches hand on, in the workspace.
struct Sorted {
  Run* run;           // [rows]
  uint32_t* tokens;   // [1] how many lie in the shard
  uint32_t* order;    // [tokens] sorted position -> index of the token
  Piece* piece;       // [slots]
  float* partial;     // [slots][cols]
};

// The lanes whose tokens are of the same row as this lane's: of those in `in`,
// the ones that agree in all `bits` bits of it.
__device__ __forceinline__ uint64_t same_row(uint64_t in, uint32_t row, uint32_t bits) {
  uint64_t same = in;
  for (uint32_t b = 0; b < bits; ++b) {
    const bool set = row >> b & 1;
    const uint64_t ones = __ballot(set);
    same &= set ? ones : ~ones;
  }
  return same;
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {   // inclusive
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t y = __shfl_up(x, d);
    if (int(threadIdx.x % kWave) >= d) x += y;
  }
  return x;
}

// Exclusive prefix sum over the workgroup; *total gets the sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* part, uint32_t* total) {
  const uint32_t inclusive = wave_scan(x);
  __syncthreads();
  if (threadIdx.x % kWave == kWave - 1) part[threadIdx.x / kWave] = inclusive;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    before += w < int(threadIdx.x / kWave) ? part[w] : 0;
    all += part[w];
  }
  *total = all;
  return before + inclusive - x;
}

// Tokens that a lane reads at once.
constexpr uint32_t kSortAhead = 8;
// Tokens of its own that a wave remembers between the passes; a wave that finds
// more reads its run again.
constexpr uint32_t kSortKept = 448;
constexpr uint32_t kOutside = 0xffffffffu;

// A token's row of the shard, kOutside for those of other shards.
template <typename I>
__device__ __forceinline__ uint32_t row_of(I token, uint64_t start, uint32_t rows) {
  const uint64_t row = uint64_t(int64_t(token)) - start;
  return row < rows ? uint32_t(row) : kOutside;
}

// f(index, row) for a wave's tokens from..to, 64 at a time in their order; every
// lane calls it, with kOutside where there is no token.
template <typename I, typename F>
__device__ __forceinline__ void for_tokens(const I* tokens, uint32_t from, uint32_t to, uint64_t start, uint32_t rows,
                                           F&& f) {
  uint32_t i = from + threadIdx.x % kWave;
  for (; from + kSortAhead * kWave <= to; from += kSortAhead * kWave) {
    I t[kSortAhead];
#pragma unroll
    for (uint32_t a = 0; a < kSortAhead; ++a) t[a] = tokens[i + a * kWave];
#pragma unroll
    for (uint32_t a = 0; a < kSortAhead; ++a) f(i + a * kWave, row_of(t[a], start, rows));
    i += kSortAhead * kWave;
  }
  for (; from < to; from += kWave, i += kWave) f(i, i < to ? row_of(tokens[i], start, rows) : kOutside);
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_kernel(const I* tokens, uint32_t n_tokens, uint32_t rows,
                                                            uint64_t start, Owners owners, uint32_t bits,
                                                            uint32_t piece, Sorted out) {
  __shared__ uint32_t count[kSortWaves * kSortRows];
  __shared__ uint32_t part[kSortWaves], start_of[kSortRows];
  __shared__ uint32_t kept[kSortWaves][kSortKept], kept_row[kSortWaves][kSortKept];
  const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const uint32_t me = blockIdx.x, range = owners.range, mask = (1u << owners.log2) - 1;
  for (uint32_t i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) count[i] = 0;
  __syncthreads();

  // Every wave takes a run of the tokens, so waves and lanes are in their order.
  const uint32_t run = (n_tokens + kSortThreads - 1) / kSortThreads * kWave;
  const uint32_t from = min(wave * run, n_tokens), to = min(from + run, n_tokens);
  uint32_t* mine = count + wave * range;
  uint32_t lower = 0, found = 0;
  for_tokens(tokens, from, to, start, rows, [&](uint32_t i, uint32_t r) {
    const uint32_t owner = r & mask;
    lower += r != kOutside && owner < me;
    const bool own = r != kOutside && owner == me;
    const uint64_t any = __ballot(own);
    if (any == 0) return;
    if (own) {
      atomicAdd(mine + (r >> owners.log2), 1u);
      const uint32_t k = found + uint32_t(__popcll(any & below));
      if (k < kSortKept) {
        kept[wave][k] = i;
        kept_row[wave][k] = r >> owners.log2;
      }
    }
    found += uint32_t(__popcll(any));
  });
  uint32_t base = 0, total = 0, pieces = 0;
  block_scan(lower, part, &base);      // the sum: where this workgroup's rows start

  // Thread q: the tokens of row q of this workgroup, and where each wave puts its part of them.
  uint32_t n = 0;
  if (threadIdx.x < range)
    for (int w = 0; w < kSortWaves; ++w) n += count[w * range + threadIdx.x];
  const uint32_t at = base + block_scan(n, part, &total);
  const uint32_t each = piece_of(n, piece);
  const uint32_t cut = n > 2 * piece ? (n + each - 1) / each : 0;
  const uint32_t slot = block_scan(cut, part, &pieces);
  if (threadIdx.x < range) {
    uint32_t next = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = count[w * range + threadIdx.x];
      count[w * range + threadIdx.x] = next;
      next += c;
    }
    const uint32_t row = (threadIdx.x << owners.log2) + me;
    start_of[threadIdx.x] = at;
    if (row < rows) {
      out.run[row].from = at;
      out.run[row].to = at + n;
    }
    if (me == mask && threadIdx.x == 0) *out.tokens = base + total;
  }
  // A workgroup of `total` tokens has the slots from 2 base / piece on.  A row is
  // cut where it has more than 2 piece tokens, into pieces of `piece` or more: at
  // most 3/2 of n / piece, so they fit; the slots left over say that they are empty.
  const uint32_t slot0 = uint32_t(2 * uint64_t(base) / piece);
  const uint32_t slot1 = uint32_t(2 * uint64_t(base + total) / piece);
  for (uint32_t k = 0; k < cut; ++k)
    out.piece[slot0 + slot + k] = {(threadIdx.x << owners.log2) + me, at + k * each, min(at + (k + 1) * each, at + n),
                                   k ? 0 : cut};
  for (uint32_t s = slot0 + pieces + threadIdx.x; s < slot1; s += kSortThreads) out.piece[s] = {kNoPiece, 0, 0, 0};
  __syncthreads();

  // Lanes of one row take consecutive places, in their order, from where the row's last ones ended.
  auto put = [&](uint32_t i, uint32_t local, bool own) {
    const uint64_t any = __ballot(own);
    if (any == 0) return;
    const uint64_t same = same_row(any, local, bits);
    const int leader = __ffsll((unsigned long long)same) - 1;
    uint32_t next = 0;
    if (own && int(lane) == leader) next = atomicAdd(mine + local, uint32_t(__popcll(same)));
    next = __shfl(next, leader & (kWave - 1));
    if (own) {
      const uint32_t p = next + uint32_t(__popcll(same & below)), nth = p - start_of[local];
      out.order[p] = i;
      if (nth < 2) out.run[(local << owners.log2) + me].token[nth] = i;
    }
  };
  if (found <= kSortKept) {
    for (uint32_t k = lane; k - lane < found; k += kWave) {
      const bool own = k < found;
      put(own ? kept[wave][k] : 0, own ? kept_row[wave][k] : 0, own);
    }
  } else {
    for_tokens(tokens, from, to, start, rows, [&](uint32_t i, uint32_t r) {
      put(i, r >> owners.log2, r != kOutside && (r & mask) == me);
    });
  }
}

// ---------------------------------------------------------------------- sum

// Where a lane loads the block of columns from c on: a row's last, shorter block
// from N columns before its end, so that it is a vector as the others.
template <int N>
__device__ __forceinline__ uint32_t block_at(uint32_t c, uint32_t cols) {
  return c + N <= cols || cols < N ? c : cols - N;
}

// A lane group's place in a grid of groups.  Where a group is whole waves
// (kWhole), it is known to be the same in all lanes, and with it what is read
// there: the addresses of rows need no vector registers.
template <bool kWhole>
__device__ __forceinline__ uint32_t task_of(const Lanes& l) {
  const uint32_t group = threadIdx.x >> l.log2;
  return (blockIdx.x << (8 - l.log2)) + (kWhole ? __builtin_amdgcn_readfirstlane(group) : group);
}

// What the launches before have written.
template <bool kWhole, typename V>
__device__ __forceinline__ V written(const V* p) {
  typedef uint32_t Words __attribute__((ext_vector_type(sizeof(V) / 4)));
  typedef const __attribute__((address_space(4))) Words* Constant;
  if constexpr (kWhole) return __builtin_bit_cast(V, *(Constant)(uintptr_t)p);
  else return *p;
}

// Adds columns c.. of the tokens at sorted positions from..to to `acc`, in
// their order; N of them, or `cols - c` of a row that has no N columns.
constexpr uint32_t kAhead = 8;        // tokens that a lane loads at once

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void sum_tokens(const T* grad_out, uint64_t stride, const uint32_t* order, uint32_t from,
                                           uint32_t to, uint32_t c, uint32_t cols, float (&acc)[N]) {
  typedef const Vec<T, N>* Vector;
  if (c + N <= cols) {
    uint32_t token[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) token[a] = from + a < to ? written<kWhole>(order + from + a) : 0;
    uint32_t i = from;
    for (; i + kAhead <= to; i += kAhead) {
      Vec<T, N> x[kAhead];
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
        x[a] = __builtin_nontemporal_load(Vector(grad_out + token[a] * stride + c));
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
        token[a] = i + kAhead + a < to ? written<kWhole>(order + i + kAhead + a) : 0;
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += float(x[a][k]);
    }
    if (i < to) {
      Vec<T, N> x[kAhead];
#pragma unroll
      for (uint32_t a = 0; a < kAhead - 1; ++a)
        if (i + a < to) x[a] = __builtin_nontemporal_load(Vector(grad_out + token[a] * stride + c));
#pragma unroll
      for (uint32_t a = 0; a < kAhead - 1; ++a)
        if (i + a < to)
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += float(x[a][k]);
    }
  } else {
    for (uint32_t i = from; i < to; ++i) {
      const T* p = grad_out + written<kWhole>(order + i) * stride + c;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (c + k < cols) acc[k] += float(p[k]);
    }
  }
}

// grad[c..] = scale * acc, plus what is there; acc holds the columns from `at`
// = block_at(c) on.  Blocks of more than 16 bytes take two stores that each leave
// gaps, for the L2 to merge: streamed, 50304 rows of 768 f32 took 56 us, not 39.
template <typename G, int N>
__device__ __forceinline__ void put_row(G* grad, uint32_t c, uint32_t at, uint32_t cols, float scale, bool accumulate,
                                        float (&acc)[N]) {
  if (c + N <= cols) {
    float old[N] = {};
    if (accumulate) load<G, N>(grad + c, old);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = fmaf(acc[k], scale, old[k]);
    if constexpr (N * sizeof(G) > 16) store<G, N>(grad + c, acc);
    else store_stream<G, N>(grad + c, acc);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (at + k >= c && at + k < cols)
        grad[at + k] = G(fmaf(acc[k], scale, accumulate ? float(grad[at + k]) : 0.0f));
  }
}

// Tasks 0..slots * U are the pieces, each of a lane's U blocks apart: they are the
// longest; the rows follow.
template <typename T, typename G, int U, bool kWhole>
__global__ __launch_bounds__(kThreads) void sum_kernel(const T* grad_out, uint64_t stride, G* grad, uint32_t rows,
                                                       uint32_t cols, uint32_t slots, uint32_t piece, float scale,
                                                       bool accumulate, Lanes l, Sorted in) {
  constexpr int N = 16 / sizeof(T);
  typedef const Vec<T, N>* Vector;
  const uint32_t task = task_of<kWhole>(l);
  const uint32_t c = first_column<N, U>(l), step = uint32_t(N) << l.log2;
  if (task < slots * U) {
    const uint32_t slot = task / U;
    const Piece p = written<kWhole>(in.piece + slot);
    if (slot >= uint32_t(2 * uint64_t(*in.tokens) / piece) || p.row == kNoPiece) return;
    const uint32_t own = c + task % U * step, at = block_at<N>(own, cols);
    if (own >= cols) return;
    float acc[N] = {};
    sum_tokens<kWhole, T, N>(grad_out, stride, in.order, p.from, p.to, at, cols, acc);
    put_row<float, N>(in.partial + uint64_t(slot) * cols, own, at, cols, 1.0f, false, acc);
    return;
  }
  const uint32_t row = task - slots * U;
  if (row >= rows || c >= cols) return;
  const Run run = written<kWhole>(in.run + row);
  const uint32_t n = run.to - run.from;
  if (n > 2 * piece || (accumulate && n == 0)) return;
  Vec<T, N> x[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (uint32_t a = 0; a < 2; ++a)
      if (a < n && c + u * step < cols && N <= cols)
        x[u][a] = __builtin_nontemporal_load(Vector(grad_out + run.token[a] * stride + block_at<N>(c + u * step, cols)));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t own = c + u * step, at = block_at<N>(own, cols);
    if (own >= cols) break;
    float acc[N] = {};
    uint32_t from = run.from;
    if (N <= cols) {
#pragma unroll
      for (uint32_t a = 0; a < 2; ++a)
        if (a < n)
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += float(x[u][a][k]);
      from += n < 2 ? n : 2;
    }
    sum_tokens<kWhole, T, N>(grad_out, stride, in.order, from, run.to, at, cols, acc);
    // a row without tokens is zeros whatever the scale is
    put_row<G, N>(grad + uint64_t(row) * cols, own, at, cols, n ? scale : 0.0f, accumulate, acc);
  }
}

template <typename G>
__global__ __launch_bounds__(kThreads) void join_kernel(G* grad, uint32_t cols, uint32_t slots, uint32_t piece,
                                                        float scale, bool accumulate, Lanes l, Sorted in) {
  constexpr int N = 4;
  constexpr uint32_t kAhead = 8;
  const uint32_t task = (blockIdx.x << (8 - l.log2)) + (threadIdx.x >> l.log2);
  if (task >= slots || task >= uint32_t(2 * uint64_t(*in.tokens) / piece)) return;
  const Piece p = in.piece[task];
  const uint32_t pieces = p.pieces;
  if (p.row == kNoPiece || pieces == 0) return;
  const uint32_t c = first_column<N, 1>(l), at = block_at<N>(c, cols);
  if (c >= cols) return;
  float acc[N] = {};
  const float* src = in.partial + uint64_t(task) * cols + at;
  uint32_t i = 0;
  if (N <= cols) {
    for (; i + kAhead <= pieces; i += kAhead) {
      float x[kAhead][N];
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) load<float, N>(src + uint64_t(i + a) * cols, x[a]);
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += x[a][k];
    }
    for (; i < pieces; ++i) {
      float x[N];
      load<float, N>(src + uint64_t(i) * cols, x);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += x[k];
    }
  } else {
    for (; i < pieces; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (at + k < cols) acc[k] += src[uint64_t(i) * cols + k];
  }
  put_row<G, N>(grad + uint64_t(p.row) * cols, c, at, cols, scale, accumulate, acc);
}

// ---------------------------------------------------------------------- host

bool aligned(const void* p, int32_t dt) { return reinterpret_cast<uintptr_t>(p) % sr_internal::dtype_size(dt) == 0; }

int check_shape(const char* who, const sr_embedding_shape* s) {
  if (s == nullptr) return fail(SR_EINVAL, "%s: null argument", who);
  if (s->reserved != 0) return fail(SR_EINVAL, "%s: shape.reserved is not 0", who);
  if (s->token_dtype != SR_DT_I32 && s->token_dtype != SR_DT_I64)
    return fail(SR_EDTYPE, "%s: tokens of dtype %d", who, s->token_dtype);
  if (!float_dtype(s->dtype)) return fail(SR_EDTYPE, "%s: dtype %d", who, s->dtype);
  if (s->n_tokens > SR_STEP_MAX_ROWS || s->rows > SR_STEP_MAX_ROWS || s->cols > SR_STEP_MAX_ROWS)
    return fail(SR_EBOUNDS, "%s: %llu tokens, %llu rows, %llu columns", who, (unsigned long long)s->n_tokens,
                (unsigned long long)s->rows, (unsigned long long)s->cols);
  // a negative start would make rows of negative tokens, which lie outside of every shard
  if (s->vocab_start < 0) return fail(SR_EINVAL, "%s: vocab_start %lld", who, (long long)s->vocab_start);
  if (s->n_tokens && s->tokens == nullptr) return fail(SR_EINVAL, "%s: tokens is null", who);
  if (!aligned(s->tokens, s->token_dtype)) return fail(SR_EALIGN, "%s: tokens not aligned", who);
  return SR_OK;
}

Extent tokens_of(const sr_embedding_shape& s) {
  return {s.tokens, s.n_tokens * sr_internal::dtype_size(s.token_dtype)};
}

// Bytes from the first element of a matrix to behind its last.
uint64_t extent(uint64_t rows, uint64_t cols, uint64_t stride, int32_t dt) {
  return rows && cols ? ((rows - 1) * stride + cols) * sr_internal::dtype_size(dt) : 0;
}

template <typename T, typename I, int U>
void launch_embedding_of(const sr_embedding_shape& s, const void* weight, uint64_t stride, void* out,
                         hipStream_t stream) {
  const Lanes l = lanes_of(s.cols, 16 / sizeof(T), kThreads, U);
  const uint32_t group = uint32_t(kThreads) >> l.log2;
  const dim3 grid(uint32_t((s.n_tokens + group - 1) / group), l.slices);
  embedding_kernel<T, I, U><<<grid, kThreads, 0, stream>>>(
      static_cast<const I*>(s.tokens), static_cast<const T*>(weight), static_cast<T*>(out), uint32_t(s.n_tokens),
      s.rows, s.cols, stride, uint64_t(s.vocab_start), s.scale, l);
}

template <typename T>
void launch_embedding(const sr_embedding_shape& s, const void* weight, uint64_t stride, void* out, hipStream_t stream) {
  if (s.token_dtype == SR_DT_I64) launch_embedding_of<T, int64_t, kLookupBlocks>(s, weight, stride, out, stream);
  else launch_embedding_of<T, int32_t, kLookupBlocks>(s, weight, stride, out, stream);
}

// The parts of the workspace.  Pieces grow with the number of tokens, so that
// a row of all tokens is joined from 1024 pieces at most.
struct Layout {
  uint32_t piece, slots;
  uint64_t count, order, pieces, partial, bytes;
};

Layout layout_of(const sr_embedding_shape& s) {
  Layout w;
  w.piece = 16;
  while (s.n_tokens / w.piece > 1024) w.piece *= 2;
  w.slots = uint32_t(2 * s.n_tokens / w.piece);
  auto up = [](uint64_t b) { return (b + 255) / 256 * 256; };
  w.count = up(s.rows * sizeof(Run));
  w.order = w.count + 256;
  w.pieces = w.order + up(s.n_tokens * 4);
  w.partial = w.pieces + up(uint64_t(w.slots) * sizeof(Piece));
  w.bytes = w.partial + uint64_t(w.slots) * s.cols * 4;
  return w;
}

// A lane takes one block of columns, or two where a row has more of them than a
// workgroup has lanes: 30011 tokens of 3584 bf16 columns 136 us with two, 141
// with one (of two workgroups a row), but 65536 tokens of 1984 columns 151 and
// 141, and 4096 tokens of 768 f32 columns 31 and 28.
template <typename T, typename G>
void launch_sum(const sr_embedding_shape& s, const Layout& w, const Sorted& sorted, const void* grad_out,
                uint64_t stride, void* grad, bool accumulate, hipStream_t stream) {
  constexpr uint32_t N = 16 / sizeof(T);
  const int each = s.cols > uint64_t(N) * kThreads ? 2 : 1;
  const Lanes l = lanes_of(s.cols, N, kThreads, each);
  const uint32_t group = uint32_t(kThreads) >> l.log2;
  const dim3 grid(uint32_t((uint64_t(w.slots) * each + s.rows + group - 1) / group), l.slices);
  auto* kernel = each == 2     ? sum_kernel<T, G, 2, true>
                 : l.log2 >= 6 ? sum_kernel<T, G, 1, true>
                               : sum_kernel<T, G, 1, false>;
  kernel<<<grid, kThreads, 0, stream>>>(static_cast<const T*>(grad_out), stride, static_cast<G*>(grad),
                                        uint32_t(s.rows), uint32_t(s.cols), w.slots, w.piece, s.scale, accumulate, l,
                                        sorted);
  if (s.n_tokens <= 2 * w.piece) return;     // no row is cut
  const Lanes j = lanes_of(s.cols, 4, kThreads, 1);
  const uint32_t joined = uint32_t(kThreads) >> j.log2;
  const dim3 join_grid((w.slots + joined - 1) / joined, j.slices);
  join_kernel<G><<<join_grid, kThreads, 0, stream>>>(static_cast<G*>(grad), uint32_t(s.cols), w.slots, w.piece, s.scale,
                                                     accumulate, j, sorted);
}

template <typename T>
void launch_sum_to(int32_t grad_dtype, const sr_embedding_shape& s, const Layout& w, const Sorted& sorted,
                   const void* grad_out, uint64_t stride, void* grad, bool accumulate, hipStream_t stream) {
  if (grad_dtype == SR_DT_F32) launch_sum<T, float>(s, w, sorted, grad_out, stride, grad, accumulate, stream);
  else if (grad_dtype == SR_DT_BF16) launch_sum<T, bf16>(s, w, sorted, grad_out, stride, grad, accumulate, stream);
  else launch_sum<T, f16>(s, w, sorted, grad_out, stride, grad, accumulate, stream);
}

}  // namespace

extern "C" {

int sr_embedding(const sr_embedding_shape* shape, const void* weight, uint64_t weight_stride, void* out,
                 hipStream_t stream) {
  if (int rc = check_shape("sr_embedding", shape)) return rc;
  const sr_embedding_shape& s = *shape;
  if (s.n_tokens == 0 || s.cols == 0) return SR_OK;
  if (out == nullptr || (s.rows && weight == nullptr)) return fail(SR_EINVAL, "sr_embedding: null argument");
  if (weight_stride < s.cols || weight_stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "sr_embedding: rows %llu apart for %llu columns", (unsigned long long)weight_stride,
                (unsigned long long)s.cols);
  if (!aligned(weight, s.dtype) || !aligned(out, s.dtype)) return fail(SR_EALIGN, "sr_embedding: not aligned to the elements");
  const Extent to{out, extent(s.n_tokens, s.cols, s.cols, s.dtype)};
  if (to.meets({weight, extent(s.rows, s.cols, weight_stride, s.dtype)}) || to.meets(tokens_of(s)))
    return fail(SR_EOVERLAP, "sr_embedding: the output overlaps an input");
  if (s.dtype == SR_DT_F32) launch_embedding<float>(s, weight, weight_stride, out, stream);
  else if (s.dtype == SR_DT_BF16) launch_embedding<bf16>(s, weight, weight_stride, out, stream);
  else launch_embedding<f16>(s, weight, weight_stride, out, stream);
  return launched("sr_embedding");
}

int sr_embedding_grad_workspace(const sr_embedding_shape* shape, uint64_t* bytes) {
  if (bytes == nullptr) return fail(SR_EINVAL, "sr_embedding_grad_workspace: null argument");
  if (int rc = check_shape("sr_embedding_grad_workspace", shape)) return rc;
  *bytes = layout_of(*shape).bytes;
  return SR_OK;
}

int sr_embedding_grad(const sr_embedding_shape* shape, const void* grad_out, uint64_t grad_out_stride, void* grad,
                      int32_t grad_dtype, int32_t accumulate, void* workspace, uint64_t workspace_bytes,
                      hipStream_t stream) {
  if (int rc = check_shape("sr_embedding_grad", shape)) return rc;
  const sr_embedding_shape& s = *shape;
  if (!float_dtype(grad_dtype)) return fail(SR_EDTYPE, "sr_embedding_grad: gradient of dtype %d", grad_dtype);
  if (s.rows == 0 || s.cols == 0) return SR_OK;
  if (grad == nullptr || (s.n_tokens && grad_out == nullptr)) return fail(SR_EINVAL, "sr_embedding_grad: null argument");
  if (grad_out_stride < s.cols || grad_out_stride > SR_STEP_MAX_ELEMENTS)
    return fail(SR_EINVAL, "sr_embedding_grad: rows %llu apart for %llu columns", (unsigned long long)grad_out_stride,
                (unsigned long long)s.cols);
  if (!aligned(grad, grad_dtype) || !aligned(grad_out, s.dtype))
    return fail(SR_EALIGN, "sr_embedding_grad: not aligned to the elements");
  const Layout w = layout_of(s);
  if (workspace == nullptr || workspace_bytes < w.bytes)
    return fail(SR_EINVAL, "sr_embedding_grad: a workspace of %llu bytes, %llu are needed",
                (unsigned long long)workspace_bytes, (unsigned long long)w.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(SR_EALIGN, "sr_embedding_grad: workspace not aligned");
  const Extent to{grad, extent(s.rows, s.cols, s.cols, grad_dtype)}, work{workspace, w.bytes};
  const Extent from{grad_out, extent(s.n_tokens, s.cols, grad_out_stride, s.dtype)};
  if (to.meets(from) || to.meets(tokens_of(s)) || to.meets(work) || work.meets(from) || work.meets(tokens_of(s)))
    return fail(SR_EOVERLAP, "sr_embedding_grad: the gradient or the workspace overlaps an input");
  char* base = static_cast<char*>(workspace);
  const Sorted sorted{reinterpret_cast<Run*>(base), reinterpret_cast<uint32_t*>(base + w.count),
                      reinterpret_cast<uint32_t*>(base + w.order),
                      reinterpret_cast<Piece*>(base + w.pieces), reinterpret_cast<float*>(base + w.partial)};
  const Owners owners = owners_of(s.rows);
  uint32_t bits = 0;
  while ((1u << bits) < owners.range) ++bits;
  auto sort = [&](auto* tokens) {
    sort_kernel<<<1u << owners.log2, kSortThreads, 0, stream>>>(tokens, uint32_t(s.n_tokens), uint32_t(s.rows),
                                                                uint64_t(s.vocab_start), owners, bits, w.piece, sorted);
  };
  if (s.token_dtype == SR_DT_I64) sort(static_cast<const int64_t*>(s.tokens));
  else sort(static_cast<const int32_t*>(s.tokens));
  if (int rc = launched("sr_embedding_grad: sort")) return rc;
  if (s.dtype == SR_DT_F32) launch_sum_to<float>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  else if (s.dtype == SR_DT_BF16) launch_sum_to<bf16>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  else launch_sum_to<f16>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  return launched("sr_embedding_grad");
}

}  // extern "C"
