// embed.hip -- rows of a vocabulary shard for given tokens, and the gradient
// of those rows (C ABI in include/suika_step.h).
//
// The gradient of row r is the sum of the outputs' gradients at the tokens
// that are r.  Adding them with atomics would make the result depend on the
// order in which workgroups run, so the tokens are sorted first (a stable
// counting sort, one launch) and every row sums its own in that order:
//
//   sort    Workgroup b owns a range of rows and reads all tokens, which come
//           from the L2: it counts those of lower rows, which is where its
//           own start in the sorted list, and those of each of its rows, and
//           places them in a second pass.  No workgroup waits for another.
//   sum     A group of lanes per row adds up the row's tokens, each lane one
//           16-byte column block.  A row of many tokens (a space, a filler) is
//           cut into pieces that are summed side by side, into 32-bit partial
//           sums.
//   join    The partial sums of such rows, added in order.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "suika_step.h"
#include "sr_step.h"

namespace {

using namespace sr_step;

constexpr int kThreads = 256;

// Lanes of one row: each takes a 16-byte block of columns, the last one what
// is left of a row.  Groups of a power of two lanes share a workgroup; rows of
// more blocks than lanes take several workgroups.
struct Lanes {
  uint32_t blocks;      // column blocks of a row
  uint32_t log2;        // lanes of a group
  uint32_t slices;      // groups along a row
};

Lanes lanes_of(uint64_t cols, uint32_t per_block) {
  Lanes l;
  l.blocks = uint32_t((cols + per_block - 1) / per_block);
  l.log2 = 0;
  while ((1u << l.log2) < l.blocks && (1u << l.log2) < kThreads) ++l.log2;
  l.slices = (l.blocks + kThreads - 1) / kThreads;
  return l;
}

// --------------------------------------------------------------------- rows

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const I* tokens, const T* weight, T* out, uint32_t n_tokens,
                                                             uint64_t rows, uint64_t cols, uint64_t stride,
                                                             int64_t start, float scale, Lanes l) {
  constexpr int N = 16 / sizeof(T);
  const uint32_t i = (blockIdx.x << (8 - l.log2)) + (threadIdx.x >> l.log2);
  const uint32_t block = blockIdx.y * kThreads + (threadIdx.x & ((1u << l.log2) - 1));
  if (i >= n_tokens || block >= l.blocks) return;
  const int64_t row = int64_t(tokens[i]) - start;
  const uint64_t c = uint64_t(block) * N;
  const bool inside = row >= 0 && uint64_t(row) < rows;
  const T* src = weight + (inside ? uint64_t(row) * stride : 0) + c;
  T* dst = out + uint64_t(i) * cols + c;
  if (c + N <= cols) {
    float x[N] = {};
    if (inside) load<T, N>(src, x);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] *= scale;
    store<T, N>(dst, x);
  } else {
    for (uint64_t k = 0; c + k < cols; ++k) dst[k] = inside ? T(float(src[k]) * scale) : T(0.0f);
  }
}

// --------------------------------------------------------------------- sort

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr uint32_t kSortRanges = 256;     // workgroups, one a compute unit
constexpr uint32_t kSortRows = 512;       // most rows of one range

// A piece of a row's tokens: sorted positions from..to, the k-th of its row.
struct alignas(16) Piece {
  uint32_t row;      // kNoPiece: none
  uint32_t from, to;
  uint32_t k;
};
constexpr uint32_t kNoPiece = 0xffffffffu;

// What the launches hand on, in the workspace.
struct Sorted {
  uint32_t* offset;   // [rows + 1] first sorted position of each row's tokens
  uint32_t* order;    // [tokens] sorted position -> index of the token
  Piece* piece;       // [slots]
  float* partial;     // [slots][cols]
};

// The lanes whose tokens are of one row are taken together: f(row, which lanes,
// the lowest of them, this lane's place among them), row after row.
template <typename F>
__device__ __forceinline__ void by_row(bool in, uint32_t row, F&& f) {
  uint64_t left = __ballot(in);
  const uint64_t below = (uint64_t(1) << (threadIdx.x % kWave)) - 1;
  while (left) {
    const int leader = __ffsll((unsigned long long)left) - 1;
    const uint32_t r = __builtin_amdgcn_readlane(row, leader);
    const uint64_t same = __ballot(in && row == r);
    f(r, same, leader, uint32_t(__popcll(same & below)));
    left &= ~same;
  }
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

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_kernel(const I* tokens, uint32_t n_tokens, uint64_t rows,
                                                            int64_t start, uint32_t range, uint32_t piece,
                                                            Sorted out) {
  __shared__ uint32_t count[kSortWaves * kSortRows];
  __shared__ uint32_t part[kSortWaves];
  const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const uint64_t first = uint64_t(blockIdx.x) * range;
  const uint32_t own = uint32_t(rows - first < range ? rows - first : range);
  for (uint32_t i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) count[i] = 0;
  __syncthreads();

  // Every wave takes a run of the tokens, so waves and lanes are in their order.
  const uint32_t run = (n_tokens + kSortThreads - 1) / kSortThreads * kWave;
  const uint32_t from = wave * run;
  const uint32_t to = from < n_tokens ? (n_tokens - from < run ? n_tokens : from + run) : from;
  uint32_t* mine = count + wave * range;
  uint32_t lower = 0;
  for (uint32_t i = from + lane; i - lane < to; i += kWave) {
    const int64_t r = i < to ? int64_t(tokens[i]) - start : -1;
    const bool here = r >= 0 && uint64_t(r) < rows;
    lower += here && uint64_t(r) < first;
    const uint64_t local = uint64_t(r) - first;
    by_row(here && uint64_t(r) >= first && local < own, uint32_t(local),
           [&](uint32_t row, uint64_t same, int leader, uint32_t) {
             if (int(lane) == leader) atomicAdd(mine + row, uint32_t(__popcll(same)));
           });
  }
  uint32_t base = 0, total = 0, pieces = 0;
  block_scan(lower, part, &base);      // the sum: where this range starts

  // Thread r: the tokens of row r, and where each wave puts its part of them.
  uint32_t n = 0;
  if (threadIdx.x < own)
    for (int w = 0; w < kSortWaves; ++w) n += count[w * range + threadIdx.x];
  const uint32_t at = base + block_scan(n, part, &total);
  const uint32_t cut = n > 2 * piece ? (n + piece - 1) / piece : 0;
  const uint32_t slot = block_scan(cut, part, &pieces);
  if (threadIdx.x < own) {
    uint32_t next = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = count[w * range + threadIdx.x];
      count[w * range + threadIdx.x] = next;
      next += c;
    }
    out.offset[first + threadIdx.x] = at;
    if (first + threadIdx.x == rows - 1) out.offset[rows] = base + total;
  }
  // A range of `total` tokens has the slots from 2 base / piece on.  A row is
  // cut where it has more than 2 piece tokens, into at most 3/2 of n / piece
  // pieces, so they fit; the slots left over say that they are empty.
  const uint32_t slot0 = uint32_t(2 * uint64_t(base) / piece);
  const uint32_t slot1 = uint32_t(2 * uint64_t(base + total) / piece);
  for (uint32_t k = 0; k < cut; ++k)
    out.piece[slot0 + slot + k] = {uint32_t(first + threadIdx.x), at + k * piece, min(at + (k + 1) * piece, at + n), k};
  for (uint32_t s = slot0 + pieces + threadIdx.x; s < slot1; s += kSortThreads) out.piece[s] = {kNoPiece, 0, 0, 0};
  __syncthreads();

  for (uint32_t i = from + lane; i - lane < to; i += kWave) {
    const int64_t r = i < to ? int64_t(tokens[i]) - start : -1;
    const uint64_t local = uint64_t(r) - first;
    const bool in = r >= 0 && uint64_t(r) >= first && local < own;
    by_row(in, uint32_t(local), [&](uint32_t row, uint64_t same, int leader, uint32_t place) {
      uint32_t next = 0;
      if (int(lane) == leader) next = atomicAdd(mine + row, uint32_t(__popcll(same)));
      next = __builtin_amdgcn_readlane(next, leader);
      if (in && uint32_t(local) == row) out.order[next + place] = i;
    });
  }
}

// ---------------------------------------------------------------------- sum

// Adds columns c.. of the tokens at sorted positions from..to to `acc`, in
// their order; N of them, or `cols - c` at a row's end.
template <typename T, int N>
__device__ __forceinline__ void sum_tokens(const T* grad_out, uint64_t stride, const uint32_t* order, uint32_t from,
                                           uint32_t to, uint64_t c, uint64_t cols, float (&acc)[N]) {
  constexpr uint32_t kAhead = 4;
  if (c + N <= cols) {
    uint32_t i = from;
    for (; i + kAhead <= to; i += kAhead) {
      float x[kAhead][N];
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) load<T, N>(grad_out + order[i + a] * stride + c, x[a]);
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += x[a][k];
    }
    for (; i < to; ++i) {
      float x[N];
      load<T, N>(grad_out + order[i] * stride + c, x);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += x[k];
    }
  } else {
    for (uint32_t i = from; i < to; ++i) {
      const T* p = grad_out + order[i] * stride + c;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (c + k < cols) acc[k] += float(p[k]);
    }
  }
}

// grad[c..] = scale * acc, plus what is there.
template <typename G, int N>
__device__ __forceinline__ void put_row(G* grad, uint64_t c, uint64_t cols, float scale, bool accumulate,
                                        float (&acc)[N]) {
  if (c + N <= cols) {
    float old[N] = {};
    if (accumulate) load<G, N>(grad + c, old);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = fmaf(acc[k], scale, old[k]);
    store<G, N>(grad + c, acc);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (c + k < cols) grad[c + k] = G(fmaf(acc[k], scale, accumulate ? float(grad[c + k]) : 0.0f));
  }
}

// Tasks 0..slots are the pieces, the rows follow.
template <typename T, typename G>
__global__ __launch_bounds__(kThreads) void sum_kernel(const T* grad_out, uint64_t stride, G* grad, uint64_t rows,
                                                       uint64_t cols, uint32_t slots, uint32_t piece, float scale,
                                                       bool accumulate, Lanes l, Sorted in) {
  constexpr int N = 16 / sizeof(T);
  const uint64_t task = (uint64_t(blockIdx.x) << (8 - l.log2)) + (threadIdx.x >> l.log2);
  const uint32_t block = blockIdx.y * kThreads + (threadIdx.x & ((1u << l.log2) - 1));
  if (task >= slots + rows || block >= l.blocks) return;
  const uint64_t c = uint64_t(block) * N;
  float acc[N] = {};
  if (task < slots) {
    if (task >= uint32_t(2 * uint64_t(in.offset[rows]) / piece)) return;
    const Piece p = in.piece[task];
    if (p.row == kNoPiece) return;
    sum_tokens<T, N>(grad_out, stride, in.order, p.from, p.to, c, cols, acc);
    float* dst = in.partial + task * cols + c;
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (c + k < cols) dst[k] = acc[k];
    return;
  }
  const uint64_t row = task - slots;
  const uint32_t from = in.offset[row], to = in.offset[row + 1];
  if (to - from > 2 * piece || (accumulate && from == to)) return;
  sum_tokens<T, N>(grad_out, stride, in.order, from, to, c, cols, acc);
  put_row<G, N>(grad + row * cols, c, cols, scale, accumulate, acc);
}

template <typename G>
__global__ __launch_bounds__(kThreads) void join_kernel(G* grad, uint64_t rows, uint64_t cols, uint32_t slots,
                                                        uint32_t piece, float scale, bool accumulate, Lanes l,
                                                        Sorted in) {
  constexpr int N = 4;
  const uint64_t task = (uint64_t(blockIdx.x) << (8 - l.log2)) + (threadIdx.x >> l.log2);
  const uint32_t block = blockIdx.y * kThreads + (threadIdx.x & ((1u << l.log2) - 1));
  if (task >= slots || block >= l.blocks || task >= uint32_t(2 * uint64_t(in.offset[rows]) / piece)) return;
  const Piece p = in.piece[task];
  if (p.row == kNoPiece || p.k != 0) return;
  const uint32_t n = in.offset[p.row + 1] - in.offset[p.row];
  const uint32_t pieces = (n + piece - 1) / piece;
  const uint64_t c = uint64_t(block) * N;
  float acc[N] = {};
  const float* src = in.partial + task * cols + c;
  for (uint32_t i = 0; i < pieces; ++i) {
    if (c + N <= cols) {
      float x[N];
      load<float, N>(src + i * cols, x);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += x[k];
    } else {
      for (int k = 0; c + k < cols; ++k) acc[k] += src[i * cols + k];
    }
  }
  put_row<G, N>(grad + uint64_t(p.row) * cols, c, cols, scale, accumulate, acc);
}

// ---------------------------------------------------------------------- host

bool float_dtype(int32_t dt) { return dt == SR_DT_F32 || dt == SR_DT_BF16 || dt == SR_DT_F16; }

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
  if (s->n_tokens && s->tokens == nullptr) return fail(SR_EINVAL, "%s: tokens is null", who);
  if (!aligned(s->tokens, s->token_dtype)) return fail(SR_EALIGN, "%s: tokens not aligned", who);
  return SR_OK;
}

bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && x < y + nb && y < x + na;
}

// Bytes from the first element of a matrix to behind its last.
uint64_t extent(uint64_t rows, uint64_t cols, uint64_t stride, int32_t dt) {
  return rows && cols ? ((rows - 1) * stride + cols) * sr_internal::dtype_size(dt) : 0;
}

template <typename T>
void launch_embedding(const sr_embedding_shape& s, const void* weight, uint64_t stride, void* out, hipStream_t stream) {
  const Lanes l = lanes_of(s.cols, 16 / sizeof(T));
  const uint32_t group = uint32_t(kThreads) >> l.log2;
  const dim3 grid(uint32_t((s.n_tokens + group - 1) / group), l.slices);
  if (s.token_dtype == SR_DT_I64)
    embedding_kernel<T, int64_t><<<grid, kThreads, 0, stream>>>(
        static_cast<const int64_t*>(s.tokens), static_cast<const T*>(weight), static_cast<T*>(out),
        uint32_t(s.n_tokens), s.rows, s.cols, stride, s.vocab_start, s.scale, l);
  else
    embedding_kernel<T, int32_t><<<grid, kThreads, 0, stream>>>(
        static_cast<const int32_t*>(s.tokens), static_cast<const T*>(weight), static_cast<T*>(out),
        uint32_t(s.n_tokens), s.rows, s.cols, stride, s.vocab_start, s.scale, l);
}

// The parts of the workspace.  Pieces grow with the number of tokens, so that
// a row of all tokens is joined from 1024 pieces at most.
struct Layout {
  uint32_t piece, slots;
  uint64_t order, pieces, partial, bytes;
};

Layout layout_of(const sr_embedding_shape& s) {
  Layout w;
  w.piece = 32;
  while (s.n_tokens / w.piece > 512) w.piece *= 2;
  w.slots = uint32_t(2 * s.n_tokens / w.piece);
  auto up = [](uint64_t b) { return (b + 255) / 256 * 256; };
  w.order = up((s.rows + 1) * 4);
  w.pieces = w.order + up(s.n_tokens * 4);
  w.partial = w.pieces + up(uint64_t(w.slots) * sizeof(Piece));
  w.bytes = w.partial + uint64_t(w.slots) * s.cols * 4;
  return w;
}

template <typename T, typename G>
void launch_sum(const sr_embedding_shape& s, const Layout& w, const Sorted& sorted, const void* grad_out,
                uint64_t stride, void* grad, bool accumulate, hipStream_t stream) {
  const Lanes l = lanes_of(s.cols, 16 / sizeof(T));
  const uint32_t group = uint32_t(kThreads) >> l.log2;
  const dim3 grid(uint32_t((w.slots + s.rows + group - 1) / group), l.slices);
  sum_kernel<T, G><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(grad_out), stride, static_cast<G*>(grad),
                                                  s.rows, s.cols, w.slots, w.piece, s.scale, accumulate, l, sorted);
  if (s.n_tokens <= 2 * w.piece) return;     // no row is cut
  const Lanes j = lanes_of(s.cols, 4);
  const uint32_t joined = uint32_t(kThreads) >> j.log2;
  const dim3 join_grid((w.slots + joined - 1) / joined, j.slices);
  join_kernel<G><<<join_grid, kThreads, 0, stream>>>(static_cast<G*>(grad), s.rows, s.cols, w.slots, w.piece, s.scale,
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
  const uint64_t out_bytes = extent(s.n_tokens, s.cols, s.cols, s.dtype);
  if (overlap(out, out_bytes, weight, extent(s.rows, s.cols, weight_stride, s.dtype)) ||
      overlap(out, out_bytes, s.tokens, s.n_tokens * sr_internal::dtype_size(s.token_dtype)))
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
  const uint64_t grad_bytes = extent(s.rows, s.cols, s.cols, grad_dtype);
  if (overlap(grad, grad_bytes, grad_out, extent(s.n_tokens, s.cols, grad_out_stride, s.dtype)) ||
      overlap(grad, grad_bytes, s.tokens, s.n_tokens * sr_internal::dtype_size(s.token_dtype)) ||
      overlap(grad, grad_bytes, workspace, w.bytes))
    return fail(SR_EOVERLAP, "sr_embedding_grad: the gradient overlaps an input");
  char* base = static_cast<char*>(workspace);
  const Sorted sorted{reinterpret_cast<uint32_t*>(base), reinterpret_cast<uint32_t*>(base + w.order),
                      reinterpret_cast<Piece*>(base + w.pieces), reinterpret_cast<float*>(base + w.partial)};
  const uint32_t range = uint32_t(std::min<uint64_t>(kSortRows, (s.rows + kSortRanges - 1) / kSortRanges));
  const uint32_t blocks = uint32_t((s.rows + range - 1) / range);
  if (s.token_dtype == SR_DT_I64)
    sort_kernel<int64_t><<<blocks, kSortThreads, 0, stream>>>(static_cast<const int64_t*>(s.tokens),
                                                             uint32_t(s.n_tokens), s.rows, s.vocab_start, range,
                                                             w.piece, sorted);
  else
    sort_kernel<int32_t><<<blocks, kSortThreads, 0, stream>>>(static_cast<const int32_t*>(s.tokens),
                                                             uint32_t(s.n_tokens), s.rows, s.vocab_start, range,
                                                             w.piece, sorted);
  if (int rc = launched("sr_embedding_grad: sort")) return rc;
  if (s.dtype == SR_DT_F32) launch_sum_to<float>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  else if (s.dtype == SR_DT_BF16) launch_sum_to<bf16>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  else launch_sum_to<f16>(grad_dtype, s, w, sorted, grad_out, grad_out_stride, grad, accumulate != 0, stream);
  return launched("sr_embedding_grad");
}

}  // extern "C"
