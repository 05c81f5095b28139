// sr_tile.h -- products of matrices in tiles on the matrix cores, shared by
// the operators on a share's matrices (not part of the C ABI).
//
//   C[m][n] = sum over k of A[m][k] B[n][k]
//
// Each operand is stored either with its k side by side (a row a line: ROW) or
// with its rows side by side (a k a line: COL), so every product of a forward
// and a backward pass works on the tensors as they are.  A tile is 256 x 256 with
// 8 waves of 128 x 64, 128 x 128 with 4 of 64 x 64, or 64 x 64 with 2 of 32 x 64
// (of floats with two sets of these).
//
//   - A step takes 128 bytes of every row: 64 values of 16 bits or 32 floats.
//     They go from memory straight into shared memory, 16 bytes a lane, into
//     the half that the step before has left, while the matrix cores work on
//     the other one: one barrier a step.
//   - 16-byte pieces are permuted within a line (by the lanes' addresses in
//     memory, as the lanes' places in shared memory are fixed), so that eight
//     lanes which read one column of pieces meet eight different bank groups.
//   - COL operands of 16 bits are transposed on the way to the registers, by
//     the read of shared memory that does so.
//   - What lies outside an operand is read as zero: such lanes ask for an
//     address beyond the buffer resource.
//
// A 256 x 256 tile of 16 bits does 128 operations for a byte that it loads, and 43
// for one that its waves read of shared memory.  The matrix cores alone reach 1.88
// PFLOP/s of bf16 here, with these reads 1.54, with the loads and barriers of whole
// products 1.25 to 1.28 (f16 pairs, below, 1.34 to 1.38): a step has one barrier, at
// which the waves meet.  128 x 128 tiles load twice as much, but two workgroups fill
// each other's gaps: 1.17 and 1.22.  They and 64 x 64 ones serve products with few
// tiles; Cost, below, says which is taken.
//
// Values of 22 bits (TWO): a matrix as two of f16, the values rounded and what
// the rounding lost, 32 of the one and 32 of the other in turn in every row.
// The product of two such matrices is three products of f16, the one of the two
// remainders, below 2^-22, left out; sums are in f32.
#ifndef SR_TILE_H
#define SR_TILE_H

#include "sr_step.h"

namespace sr_tile {

using sr_step::bf16;
using sr_step::f16;
using sr_step::kWave;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char* Shared;

constexpr int kLine = 128;                       // bytes of a row in a step
constexpr uint32_t kOutside = 0x80000000u;       // an offset beyond every resource
constexpr uint32_t kResource = 0x7fffffffu;
constexpr uint64_t kMostStride = uint64_t(1) << 22;     // bytes from row to row: 256 rows within a resource

constexpr int kAllLoads = 0x0f70;                // s_waitcnt vmcnt(0)

// Threads of a workgroup; `halves`: sets of waves that share out a step's k.  Two for
// 64 x 64 tiles of floats, whose products take long where a compute unit has but one.
template <typename T> constexpr int halves(int size) { return size == 64 && sizeof(T) == 4 ? 2 : 1; }
template <typename T> constexpr int threads(int size) {
  return size == 256 ? 512 : size == 128 ? 256 : 128 * halves<T>(64);
}

enum Side { ROW, COL };

// A matrix with its rows or its k side by side, as a kernel takes it.
struct Operand {
  uint64_t data;
  uint64_t stride;     // bytes from line to line
  uint32_t rows;       // values of a COL operand's line, or lines of a ROW one (padded: see TWO)
};

// ------------------------------------------------------- blocks of 32 x 32

template <typename T> struct Block;

template <> struct Block<bf16> {
  typedef __bf16 Frag __attribute__((ext_vector_type(8)));
  __device__ static void add(const Frag& b, const Frag& a, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, a, c, 0, 0, 0);
  }
};

template <> struct Block<f16> {
  typedef _Float16 Frag __attribute__((ext_vector_type(8)));
  __device__ static void add(const Frag& b, const Frag& a, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(b, a, c, 0, 0, 0);
  }
};

// Four k a lane: which four does not matter as long as both operands agree.
template <> struct Block<float> {
  typedef f32x4 Frag;
  __device__ static void add(const Frag& b, const Frag& a, f32x16& c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j], a[j], c, 0, 0, 0);
  }
};

// ---------------------------------------------------------------- operands

// One operand's part of a tile: ROWS rows, a step's k.  PAIR: the rows of two
// matrices in turn, 32 * PAIR of the one and as many of the other.
template <typename T, bool TWO, Side SIDE, int ROWS, int PAIR, int kThreads>
struct Part {
  static constexpr int kEach = 16 / sizeof(T);                       // values of a piece
  static constexpr int kK = kLine / int(sizeof(T)) / (TWO ? 2 : 1);  // of a step
  static constexpr int kBytes = ROWS * kLine;
  static constexpr int kLoads = kBytes / (kThreads * 16);
  // pieces of a line in shared memory
  static constexpr int kPieces = SIDE == ROW ? kLine / 16 : ROWS * int(sizeof(T)) * (TWO ? 2 : 1) / 16;
  static constexpr int kLines = kThreads / kPieces;                  // of one load
  static_assert(kThreads % kPieces == 0 && (PAIR == 0 || SIDE == ROW), "whole lines a load");

  uint64_t data[2];       // of both matrices
  uint32_t at[kLoads];     // bytes from data, or kOutside
  uint32_t piece;          // of a line: which of its pieces this lane loads
  uint64_t step;           // bytes from step to step

  // How a piece's place in its line is permuted: sixteen lanes that read a column
  // of pieces (ROW), or four lines of two pieces and their neighbours' (COL), meet
  // all 64 banks.
  __device__ static uint32_t turn(uint32_t line) {
    static_assert(kPieces >= 8, "a permuted place is one of the line's");
    return SIDE == ROW ? line / 2 & 7 : (line & 3) << (kPieces == 8 ? 1 : 2);
  }

  // Which matrix a wave's lines of a load are of.
  static constexpr int kTurn = PAIR ? 32 * PAIR : 1;
  __device__ __forceinline__ static int half_of(int i) {
    if (!PAIR) return 0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    return (i * kLines + wave * (kWave / kPieces)) / kTurn % 2;
  }

  // Rows from `first` on, k from `k` on.
  __device__ __forceinline__ void start(const Operand& o, const Operand& other, uint32_t first, uint32_t k) {
    const uint32_t line = threadIdx.x / kPieces;
    piece = threadIdx.x % kPieces;
    static_assert(SIDE == COL || kLines % 8 == 0, "a lane's lines are permuted alike");
    step = SIDE == ROW ? kLine : kK * o.stride;
    const uint64_t along = (TWO ? 2 : 1) * sizeof(T);
    data[0] = o.data + (SIDE == ROW ? first * o.stride + k * along : first * along + k * o.stride);
    if (PAIR) data[1] = other.data + first * other.stride + k * along;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t l = i * kLines + line;
      if (SIDE == ROW) {
        const uint32_t r = PAIR ? l / (2 * kTurn) * kTurn + l % kTurn : l;
        const uint64_t mine = o.stride, others = other.stride, stride = PAIR && half_of(i) ? others : mine;
        at[i] = first + r < o.rows ? uint32_t(r * stride) + (piece ^ turn(l)) * 16 : kOutside;
      } else {
        const uint32_t p = piece ^ turn(l);
        at[i] = first * (TWO ? 2 : 1) + p * kEach < o.rows ? uint32_t(l * o.stride) + p * 16 : kOutside;
      }
    }
    if (SIDE == ROW) piece ^= turn(line);
  }

  // Loads a step into shared memory; `left`: k from here to the end.
  __device__ __forceinline__ void load(Shared to, uint32_t left) const {
    const Shared mine = to + threadIdx.x / kWave * (kWave * 16);
    const bool whole = left >= kK;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t offset = at[i];
      if (!whole) {
        // (TWO: rows are padded to whole steps)
        const bool in = SIDE == ROW ? TWO || piece * kEach < left : i * kLines + threadIdx.x / kPieces < left;
        offset = in ? offset : kOutside;
      }
      const uint64_t first = data[0], second = data[1];
      const sr_step::Region from = sr_step::region(reinterpret_cast<void*>(half_of(i) ? second : first), kResource);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, mine + i * kThreads * 16, 16, offset, 0, 0, 0);
    }
  }

  __device__ __forceinline__ void next() {
    data[0] += step;
    if (PAIR) data[1] += step;
  }

  // The block of 32 rows from `first` on (a multiple of 32), k group `s` of the
  // step; LOW: of the remainders.
  template <bool LOW>
  __device__ static __forceinline__ typename Block<T>::Frag frag(Shared from, int first, int s) {
    const uint32_t lane = threadIdx.x % kWave;
    if constexpr (SIDE == ROW) {
      const uint32_t line = first + lane % 32;
      const uint32_t p = (2 * s + lane / 32 + (LOW ? 4 : 0)) ^ turn(line);
      typedef __attribute__((address_space(3))) const typename Block<T>::Frag* Source;
      return *(Source)(from + line * kLine + p * 16);
    } else if constexpr (sizeof(T) == 2) {
      // Sixteen lanes read 4 lines of 16 values and get a column of 4 each.
      const uint32_t column = (TWO ? 2 : 1) * first + (LOW ? 32 : 0) + lane / 16 % 2 * 16 + lane % 4 * 4;
      s16x4 half[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t line = 16 * s + lane / 32 * 8 + 4 * j + lane % 16 / 4;
        const uint32_t p = (column / 8) ^ turn(line);
        typedef __attribute__((address_space(3))) s16x4* Source;
        half[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Source)(from + line * (kPieces * 16) + p * 16 + column % 8 * 2));
      }
      const s16x8 both = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(typename Block<T>::Frag, both);
    } else {
      typename Block<T>::Frag f;
      const uint32_t column = first + lane % 32;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t line = 8 * s + lane / 32 * 4 + j;
        const uint32_t p = (column / 4) ^ turn(line);
        typedef __attribute__((address_space(3))) const float* Source;
        f[j] = *(Source)(from + line * (kPieces * 16) + p * 16 + column % 4 * 4);
      }
      return f;
    }
  }
};

// ------------------------------------------------------------------- tiles

// One tile: T: the operands' type, TWO: values of 22 bits, SIZE: rows and
// columns, A, B: how they are stored, PAIR: B's rows are those of two matrices
// in turn, so that a wave has both products of the same columns.
template <typename T, bool TWO_, int SIZE_, Side A, Side B, bool PAIR_ = false>
struct Tile {
  static constexpr int SIZE = SIZE_;
  static constexpr bool TWO = TWO_, PAIR = PAIR_;
  static constexpr int kThreads = threads<T>(SIZE), kHalves = halves<T>(SIZE);
  static constexpr int WAVES = kThreads / kWave / kHalves;       // of a half
  static constexpr int kRows = SIZE / 2, kSpan = SIZE / (WAVES / 2);     // of a wave
  static constexpr int kI = kRows / 32, kJ = kSpan / 32;
  static constexpr int kColumns = PAIR ? SIZE / 2 : SIZE;     // of C
  typedef Part<T, TWO, A, SIZE, 0, kThreads> PartA;
  typedef Part<T, TWO, B, SIZE, PAIR ? kSpan / 64 : 0, kThreads> PartB;
  static constexpr int kK = PartA::kK;
  static constexpr int kGroups = kLine / 32 / (TWO ? 2 : 1) / kHalves;       // k groups of a step, of a half
  // floats of a slab's row; four more, where there is room, turn the banks of the next
  static constexpr int kWide = SIZE == 64 ? 64 : 64 + 4;
  static constexpr int kSlab = 32 * kWide * 4;
  static_assert(kJ % 2 == 0, "slabs of two blocks");
  static constexpr int kSlabs = SIZE * kLine / kSlab;       // in the memory of an operand
  static_assert(WAVES <= 4 * kSlabs, "the waves' slabs fit where the operands were");

  f32x16 c[kI][kJ];

  // Sums of floats are formed of sums over 256 k: one over 2120 k is 1.3e-6 of the
  // result's size off, 5e-7 in parts.  What 16 bits round off hides that.
  static constexpr bool kParts = sizeof(T) == 4;
  static constexpr uint32_t kPart = 8;      // steps
  f32x16 whole[kParts ? kI : 1][kParts ? kJ : 1];

  __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) % WAVES; }
  __device__ __forceinline__ static int half() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) / WAVES; }
  __device__ __forceinline__ static int wave_row() { return wave() % 2 * kRows; }
  __device__ __forceinline__ static int wave_column() { return wave() / 2 * kSpan; }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        c[i][j] = f32x16(0.0f);
        if constexpr (kParts) whole[i][j] = f32x16(0.0f);
      }
  }

  // The end of a part.
  __device__ __forceinline__ void part() {
    if constexpr (kParts) {
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          whole[i][j] += c[i][j];
          c[i][j] = f32x16(0.0f);
        }
    }
  }

  // The sums, in `c` of the first half's waves; every wave comes by.  The second
  // half's go through the slabs, of which its waves have none.
  __device__ __forceinline__ void join(Shared a0, Shared a1, Shared b0, Shared b1) {
    if constexpr (kParts) {
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) c[i][j] += whole[i][j];
    }
    if constexpr (kHalves > 1) {
      static_assert(kHalves == 2 && kI * kJ * 16 * kWave * 4 <= kSlab, "a wave's sums fit its slab");
      typedef __attribute__((address_space(3))) f32x4* Fours;
      const Fours mine = (Fours)slab(a0, a1, b0, b1) + threadIdx.x % kWave;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (half() != r) {
#pragma unroll
          for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const Fours at = mine + ((i * kJ + j) * 4 + q) * kWave;
                f32x16& x = c[i][j];
                if (r == 0) {
                  *at = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                } else {
                  const f32x4 more = *at;
#pragma unroll
                  for (int e = 0; e < 4; ++e) x[4 * q + e] += more[e];
                }
              }
        }
        if (r == 0) __syncthreads();
      }
    }
  }

  // The operands of a k group.
  struct Group {
    typename Block<T>::Frag a[kI], b[kJ], low_a[TWO ? kI : 1], low_b[TWO ? kJ : 1];

    __device__ __forceinline__ void read(Shared sa, Shared sb, int s) {
      const int row = wave_row(), column = wave_column();
      if (kHalves > 1) s += half() * kGroups;
#pragma unroll
      for (int j = 0; j < kJ; ++j) b[j] = PartB::template frag<false>(sb, column + 32 * j, s);
#pragma unroll
      for (int i = 0; i < kI; ++i) a[i] = PartA::template frag<false>(sa, row + 32 * i, s);
      if constexpr (TWO) {
#pragma unroll
        for (int j = 0; j < kJ; ++j) low_b[j] = PartB::template frag<true>(sb, column + 32 * j, s);
#pragma unroll
        for (int i = 0; i < kI; ++i) low_a[i] = PartA::template frag<true>(sa, row + 32 * i, s);
      }
    }
  };

  // The products of a k group.  With 128 x 128 tiles a wave that multiplies goes
  // before those of the other workgroup, whose loads and barriers fill its gaps
  // (bf16 1.10 to 1.17 PFLOP/s, values of 22 bits 1.19 to 1.27; with 256 x 256
  // tiles 1-2% slower).
  __device__ __forceinline__ void multiply(const Group& x) {
    typedef Block<T> K;
    auto each = [&](const auto& fb, const auto& fa) {
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) K::add(fb[j], fa[i], c[i][j]);
    };
    if (SIZE == 128) __builtin_amdgcn_s_setprio(1);
    each(x.b, x.a);
    if constexpr (TWO) {
      each(x.b, x.low_a);
      each(x.low_b, x.a);
    }
    if (SIZE == 128) __builtin_amdgcn_s_setprio(0);
  }

  // A step's products but for the last group's, which are left in `g`, as the
  // first group's are at the start.
  __device__ __forceinline__ void most_products(Group (&g)[2], Shared sa, Shared sb) {
#pragma unroll
    for (int s = 0; s + 1 < kGroups; ++s) {
      g[(s + 1) % 2].read(sa, sb, s + 1);
      multiply(g[s % 2]);
      // reads of the next group between this one's products (3% for 256 x 256 of ROW)
      constexpr int kReads = (kI + kJ) * (TWO ? 2 : 1), kProducts = kI * kJ * (TWO ? 3 : 1);
#pragma unroll
      for (int q = 0; q < kReads; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, kProducts / kReads, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ void last_products(const Group (&g)[2]) {
    multiply(g[(kGroups - 1) % 2]);
    __builtin_amdgcn_sched_barrier(0);
  }

  // f(row, column, values) on this wave's values as they lie in its registers:
  // four columns of a row a lane.
  template <typename F>
  __device__ __forceinline__ void values(F&& f) {
    const uint32_t lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4] = {c[i][j][4 * q], c[i][j][4 * q + 1], c[i][j][4 * q + 2], c[i][j][4 * q + 3]};
          f(uint32_t(wave_row() + 32 * i) + lane % 32, uint32_t(wave_column() + 32 * j + 8 * q) + lane / 32 * 4, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[i][j][4 * q + e] = v[e];
        }
  }

  // This wave's slab, where the operands were.
  __device__ __forceinline__ static Shared slab(Shared a0, Shared a1, Shared b0, Shared b1) {
    const int in = wave() / kSlabs;
    return (in == 0 ? a0 : in == 1 ? a1 : in == 2 ? b0 : b1) + wave() % kSlabs * kSlab;
  }

  // The rows and columns of this wave, eight values a lane: f(row, column,
  // values, what load(row, column) has returned) with the row and the first column
  // in the tile.  FLIP: of the transpose of C.  With PAIR, the values of the second
  // matrix come behind the first one's.  What is loaded for 32 rows is on its way
  // at once or, with ROLLED, for the next 8 while these are worked on, in a loop
  // that stays one: for so much work a value that the compiler would not unroll the
  // loop around it, without which C has no registers.  `slab`: the wave's, no
  // longer read as operands.
  template <bool FLIP, bool ROLLED, typename L, typename F>
  __device__ __forceinline__ void results(Shared slab, L&& load, F&& f) const {
    static_assert(!(FLIP && (PAIR || kI % 2)), "slabs of two blocks");
    if (kHalves > 1 && half()) return;
    const uint32_t lane = threadIdx.x % kWave;
    const int row0 = FLIP ? wave_column() : wave_row();
    const int column0 = PAIR ? wave_column() / 2 : FLIP ? wave_row() : wave_column();
    typedef __attribute__((address_space(3))) float* Floats;
    typedef __attribute__((address_space(3))) f32x4* Fours;
    const Floats mine = (Floats)slab;
    constexpr int kDown = FLIP ? kJ : kI, kAcross = FLIP ? kI : kJ;      // blocks
#pragma unroll
    for (int i = 0; i < kDown; ++i)
#pragma unroll
      for (int j = 0; j < kAcross / 2; ++j) {
        constexpr int kLanes = (PAIR ? 32 : 64) / 8;     // of a row
        constexpr int kPasses = 32 * kLanes / kWave;
        auto row_of = [&](int p) { return uint32_t(row0 + 32 * i + p * (kWave / kLanes)) + lane / kLanes; };
        const uint32_t column = uint32_t(column0 + (PAIR ? 32 : 64) * j) + lane % kLanes * 8;
        decltype(load(0u, 0u)) loaded[ROLLED ? 1 : kPasses];
#pragma unroll
        for (int p = 0; p < (ROLLED ? 1 : kPasses); ++p) loaded[p] = load(row_of(p), column);
        // two blocks; a lane has the column lane % 32 of a block's transpose, four rows together
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int across = PAIR ? j + h * (kAcross / 2) : 2 * j + h;
          const f32x16& x = FLIP ? c[across][i] : c[i][across];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = 8 * q + lane / 32 * 4;
            if (!FLIP) {
              *(Fours)(mine + lane % 32 * kWide + 32 * h + n) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) mine[(n + r) * kWide + 32 * h + lane % 32] = x[4 * q + r];
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");     // the wave's own writes, read by other lanes
        __builtin_amdgcn_wave_barrier();
        auto pass = [&](int p, const auto& with) {
          const int r = p * (kWave / kLanes) + lane / kLanes, n = lane % kLanes * 8;
          float v[8], w[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x4 x = *(Fours)(mine + r * kWide + n + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * h + e] = x[e];
            if constexpr (PAIR) {
              const f32x4 y = *(Fours)(mine + r * kWide + 32 + n + 4 * h);
#pragma unroll
              for (int e = 0; e < 4; ++e) w[4 * h + e] = y[e];
            }
          }
          if constexpr (PAIR) f(row_of(p), column, v, w, with);
          else f(row_of(p), column, v, with);
        };
        if constexpr (ROLLED) {
#pragma unroll 1
          for (int p = 0; p < kPasses; ++p) {
            const auto now = loaded[0];
            if (p + 1 < kPasses) loaded[0] = load(row_of(p + 1), column);
            pass(p, now);
          }
        } else {
#pragma unroll
          for (int p = 0; p < kPasses; ++p) pass(p, loaded[p]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
      }
  }
};

// Two operands, and a second pair whose products are added (its data 0: none)
// or, with PAIR, whose B has the second matrix's rows.
struct Product {
  Operand a, b, a2, b2;
  uint32_t k;          // of one pair
};

// All steps from `from` to `to` (steps of the second pair are counted on) of
// the tile at (row, column).  A macro's worth of memory: the halves are arrays
// of their own, so that a read of the one does not wait for loads to the other.
template <typename Tile>
__device__ __forceinline__ void run(Tile& tile, const Product& p, uint32_t row, uint32_t column, uint32_t from,
                                    uint32_t to, Shared a0, Shared a1, Shared b0, Shared b1) {
  typename Tile::PartA a;
  typename Tile::PartB b;
  const uint32_t each = (p.k + Tile::kK - 1) / Tile::kK;     // steps of a pair
  uint32_t left = 0;
  auto seek = [&](uint32_t s) {
    const bool second = !Tile::PAIR && s >= each;
    const uint32_t k = (second ? s - each : s) * Tile::kK;
    a.start(second ? p.a2 : p.a, p.a2, row, k);
    b.start(second ? p.b2 : p.b, p.b2, column, k);
    left = p.k - k;
  };
  auto fetch = [&](uint32_t s, Shared to_a, Shared to_b) {
    if (!Tile::PAIR && s == each) seek(s);
    a.load(to_a, left);
    b.load(to_b, left);
    a.next();
    b.next();
    left -= Tile::kK;
  };
  tile.clear();
  if (from >= to) return;
  seek(from);
  typename Tile::Group g[2];
  // The barrier: the next step has arrived, and this one's operands have all been
  // read; its last group is still to be multiplied, which hides the first reads
  // of the next step.
  // The wait for this wave's own loads is written out: a barrier by itself orders
  // shared memory's reads and writes, but not what loads write there.
  auto turn_over = [&] {
    __builtin_amdgcn_s_waitcnt(kAllLoads);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };
  fetch(from, a0, b0);
  turn_over();
  if (from + 1 < to) fetch(from + 1, a1, b1);
  g[0].read(a0, b0, 0);
  uint32_t s = from;
  for (; s + 2 <= to; s += 2) {
    tile.most_products(g, a0, b0);
    turn_over();
    if (s + 2 < to) fetch(s + 2, a0, b0);
    g[0].read(a1, b1, 0);
    tile.last_products(g);
    tile.most_products(g, a1, b1);
    turn_over();
    if (s + 3 < to) fetch(s + 3, a1, b1);
    if (s + 2 < to) g[0].read(a0, b0, 0);
    tile.last_products(g);
    if (Tile::kParts && (s - from + 2) % Tile::kPart == 0) tile.part();
  }
  if (s < to) {
    tile.most_products(g, a0, b0);
    tile.last_products(g);
  }
  tile.join(a0, a1, b0, b1);
}

// What a workgroup of these kernels has of shared memory: two halves of both
// operands, arrays of their own (see sr_tile::run), then the waves' slabs.
#define SR_TILE_MEMORY(Tile)                                                     \
  __shared__ __attribute__((aligned(1024))) char a0[Tile::PartA::kBytes];        \
  __shared__ __attribute__((aligned(1024))) char a1[Tile::PartA::kBytes];        \
  __shared__ __attribute__((aligned(1024))) char b0[Tile::PartB::kBytes];        \
  __shared__ __attribute__((aligned(1024))) char b1[Tile::PartB::kBytes]
#define SR_TILE_SLAB(Tile) \
  Tile::slab((sr_tile::Shared)a0, (sr_tile::Shared)a1, (sr_tile::Shared)b0, (sr_tile::Shared)b1)

// Items of a launch in the order that workgroups take them: as many neighbours
// on one die as run there at once, die after die, so that they share rows and
// columns in its L2 and all dies have the same mix of long and short ones (an
// eighth of the items each: where the long ones come first, 2.1 ms instead of
// 1.6).  What is left behind whole rounds goes to the dies by eighths.
constexpr uint32_t at_once(int size) { return size == 256 ? 32 : size == 128 ? 64 : 128; }      // of a die's 32 compute units

inline uint32_t blocks_of(uint32_t items, int size) {
  const uint32_t round = at_once(size) * sr_step::kXcds;
  return items / round * round + sr_step::xcd_blocks(items % round);
}

__device__ __forceinline__ uint32_t item_of(uint32_t block, uint32_t items, int size) {
  const uint32_t round = at_once(size) * sr_step::kXcds, first = block / round * round, in = block - first;
  if (first + round <= items) return first + in % sr_step::kXcds * at_once(size) + in / sr_step::kXcds;
  return first + sr_step::xcd_order(in, items - first);
}

// A launch's tiles and items.
struct Grid {
  uint32_t rows, columns;
  uint32_t items;
};

// Most workgroups of a launch: a grid has fewer than 2^32 threads, 512 a workgroup.
constexpr uint64_t kMostItems = (uint64_t(1) << 23) - 2 * sr_step::kXcds;

// For results that nothing is loaded for.
struct Nothing {};
__device__ __forceinline__ Nothing nothing(uint32_t, uint32_t) { return {}; }

// How long a launch of tiles takes, in units of 0.4 us, a quarter of a 256 x 256
// tile's step of 16-bit operands.  Of tiles alike, the compute unit with the most of
// them counts.  256 x 256 tiles run one after another on it; smaller ones share it,
// and have its latencies to themselves where there are few.  Measured, n tiles a
// unit: 4.0 n a step, 1.15 n + 0.8 for 128 x 128 (2.0, 3.1, 4.0 and 13.5 for 1, 2, 3 and
// 13), 0.5 n + 0.8 for 64 x 64 (1.4, 1.5, 3.4 and 4.6 for 2, 3, 5 and 10); floats,
// which the matrix cores take 16 times as long for, 3.7 n + 1.4 and n + 1 (with 3.1 n + 2
// and n + 2.5, that take larger tiles more often, 4096 x 1024 x 1024 782 us instead of
// 675).  Of a mixture the sum counts, and half of the longest tile, which ends last.  Six steps
// are added for a tile's first loads and its results.
class Cost {
 public:
  Cost(int size, bool f32) : size_(size), f32_(f32) {}

  void add(uint64_t tiles, uint64_t steps) {
    if (tiles == 0) return;
    const double t = double(steps) + 6;
    alike_ = alike_ && (tiles_ == 0 || t == longest_);
    tiles_ += tiles;
    sum_ += double(tiles) * t;
    longest_ = t > longest_ ? t : longest_;
  }
  double time() const {
    if (!alike_) return (sum_ / kUnits + longest_ / 2) * shared();
    const double each = double((tiles_ + kUnits - 1) / kUnits);
    return (each * shared() + alone()) * longest_;
  }

 private:
  static constexpr uint64_t kUnits = 256;      // compute units

  double shared() const {
    if (f32_) return size_ == 128 ? 3.7 : 1.0;
    return size_ == 256 ? 4.0 : size_ == 128 ? 1.15 : 0.5;
  }
  double alone() const {
    if (f32_) return size_ == 128 ? 1.4 : 1.0;
    return size_ == 256 ? 0.0 : 0.8;
  }

  int size_;
  bool f32_, alike_ = true;
  uint64_t tiles_ = 0;
  double sum_ = 0, longest_ = 0;
};

// The tile of a work item, in bands of 8 tiles' rows: the tiles of neighbouring
// items share rows and columns.
__device__ __forceinline__ void banded(uint32_t item, uint32_t rows, uint32_t columns, uint32_t& row, uint32_t& column) {
  constexpr uint32_t kBand = 8;
  const uint32_t band = item / (kBand * columns) * kBand, in = item - band * columns;
  const uint32_t high = rows - band < kBand ? rows - band : kBand;
  row = band + in % high;
  column = in / high;
}

}  // namespace sr_tile

#endif  // SR_TILE_H
