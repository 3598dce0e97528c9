// Device helpers shared by the decayed linear attention and the window attention kernels:
// matrix tiles in LDS, operands of the matrix instructions, and the map from blocks to
// sequences.
//
// Everything is built from one product, D[16 x 16] += A[16 x 32] B[32 x 16] in float32.  Lane
// l = 16 g + c of a wave holds A[c][8 g .. 8 g + 7], B[8 g .. 8 g + 7][c] and D[4 g + r][c],
// r = 0..3.  For the 16-bit types that is v_mfma_f32_16x16x32; for float32 the same operands
// are fed to eight v_mfma_f32_16x16x4 (the order of the 32 terms is free as long as A and B
// agree), so that a kernel is written once for all three types.
//
// Two ways of reading an operand from a row-major tile exist.  Along a row (the summed index is
// the column): 8 neighbouring elements.  Down a column (the summed index is the row): lanes of
// group g take rows 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 of a block of 32, with the
// transposing LDS read of gfx950 for the 16-bit types.  That choice of rows is the one in which
// two D tiles, one below the other, already lie: a product's result is the next product's
// operand without leaving the registers of its lane (operand_of).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/rosa_soft_hip.h"

namespace rosa_mixer {

constexpr int kThreads = 256;      // four waves
constexpr int kGroups = 8;         // XCDs; consecutive blocks go to them in turn

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T> using Frag = T __attribute__((ext_vector_type(8)));
template <typename T> using Quad = T __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mma(Frag<__bf16> a, Frag<__bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Frag<_Float16> a, Frag<_Float16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Frag<float> a, Frag<float> b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }

// lambda^n from log2(lambda); lambda^0 is 1 for lambda = 0 too
__device__ __forceinline__ float power_of(float log2_rate, int n) {
  return n == 0 ? 1.0f : exp2_of(log2_rate * static_cast<float>(n));
}

// Over the four lanes of a column.  The exchanges of gfx950 swap half of one register with the
// other half of another: of two copies of x they leave x of this half and of the other one.
template <typename Join>
__device__ __forceinline__ float over_groups(float x, Join&& join) {
  const int bits = __float_as_int(x);
  const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  const int pair = __float_as_int(join(__int_as_float(rows[0]), __int_as_float(rows[1])));
  const auto halves = __builtin_amdgcn_permlane32_swap(pair, pair, false, false);
  return join(__int_as_float(halves[0]), __int_as_float(halves[1]));
}
__device__ __forceinline__ float over_groups_max(float x) {
  return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float over_groups_sum(float x) {
  return over_groups(x, [](float a, float b) { return a + b; });
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------

// Elements from one row of a tile to the next: 16 bytes more than the row, so that the 16 rows
// that a row-wise operand reads start in 16 different groups of four banks.
template <typename T, int WIDTH>
constexpr int kPitch = WIDTH + 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ Frag<T> load8(const T* p) {
  return *reinterpret_cast<const Frag<T>*>(p);
}

// operand whose summed index runs along the row: row `row0 + c`, columns col0 + 8 g ...
template <typename T, int WIDTH>
__device__ __forceinline__ Frag<T> row_operand(const T* tile, int row0, int col0, int lane) {
  return load8(tile + (row0 + (lane & 15)) * kPitch<T, WIDTH> + col0 + 8 * (lane >> 4));
}

// operand whose summed index runs down the rows of the block [row0, row0 + 32): column col0 + c
template <typename T, int WIDTH>
__device__ __forceinline__ Frag<T> column_operand(const T* tile, int row0, int col0, int lane) {
  Frag<T> out;
  if constexpr (sizeof(T) == 2) {
    // 16 lanes hand in four rows of 16 elements, 8 bytes each, and get a column each
    const T* at = tile + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * kPitch<T, WIDTH> + col0 +
                  4 * (lane & 3);
    typedef __attribute__((address_space(3))) s16x4 LdsQuad;
    const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(at));
    const s16x4 high =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(at + 16 * kPitch<T, WIDTH>));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    out = __builtin_bit_cast(Frag<T>, both);
  } else {
    const T* at = tile + (row0 + 4 * (lane >> 4)) * kPitch<T, WIDTH> + col0 + (lane & 15);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = at[((e & 3) + 16 * (e >> 2)) * kPitch<T, WIDTH>];
  }
  return out;
}

// two results, rows [0, 16) and [16, 32) of the summed index, as the operand of the next product
template <typename T>
__device__ __forceinline__ Frag<T> operand_of(f32x4 low, f32x4 high) {
  Frag<T> out;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    out[r] = static_cast<T>(low[r]);
    out[r + 4] = static_cast<T>(high[r]);
  }
  return out;
}

// A tile of ROWS x WIDTH on its way from memory to LDS through the registers of the block.
// `row_pointer` gives an existing row for every row of the tile (a caller repeats its last one and
// masks what comes of it), so that loads are never predicated; columns from `width` on are zeros.
// WHOLE: rows are whole 16-byte pieces at 16-byte addresses.
template <typename T, int ROWS, int WIDTH, bool WHOLE>
struct TileMove {
  static constexpr int kElements = 16 / static_cast<int>(sizeof(T));
  static constexpr int kPerRow = WIDTH / kElements;
  static constexpr int kPieces = ROWS * kPerRow / kThreads;
  static_assert(ROWS * kPerRow % kThreads == 0, "tiles are moved in whole pieces per thread");
  typedef T Piece __attribute__((ext_vector_type(kElements)));

  Piece held[kPieces];

  template <typename RowPointer>
  __device__ __forceinline__ void fetch(RowPointer&& row_pointer, int width, int tid) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * kThreads + tid, col = piece % kPerRow * kElements;
      const T* row = row_pointer(piece / kPerRow);
      if constexpr (WHOLE) {
        held[i] = *reinterpret_cast<const Piece*>(row + min(col, width - kElements));
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e) held[i][e] = row[min(col + e, width - 1)];
      }
    }
    if (width < WIDTH) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int col = (i * kThreads + tid) % kPerRow * kElements;
#pragma unroll
        for (int e = 0; e < kElements; ++e)
          held[i][e] = col + e < width ? held[i][e] : static_cast<T>(0.0f);
      }
    }
  }

  __device__ __forceinline__ void store(T* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * kThreads + tid;
      *reinterpret_cast<Piece*>(tile + piece / kPerRow * kPitch<T, WIDTH> +
                                piece % kPerRow * kElements) = held[i];
    }
  }
};

// row-wise operand straight from memory: `row` is the lane's own row
template <bool WHOLE, typename T>
__device__ __forceinline__ Frag<T> memory_operand(const T* row, int col, int width) {
  Frag<T> out;
  if constexpr (WHOLE && sizeof(T) == 2) {
    out = load8(row + min(col, width - 8));
    if (col >= width) out = Frag<T>(static_cast<T>(0.0f));
  } else if constexpr (WHOLE) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f32x4 part = *reinterpret_cast<const f32x4*>(row + min(col + 4 * half, width - 4));
      if (col + 4 * half >= width) part = f32x4(0.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * half + e] = part[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T element = row[min(col + e, width - 1)];
      out[e] = col + e < width ? element : static_cast<T>(0.0f);
    }
  }
  return out;
}

// four neighbouring elements of a contiguous output row
template <typename T>
__device__ __forceinline__ void store4(T* row, int col, f32x4 value, int width, bool quads) {
  if (quads) {
    if (col < width) {
      Quad<T> out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(value[e]);
      *reinterpret_cast<Quad<T>*>(row + col) = out;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < width) row[col + e] = static_cast<T>(value[e]);
  }
}

// The power of two that brings a largest value into float16's upper range, [2^13, 2^14): float16
// has few exponents, and what is rounded to it loses bits below 2^-14 and everything above 2^16.
// The other types take values as they are.
template <typename T> constexpr bool kNarrow = std::is_same_v<T, _Float16>;
__device__ __forceinline__ float lift_of(float largest) {
  return largest > 0.0f && largest < __builtin_inff() ? exp2_of(13.0f - floorf(log2_of(largest)))
                                                      : 1.0f;
}

// A factor for a sum over many tiles: set by the first tile that is not zero, lowered when a later
// one would pass float16's range.  Returns what the sum so far is to be multiplied by.
__device__ __forceinline__ float follow_range(float* lift, float largest) {
  const bool fresh = *lift == 0.0f;
  if (!(largest > 0.0f) || (!fresh && !(largest * *lift > 32768.0f))) return 1.0f;
  const float before = *lift;
  *lift = lift_of(largest);
  return fresh ? *lift : *lift / before;
}

// ---------------------------------------------------------------------------
// tensors, sequences, work items
// ---------------------------------------------------------------------------

// [.., tokens, heads, width] with neighbouring elements inside a head
template <typename T>
struct View {
  T* data;
  int64_t batch_stride, token_stride, head_stride;
  __device__ __forceinline__ T* row(int64_t batch, int64_t token, int head) const {
    return data + batch * batch_stride + token * token_stride + head * head_stride;
  }
};

// The sequences of a call: B of T tokens each, or S that `offsets` cuts out of N tokens.
struct Sequences {
  const int32_t* offsets;  // null: dense
  int count, length, tokens;
};

// A run of `rows` tokens of one sequence.  `batch` and `begin` address its tensors, `first` is its
// number among all tokens.
struct Run {
  int sequence, length, tile;
  int64_t batch, begin, first;
};

// Work items come in `slots`: tile i of sequence s has slot offsets[s] / rows + s + i, which
// leaves every sequence room for all its tiles (a sequence of n tokens has at most
// (begin + n) / rows - begin / rows + 1 of them) and needs no table; dense sequences have a
// fixed number of tiles each.
__host__ __device__ __forceinline__ int64_t slots_of(const Sequences& q, int rows) {
  return q.offsets == nullptr ? static_cast<int64_t>(q.count) * ((q.length + rows - 1) / rows)
                              : static_cast<int64_t>(q.tokens) / rows + q.count;
}

enum class Found { kRun, kNothing, kInvalid };

// The run of a slot, for a whole block.  Offsets that do not start at zero, decrease or do not
// end at the number of tokens make the call invalid.
__device__ __forceinline__ Found find_run(const Sequences& q, int64_t slot, int rows, int tid,
                                          Run* run) {
  if (q.offsets == nullptr) {
    const int tiles = (q.length + rows - 1) / rows;
    run->sequence = static_cast<int>(slot / tiles);
    run->tile = static_cast<int>(slot % tiles);
    run->length = q.length;
    run->batch = run->sequence;
    run->begin = 0;
    run->first = static_cast<int64_t>(run->sequence) * q.length;
    return Found::kRun;
  }
  int upto = 0, bad = 0;
  for (int base = 0; base < q.count; base += kThreads) {
    const int s = base + tid;
    bool below = false;
    if (s < q.count) {
      const int begin = q.offsets[s], end = q.offsets[s + 1];
      bad |= begin > end || (s == 0 && begin != 0) || (s == q.count - 1 && end != q.tokens);
      below = static_cast<int64_t>(begin / rows) + s <= slot;
    }
    upto += __syncthreads_count(below);
  }
  if (__syncthreads_or(bad)) return Found::kInvalid;
  run->sequence = __builtin_amdgcn_readfirstlane(upto - 1);
  const int begin = q.offsets[run->sequence];
  run->length = q.offsets[run->sequence + 1] - begin;
  run->tile = static_cast<int>(slot - (begin / rows + run->sequence));
  run->batch = 0;
  run->begin = begin;
  run->first = begin;
  return static_cast<int64_t>(run->tile) * rows < run->length ? Found::kRun : Found::kNothing;
}

// The slot of a sequence's first tile.
__device__ __forceinline__ int64_t first_slot(const Sequences& q, const Run& run, int rows) {
  return q.offsets == nullptr ? static_cast<int64_t>(run.sequence) * ((q.length + rows - 1) / rows)
                              : run.begin / rows + run.sequence;
}

// Blocks are handed to the XCDs in turn; neighbouring work items, which share keys, values or
// states, go to the same one: block b works on item (b mod 8) ceil(items / 8) + b / 8.
__host__ __device__ __forceinline__ int64_t grid_of(int64_t items) {
  return (items + kGroups - 1) / kGroups * kGroups;
}
__device__ __forceinline__ int64_t item_of_block(int64_t items) {
  const int64_t block = blockIdx.x;
  return block % kGroups * ((items + kGroups - 1) / kGroups) + block / kGroups;
}

// Rows [first, last) of a head of a contiguous [tokens, heads, width] tensor become NaN: what a
// call with invalid offsets returns.
template <typename T>
__device__ __forceinline__ void fill_nan(T* data, int64_t first, int64_t last, int heads, int head,
                                         int width, int tid) {
  if (data == nullptr) return;
  for (int64_t row = first; row < last; ++row)
    for (int d = tid; d < width; d += kThreads)
      data[(row * heads + head) * width + d] = static_cast<T>(__builtin_nanf(""));
}

// ---------------------------------------------------------------------------
// what the launches share
// ---------------------------------------------------------------------------

inline Sequences sequences_of(const rosa_mixer_problem& p) {
  return {p.cu_seqlens, p.cu_seqlens ? p.S : p.B, p.T, p.N};
}

template <typename T>
View<const T> view_of(const rosa_mixer_tensor& t) {
  return {static_cast<const T*>(t.data), t.batch_stride, t.token_stride, t.head_stride};
}

// rows of whole 16-byte pieces at 16-byte addresses
template <typename T>
bool whole_pieces(const rosa_mixer_tensor& t, int width) {
  const int64_t piece = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && width % piece == 0 &&
         t.batch_stride % piece == 0 && t.token_stride % piece == 0 && t.head_stride % piece == 0;
}

}  // namespace rosa_mixer
