// Device helpers shared by the decayed linear attention and the window attention kernels:
// matrix tiles in LDS, operands of the matrix instructions, and the map from blocks to
// sequences.
//
// Everything is built from one product, D[16 x 16] += A[16 x 32] B[32 x 16] in float32.  Lane
// l = 16 g + c of a wave holds A[c][8 g .. 8 g + 7], B[8 g .. 8 g + 7][c] and D[4 g + r][c],
// r = 0..3.  For the 16-bit types that is v_mfma_f32_16x16x32 (16 cycles).  A float32 operand is
// the sum of three bfloat16 ones, 2^-27 from it at most, and a product the six of their nine
// products that reach 2^-24 of it: 96 cycles, where the eight v_mfma_f32_16x16x4 that take
// float32 as it is need 256.  A kernel is written once for all three types.
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

struct SplitOperand {
  Frag<__bf16> part[3];  // falling by 2^-8 or more
};
template <typename T> using Operand = std::conditional_t<sizeof(T) == 4, SplitOperand, Frag<T>>;
// what tiles in LDS hold: one plane, or one for each part
template <typename T> using Stored = std::conditional_t<sizeof(T) == 4, __bf16, T>;
template <typename T> constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;

__device__ __forceinline__ f32x4 mma(const SplitOperand& a, const SplitOperand& b, f32x4 c) {
#pragma unroll
  for (int order = 2; order >= 0; --order)
#pragma unroll
    for (int i = 0; i <= order; ++i) c = mma(a.part[i], b.part[order - i], c);
  return c;
}

// N float32 as their parts
template <int N>
__device__ __forceinline__ void split(const float (&x)[N],
                                      __bf16 __attribute__((ext_vector_type(N))) (&part)[3]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float left = x[e];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      part[p][e] = static_cast<__bf16>(left);
      left -= static_cast<float>(part[p][e]);
    }
  }
}

// eight neighbouring elements as an operand
template <typename T>
__device__ __forceinline__ Operand<T> as_operand(Frag<T> x) {
  if constexpr (sizeof(T) == 4) {
    float values[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) values[e] = x[e];
    SplitOperand out;
    split<8>(values, out.part);
    return out;
  } else {
    return x;
  }
}

// c + the sums over the columns of an operand B, in every row
template <typename T>
__device__ __forceinline__ f32x4 add_sums(const Operand<T>& b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int p = 2; p >= 0; --p) c = mma(Frag<__bf16>(static_cast<__bf16>(1.0f)), b.part[p], c);
    return c;
  } else {
    return mma(Frag<T>(static_cast<T>(1.0f)), b, c);
  }
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

// Elements from one row of a tile to the next: 32 bytes more than the row, so that eight rows lie
// in eight different eighths of the 64 banks and both kinds of operand are read without bank
// conflicts (16 bytes: half of the LDS time of every kernel was conflicts).  The three planes of
// float32 tiles have room for 16.
template <typename T, int WIDTH> constexpr int kPitch = WIDTH + (sizeof(T) == 4 ? 8 : 16);
template <typename T, int ROWS, int WIDTH>
constexpr int kTileElements = kPlanes<T> * ROWS * kPitch<T, WIDTH>;

template <typename T>
__device__ __forceinline__ Frag<T> load8(const T* p) {
  return *reinterpret_cast<const Frag<T>*>(p);
}

// operand whose summed index runs along the row: row `row0 + c`, columns col0 + 8 g ...
template <typename T, int ROWS, int WIDTH>
__device__ __forceinline__ Operand<T> row_operand(const Stored<T>* tile, int row0, int col0, int lane) {
  const Stored<T>* at = tile + (row0 + (lane & 15)) * kPitch<T, WIDTH> + col0 + 8 * (lane >> 4);
  if constexpr (sizeof(T) == 4) {
    SplitOperand out;
#pragma unroll
    for (int p = 0; p < 3; ++p) out.part[p] = load8(at + p * ROWS * kPitch<T, WIDTH>);
    return out;
  } else {
    return load8(at);
  }
}

// operand whose summed index runs down the rows of the block [row0, row0 + 32): column col0 + c
template <typename T, int ROWS, int WIDTH>
__device__ __forceinline__ Operand<T> column_operand(const Stored<T>* tile, int row0, int col0, int lane) {
  // 16 lanes hand in four rows of 16 elements, 8 bytes each, and get a column each
  const Stored<T>* at = tile + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * kPitch<T, WIDTH> + col0 +
                        4 * (lane & 3);
  const auto read = [](const Stored<T>* from) {
    typedef __attribute__((address_space(3))) s16x4 LdsQuad;
    const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(from));
    const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(from + 16 * kPitch<T, WIDTH>));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<Stored<T>>, both);
  };
  if constexpr (sizeof(T) == 4) {
    SplitOperand out;
#pragma unroll
    for (int p = 0; p < 3; ++p) out.part[p] = read(at + p * ROWS * kPitch<T, WIDTH>);
    return out;
  } else {
    return read(at);
  }
}

// N neighbouring values of a row of a tile
template <typename T, int ROWS, int WIDTH, int N>
__device__ __forceinline__ void store_row(Stored<T>* tile, int row, int col, const float (&values)[N]) {
  typedef Stored<T> Part __attribute__((ext_vector_type(N)));
  Stored<T>* at = tile + row * kPitch<T, WIDTH> + col;
  if constexpr (sizeof(T) == 4) {
    Part part[3];
    split<N>(values, part);
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<Part*>(at + p * ROWS * kPitch<T, WIDTH>) = part[p];
  } else {
    Part rounded;
#pragma unroll
    for (int e = 0; e < N; ++e) rounded[e] = static_cast<T>(values[e]);
    *reinterpret_cast<Part*>(at) = rounded;
  }
}

// two results, rows [0, 16) and [16, 32) of the summed index, as the operand of the next product
template <typename T>
__device__ __forceinline__ Operand<T> operand_of(f32x4 low, f32x4 high) {
  if constexpr (sizeof(T) == 4) {
    const float values[8] = {low[0], low[1], low[2], low[3], high[0], high[1], high[2], high[3]};
    SplitOperand out;
    split<8>(values, out.part);
    return out;
  } else {
    Frag<T> out;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      out[r] = static_cast<T>(low[r]);
      out[r + 4] = static_cast<T>(high[r]);
    }
    return out;
  }
}

// Rows of a head in memory: `stride` elements apart from `base` on, the last of them number `last`.
template <typename T>
struct Rows {
  const T* base;
  int64_t stride;
  int last;
};

// `count` of them from number `first` on
template <typename T>
__device__ __forceinline__ Rows<T> rows_from(const Rows<T>& rows, int first, int count) {
  return {rows.base + first * rows.stride, rows.stride, count - 1};
}

// Where element `col` of a row lies.  WHOLE: the stride is below 2^24 bytes, so that a 32-bit
// offset from a base that the whole block shares is enough: no 64-bit arithmetic per load.
template <bool WHOLE, typename T>
__device__ __forceinline__ const T* place_of(const Rows<T>& rows, int row, int col) {
  if constexpr (WHOLE) {
    const uint32_t offset = __umul24(static_cast<uint32_t>(row),
                                     static_cast<uint32_t>(rows.stride) * static_cast<uint32_t>(sizeof(T))) +
                            static_cast<uint32_t>(col) * static_cast<uint32_t>(sizeof(T));
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(rows.base) + offset);
  } else {
    return rows.base + row * rows.stride + col;
  }
}

// A tile of ROWS x WIDTH on its way from memory to LDS through the registers of the block.  Rows
// that do not exist are the last one again (a caller masks what comes of it), so that loads are
// never predicated.  WHOLE: rows are whole 16-byte pieces at 16-byte addresses.
template <typename T, int ROWS, int WIDTH, bool WHOLE, int THREADS = kThreads>
struct TileMove {
  static constexpr int kElements = 16 / static_cast<int>(sizeof(T));
  static constexpr int kPerRow = WIDTH / kElements;
  static constexpr bool kSpare = ROWS * kPerRow < THREADS;  // threads without a piece
  static constexpr int kPieces = kSpare ? 1 : ROWS * kPerRow / THREADS;
  static_assert(kSpare || ROWS * kPerRow % THREADS == 0, "tiles are moved in whole pieces per thread");
  typedef T Piece __attribute__((ext_vector_type(kElements)));

  Piece held[kPieces];

  static __device__ __forceinline__ int row_of(int i, int tid) {
    return i * (THREADS / kPerRow) + tid / kPerRow;
  }
  static __device__ __forceinline__ int col_of(int tid) { return tid % kPerRow * kElements; }

  // `place(row, col)`: the address of an element
  template <typename Place>
  __device__ __forceinline__ void fetch_from(Place&& place, int width, int tid) {
    const int col = col_of(tid);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i, tid);
      if constexpr (WHOLE) {
        held[i] = *reinterpret_cast<const Piece*>(place(row, min(col, width - kElements)));
      } else {
        const T* from = place(row, 0);
#pragma unroll
        for (int e = 0; e < kElements; ++e) held[i][e] = from[min(col + e, width - 1)];
      }
    }
  }

  __device__ __forceinline__ void fetch(const Rows<T>& rows, int width, int tid) {
    fetch_from([&](int row, int col) { return place_of<WHOLE>(rows, min(row, rows.last), col); }, width,
               tid);
  }

  // Columns from `width` on become zeros here, not where the loads were issued: touching a loaded
  // register there would wait for it.
  __device__ __forceinline__ void clear_padding(int width, int tid) {
    if (width >= WIDTH) return;  // (a branch of the whole block; selects would cost every full tile)
    const int col = col_of(tid);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if constexpr (WHOLE) {  // all of a piece or nothing
        held[i] = col < width ? held[i] : Piece(static_cast<T>(0.0f));
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e)
          held[i][e] = col + e < width ? held[i][e] : static_cast<T>(0.0f);
      }
    }
  }

  // row r of a walk that runs backwards over `flip` rows of memory
  static __device__ __forceinline__ int walk_row(int row, int flip) {
    return row < flip ? flip - 1 - row : row;
  }

  static __device__ __forceinline__ bool holds(int tid) { return !kSpare || row_of(0, tid) < ROWS; }

  __device__ __forceinline__ void store(Stored<T>* tile, int width, int tid, int flip = 0) {
    clear_padding(width, tid);
    if (!holds(tid)) return;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = walk_row(row_of(i, tid), flip);
      if constexpr (sizeof(T) == 4) {
        const float values[4] = {held[i][0], held[i][1], held[i][2], held[i][3]};
        store_row<T, ROWS, WIDTH, 4>(tile, row, col_of(tid), values);
      } else {
        *reinterpret_cast<Piece*>(tile + row * kPitch<T, WIDTH> + col_of(tid)) = held[i];
      }
    }
  }
};

// row-wise operand straight from memory, of the lane's own row; columns from `width` on are some
// other elements of it until clear_operand
template <bool WHOLE, typename T>
__device__ __forceinline__ Frag<T> memory_operand(const Rows<T>& rows, int row, int col, int width) {
  Frag<T> out;
  row = min(row, rows.last);
  if constexpr (WHOLE && sizeof(T) == 2) {
    out = load8(place_of<WHOLE>(rows, row, min(col, width - 8)));
  } else if constexpr (WHOLE) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const f32x4 part =
          *reinterpret_cast<const f32x4*>(place_of<WHOLE>(rows, row, min(col + 4 * half, width - 4)));
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * half + e] = part[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = *place_of<WHOLE>(rows, row, min(col + e, width - 1));
  }
  return out;
}

// operand of columns [col0, col0 + 32)
template <bool WHOLE, typename T>
__device__ __forceinline__ void clear_operand(Frag<T>& operand, int col0, int group, int width) {
  if (width >= col0 + 32) return;
  const int col = col0 + 8 * group;
  if constexpr (WHOLE && sizeof(T) == 2) {  // all or nothing
    operand = col < width ? operand : Frag<T>(static_cast<T>(0.0f));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) operand[e] = col + e < width ? operand[e] : static_cast<T>(0.0f);
  }
}

// four neighbouring elements of a contiguous output row; `quads`: it is whole quads at their addresses
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

// float16 has few exponents (see lift_of)
template <typename T> constexpr bool kNarrow = std::is_same_v<T, _Float16>;

// A result of TILES tiles of 16 columns, times `by`, to a row of an output.  Where rows are whole
// 16-byte pieces of 16-bit elements, the lanes of a column exchange their quads of two neighbouring
// tiles: each has a whole piece then, and a store fills 64 bytes of a row instead of 32.  The
// products are rounded to float32 first in either form (left to itself the compiler makes one
// float16 instruction of product and rounding in one of them, and strides would change results).
// STREAM: past the caches, which keeps what other blocks are about to read in them.
template <bool WHOLE, bool STREAM, typename T, int TILES>
__device__ __forceinline__ void store_tiles(T* row, const f32x4 (&value)[TILES], float by, int group,
                                            int width) {
  f32x4 scaled[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float product = value[t][e] * by;
      if constexpr (kNarrow<T>) asm("" : "+v"(product));
      scaled[t][e] = product;
    }
  if constexpr (WHOLE && sizeof(T) == 2) {
    static_assert(TILES % 2 == 0, "tiles are stored in pairs");
    const int col = (group & 1) * 16 + (group >> 1) * 8;
#pragma unroll
    for (int t = 0; t < TILES; t += 2) {
      typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      Quad<T> quad[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) quad[h][e] = static_cast<T>(scaled[t + h][e]);
      const u32x2 low = __builtin_bit_cast(u32x2, quad[0]), high = __builtin_bit_cast(u32x2, quad[1]);
      u32x4 piece;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto swapped = __builtin_amdgcn_permlane16_swap(low[e], high[e], false, false);
        piece[e] = swapped[0];
        piece[2 + e] = swapped[1];
      }
      if (t * 16 + col < width) {
        u32x4* to = reinterpret_cast<u32x4*>(row + t * 16 + col);
        if constexpr (STREAM)
          __builtin_nontemporal_store(piece, to);
        else
          *to = piece;
      }
    }
  } else {
    const bool quads = WHOLE || (width % 4 == 0 && reinterpret_cast<uintptr_t>(row) % sizeof(Quad<T>) == 0);
#pragma unroll
    for (int t = 0; t < TILES; ++t) store4(row, t * 16 + 4 * group, scaled[t], width, quads);
  }
}

// The power of two that brings a largest value into float16's upper range, [2^13, 2^14): float16
// has few exponents, and what is rounded to it loses bits below 2^-14 and everything above 2^16.
// The other types take values as they are.  At most 2^60: what stays below 2^-47 then keeps steps
// of 2^-84 and less, far below what a float16 result shows, and neither the factor (the logarithm of
// a subnormal number is -inf) nor a sum times it passes float32's range.
constexpr float kMostLift = 60.0f;
__device__ __forceinline__ float lift_of(float largest) {
  return largest > 0.0f && largest < __builtin_inff()
             ? exp2_of(fminf(13.0f - floorf(log2_of(largest)), kMostLift))
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
  // `count` tokens from `token` on
  __device__ __forceinline__ Rows<std::remove_const_t<T>> rows(int64_t batch, int64_t token, int head,
                                                               int count, int col = 0) const {
    return {row(batch, token, head) + col, token_stride, count - 1};
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
__host__ __device__ __forceinline__ int tiles_of(int length, int rows) {
  return length > 0 ? (length - 1) / rows + 1 : 0;  // (length + rows may pass 32 bits)
}
__host__ __device__ __forceinline__ int64_t slots_of(const Sequences& q, int rows) {
  return q.offsets == nullptr ? static_cast<int64_t>(q.count) * tiles_of(q.length, rows)
                              : static_cast<int64_t>(q.tokens) / rows + q.count;
}

enum class Found { kRun, kNothing, kInvalid };

// The run of a slot, for a whole block.  Offsets that do not start at zero, decrease or do not
// end at the number of tokens make the call invalid.
template <int THREADS = kThreads>
__device__ __forceinline__ Found find_run(const Sequences& q, int64_t slot, int rows, int tid,
                                          Run* run) {
  if (q.offsets == nullptr) {
    const int tiles = tiles_of(q.length, rows);
    run->sequence = static_cast<int>(slot / tiles);
    run->tile = static_cast<int>(slot % tiles);
    run->length = q.length;
    run->batch = run->sequence;
    run->begin = 0;
    run->first = static_cast<int64_t>(run->sequence) * q.length;
    return Found::kRun;
  }
  // How many sequences begin at this slot or before it: with one a thread a count of the block, with
  // more a sum, so that all loads are under way at once (16 rounds with a barrier each made 4096
  // sequences of 16 tokens five times as long).
  int upto = 0, bad = 0;
  const auto look_at = [&](int s) {
    const int begin = q.offsets[s], end = q.offsets[s + 1];
    bad |= begin > end || (s == 0 && begin != 0) || (s == q.count - 1 && end != q.tokens);
    return static_cast<int64_t>(begin / rows) + s <= slot ? 1 : 0;
  };
  if (q.count <= THREADS) {
    upto = __syncthreads_count(tid < q.count ? look_at(tid) : 0);
  } else {
    __shared__ int total;
    if (tid == 0) total = 0;
#pragma unroll 4
    for (int s = tid; s < q.count; s += THREADS) upto += look_at(s);
    __syncthreads();
    atomicAdd(&total, upto);
    __syncthreads();
    upto = total;
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

// The whole of a sequence; of length -1 where its offsets do not lie among the tokens.
__device__ __forceinline__ Run run_of_sequence(const Sequences& q, int sequence) {
  if (q.offsets == nullptr)
    return {sequence, q.length, 0, sequence, 0, static_cast<int64_t>(sequence) * q.length};
  const int begin = q.offsets[sequence], end = q.offsets[sequence + 1];
  return {sequence, begin < 0 || end < begin || end > q.tokens ? -1 : end - begin, 0, 0, begin, begin};
}

// The slot of a sequence's first tile.
__device__ __forceinline__ int64_t first_slot(const Sequences& q, const Run& run, int rows) {
  return q.offsets == nullptr ? static_cast<int64_t>(run.sequence) * tiles_of(q.length, rows)
                              : run.begin / rows + run.sequence;
}

// A launch has less than 2^32 threads in a dimension, and drops the others without an error: grids of
// more blocks than a row holds go on in further rows (the decay's backward has 2^32 threads at 1.4
// million sequences times heads of 128 columns).  Blocks behind the last item have nothing to do.
constexpr int kGridRow = 1 << 22;
inline dim3 grid_of(int64_t blocks) {
  return blocks <= kGridRow ? dim3(static_cast<unsigned>(blocks))
                            : dim3(kGridRow, static_cast<unsigned>((blocks + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ uint32_t block_number() { return blockIdx.y * kGridRow + blockIdx.x; }

// Blocks are handed to the XCDs in turn; neighbouring work items, which share keys, values or
// states, go to the same one: block b works on item (b mod 8) ceil(items / 8) + b / 8.
inline dim3 grid_of_items(int64_t items) { return grid_of((items + kGroups - 1) / kGroups * kGroups); }
__device__ __forceinline__ int64_t item_of_block(int64_t items) {
  const uint32_t block = block_number(), share = static_cast<uint32_t>((items + kGroups - 1) / kGroups);
  return block / kGroups < share ? static_cast<int64_t>(block % kGroups) * share + block / kGroups : items;
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

// rows of whole 16-byte pieces at 16-byte addresses, less than 2^24 bytes apart
inline bool whole_address(const void* data) { return reinterpret_cast<uintptr_t>(data) % 16 == 0; }
template <typename T>
bool whole_stride(int64_t stride) {
  return stride >= 0 && stride < (1 << 24) / static_cast<int64_t>(sizeof(T));
}
template <typename T>
bool whole_pieces(const rosa_mixer_tensor& t, int width) {
  const int64_t piece = 16 / sizeof(T);
  return whole_address(t.data) && width % piece == 0 &&
         t.batch_stride % piece == 0 && t.token_stride % piece == 0 && t.head_stride % piece == 0 &&
         whole_stride<T>(t.token_stride);
}

}  // namespace rosa_mixer
