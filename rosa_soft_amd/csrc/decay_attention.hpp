// Linear attention with a decay for each head.
//
//   S_t = lambda S_{t-1} + k_t v_t^T,   o_t = scale q_t^T S_t
//
// A chunk of 64 tokens that starts from the state S is three products (i, j inside the chunk):
//   o_i = scale (lambda^(i+1) q_i^T S + sum_{j<=i} lambda^(i-j) (q_i . k_j) v_j)
//   S'  = lambda^64 S + sum_j lambda^(63-j) k_j v_j^T
// so a block walks its sequence chunk by chunk with the state in the registers of four of its
// waves: one pass over the data, no state in memory.
//
// The gradients are the same operator on other operands, two of them from the last token to the
// first:  dq = F(dO, v, k),  dv = F_reversed(k, q, dO),  dk = F_reversed(v, dO, q).
#pragma once

#include "mixer_calls.hpp"
#include "mixer_device.hpp"

namespace rosa_mixer {

constexpr int kChunk = 64;

template <typename T>
struct DecayPass {
  View<const T> query, key, value;
  int query_share, key_share, value_share;  // heads of the call to one head of the tensor
  int key_width, value_width;
  T* out;                                    // [tokens][H][value_width]
  float* partial;                            // instead of it: before the sum over shared heads
  bool reverse;
};

template <typename T>
struct DecayArgs {
  DecayPass<T> pass[3];
  int passes, heads, slices, segment;        // slices of all passes together
  int64_t slots, items;
  Sequences sequences;
  const float* log_decay;
  float scale;
  float* segment_states;                     // [pass][slot][head][key_width][value_width] or null
  const float* state_in;                     // [sequence][head][key_width][value_width] or null
  float* state_out;
};

// Terms of a value times its weight in the state's sum.  The state is a float32 sum, so its
// bfloat16 operands are split: three terms where the state itself is an answer (2^-25 relative),
// fewer where it is only read again through 16-bit operands.
template <typename T>
using StateType = std::conditional_t<sizeof(T) == 4, float, __bf16>;

template <typename T, int WIDTH, bool STATE_ONLY, bool WHOLE>
constexpr int kDecayWaves = STATE_ONLY || sizeof(T) == 4 || !WHOLE ? 2 : 4;

// Four waves take the outputs of 16 tokens each, four others the state, between the same barriers:
// neither holds the registers of the other, and what one waits for the other fills.  Summing
// states alone takes four waves.
//
// Values are cut into slices of 64 columns, each with its part of the state (128 x 64 float32 are
// 32 registers of four waves), rounded to the inputs' type once a chunk as the operand of the
// queries' product.  Rounded so too: the scores; weighted values by TERMS.  Measured in bfloat16,
// 2 x 4096 tokens, 32 heads of 128: 72 us forward, 303 MB in and out of HBM at 4.2 TB/s (and 31 and
// 8 us for the segments' states), 210 us for the three passes of the backward, 761 MB at 3.6 TB/s;
// a large copy reaches 4.9.  What bounds it besides: a chunk takes a block 2.5 us alone on its
// compute unit and two of them 4.1, of which no part is more than a sixth; left out one at a
// time, of 154 us (mean of both directions): loads 24, stores 21, scores 14, the state's products
// 14, the queries' 10, weighted values 9, rounded state 8.
template <bool STATE_ONLY> constexpr int kDecayThreads = STATE_ONLY ? kThreads : 2 * kThreads;

template <typename T, int WIDTH, int SLICE, int TERMS, bool STATE_ONLY, bool WHOLE>
__global__ __launch_bounds__(kDecayThreads<STATE_ONLY>)
    __attribute__((amdgpu_waves_per_eu(kDecayWaves<T, WIDTH, STATE_ONLY, WHOLE>))) void
    decay_chunks_kernel(DecayArgs<T> a) {
  using ST = StateType<T>;
  constexpr int kBlock = kDecayThreads<STATE_ONLY>;
  constexpr int kColTiles = SLICE / 16;
  constexpr int kTiles = WIDTH / 16 * kColTiles / 4;   // state tiles of a wave
  constexpr int kWaveCols = kTiles < kColTiles ? kTiles : kColTiles;
  constexpr int kWaveRows = kTiles / kWaveCols;
  constexpr int kSteps = WIDTH / 32;

  constexpr int kTerm = kTileElements<ST, kChunk, SLICE>;  // of the weighted values
  __shared__ __attribute__((aligned(16))) Stored<T> keys[kTileElements<T, kChunk, WIDTH>];
  __shared__ __attribute__((aligned(16))) Stored<T> values[STATE_ONLY ? 16 : kTileElements<T, kChunk, SLICE>];
  __shared__ __attribute__((aligned(16))) Stored<ST> weighted[TERMS * kTerm];
  __shared__ __attribute__((aligned(16))) Stored<T> state_rows[STATE_ONLY ? 16 : kTileElements<T, SLICE, WIDTH>];
  __shared__ float largest[4];

  const int64_t item = item_of_block(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int place = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = place & 3;  // of those with the same task
  // Neighbours on one XCD, whose cache they share: the slices of a sequence, which read the same
  // keys and queries, then the passes, which read the same four tensors.
  // No item is empty for its pass alone: workgroups go round the shader engines of an XCD in turn,
  // and empty ones in a regular pattern leave some engines twice the work of others.
  int slice = static_cast<int>(item % a.slices), pass_index = 0;
  for (; pass_index + 1 < a.passes; ++pass_index) {
    const int slices = (a.pass[pass_index].value_width + SLICE - 1) / SLICE;
    if (slice < slices) break;
    slice -= slices;
  }
  const int64_t slot = item / a.slices % a.slots;
  const int head = static_cast<int>(item / a.slices / a.slots);
  const DecayPass<T>& p = a.pass[pass_index];
  const int col0 = slice * SLICE;

  Run run;
  const Found found = find_run<kBlock>(a.sequences, slot, a.segment, tid, &run);
  const int64_t state_size = static_cast<int64_t>(p.key_width) * p.value_width;
  if (found != Found::kRun) {
    if constexpr (!STATE_ONLY) {
      if (found == Found::kInvalid) {  // no offset can be relied on: everything is NaN
        const int64_t first = slot * a.segment;
        const int64_t last = min(first + a.segment, static_cast<int64_t>(a.sequences.tokens));
        if (slice == 0) {
          fill_nan(p.partial ? nullptr : p.out, first, last, a.heads, head, p.value_width, tid);
          fill_nan(p.partial, first, last, a.heads, head, p.value_width, tid);
        }
      }
      // a slot without new tokens keeps its state
      const int64_t kept = found == Found::kInvalid ? slot : run.length == 0 ? run.sequence : -1;
      if (slice == 0 && a.state_out != a.state_in && kept >= 0 && kept < a.sequences.count &&
          (found == Found::kInvalid || run.tile == 0)) {
        const int64_t at = (kept * a.heads + head) * state_size;
        for (int64_t e = tid; e < state_size; e += kBlock) a.state_out[at + e] = a.state_in[at + e];
      }
    }
    return;
  }
  const int start = run.tile * a.segment;                       // in the order of the walk
  const int stop = start + min(a.segment, run.length - start);
  if (STATE_ONLY && stop == run.length) return;                 // nothing follows this segment
  const float rate = a.log_decay[head] * 1.4426950408889634f;

  const int query_head = head / p.query_share, key_head = head / p.key_share,
            value_head = head / p.value_share;
  const Rows<T> key_rows = p.key.rows(run.batch, run.begin, key_head, run.length),
                value_rows = p.value.rows(run.batch, run.begin, value_head, run.length, col0);
  TileMove<T, kChunk, WIDTH, WHOLE, kBlock> key_move;
  TileMove<T, kChunk, SLICE, WHOLE, kBlock> value_move;
  // the tokens of the chunk at `at` as they lie in memory
  const auto fill_of = [&](int at) { return min(kChunk, stop - at); };
  const auto first_of = [&](int at, int fill) { return p.reverse ? run.length - at - fill : at; };
  const auto fetch = [&](int at) {
    const int fill = fill_of(at), first = first_of(at, fill);
    key_move.fetch(rows_from(key_rows, first, fill), p.key_width, tid);
    value_move.fetch(rows_from(value_rows, first, fill), p.value_width - col0, tid);
  };
  fetch(start);
  // what a row of values counts for in the state behind a whole chunk
  float whole_chunk[value_move.kPieces];
#pragma unroll
  for (int i = 0; i < value_move.kPieces; ++i)
    whole_chunk[i] = power_of(
        rate, kChunk - 1 - value_move.walk_row(value_move.row_of(i, tid), p.reverse ? kChunk : 0));

  // keys, values and weighted values of a chunk go to LDS
  const auto store_tiles_of = [&](int fill) {
    const int flip = p.reverse ? fill : 0;
    key_move.store(keys, p.key_width, tid, flip);
    if constexpr (!STATE_ONLY)
      value_move.store(values, p.value_width - col0, tid, flip);
    else
      value_move.clear_padding(p.value_width - col0, tid);
    if (!value_move.holds(tid)) return;
#pragma unroll
    for (int i = 0; i < value_move.kPieces; ++i) {
      constexpr int kElements = value_move.kElements;
      const int row = value_move.walk_row(value_move.row_of(i, tid), flip);
      float by = whole_chunk[i];
      if (fill < kChunk) by = row < fill ? power_of(rate, fill - 1 - row) : 0.0f;
      float left[kElements];
#pragma unroll
      for (int e = 0; e < kElements; ++e) left[e] = static_cast<float>(value_move.held[i][e]) * by;
      if constexpr (sizeof(T) == 4) {
        store_row<ST, kChunk, SLICE>(weighted, row, value_move.col_of(tid), left);
      } else {
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          typedef ST Piece __attribute__((ext_vector_type(kElements)));
          Piece term;
#pragma unroll
          for (int e = 0; e < kElements; ++e) {
            term[e] = static_cast<ST>(left[e]);
            left[e] -= static_cast<float>(term[e]);
          }
          *reinterpret_cast<Piece*>(weighted + t * kTerm + row * kPitch<ST, SLICE> + value_move.col_of(tid)) = term;
        }
      }
    }
  };
  // float16: brings the rounded state into range
  const auto unit_of_state = [&] {
    return lift_of(fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3])));
  };

  if (!STATE_ONLY && place < 4) {
    // Weights of a token's scores, scale lambda^(i - j): of the tile of 16 keys that its own tile
    // is, and of the tile before it, from which the ones before that are powers of lambda^16 away.
    const int own = wave * 16 + column;
    float diagonal[4], before[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int apart = column - 4 * group - r;
      diagonal[r] = apart >= 0 ? a.scale * power_of(rate, apart) : 0.0f;
      before[r] = a.scale * power_of(rate, 16 + apart);
    }
    const float carry = a.scale * power_of(rate, own + 1);
    const float tile_rate = power_of(rate, 16);

    const Rows<T> query_rows = p.query.rows(run.batch, run.begin, query_head, run.length);
    Frag<T> next_query[kSteps];
    const auto fetch_query = [&](int at) {
      const int fill = fill_of(at);
      const Rows<T> queries = rows_from(query_rows, first_of(at, fill), fill);
      const int row = p.reverse ? max(fill - 1 - own, 0) : own;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        next_query[s] = memory_operand<WHOLE>(queries, row, s * 32 + 8 * group, p.key_width);
    };
    fetch_query(start);

    if constexpr (kNarrow<T>) __syncthreads();

    for (int at = start; at < stop; at += kChunk) {
      const int fill = fill_of(at);
      store_tiles_of(fill);
      const float unit = kNarrow<T> ? unit_of_state() : 1.0f;
      Operand<T> query[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        clear_operand<WHOLE>(next_query[s], s * 32, group, p.key_width);
        query[s] = as_operand<T>(next_query[s]);
      }
      __syncthreads();
      if (at + kChunk < stop) {
        fetch(at + kChunk);
        fetch_query(at + kChunk);
      }
      if (wave * 16 < fill) {
        // outputs transposed: rows are value columns, columns are this wave's 16 tokens
        f32x4 out[kColTiles];
#pragma unroll
        for (int t = 0; t < kColTiles; ++t) out[t] = f32x4(0.0f);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int t = 0; t < kColTiles; ++t)
            out[t] = mma(row_operand<T, SLICE, WIDTH>(state_rows, t * 16, s * 32, lane), query[s], out[t]);
        // (only tiles of earlier keys: with all four for every wave, and no branches, 7 % longer)
        f32x4 score[4];
        float step = 1.0f;  // lambda^16 for every tile further back
#pragma unroll
        for (int t = 3; t >= 0; --t) {
          score[t] = f32x4(0.0f);
          if (t <= wave) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
              score[t] = mma(row_operand<T, kChunk, WIDTH>(keys, t * 16, s * 32, lane), query[s], score[t]);
            if (t == wave) {
#pragma unroll
              for (int r = 0; r < 4; ++r)  // (a select, so that later keys never reach a token)
                score[t][r] = 4 * group + r <= column ? score[t][r] * diagonal[r] : 0.0f;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) score[t][r] *= before[r] * step;
              step *= tile_rate;
            }
          }
        }
        float carried = carry;
        float range = 1.0f;  // float16: the same for the scores of a token
        if constexpr (kNarrow<T>) {
          float most = 0.0f;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(score[t][r]));
          range = lift_of(over_groups_max(most));
#pragma unroll
          for (int t = 0; t < 4; ++t) score[t] *= range;
          carried = carried * range / unit;  // (range / unit may pass float32's range)
        }
#pragma unroll
        for (int t = 0; t < kColTiles; ++t) out[t] *= carried;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (2 * half <= wave) {
            const Operand<T> scores = operand_of<T>(score[2 * half], score[2 * half + 1]);
#pragma unroll
            for (int t = 0; t < kColTiles; ++t)
              out[t] = mma(column_operand<T, kChunk, SLICE>(values, half * 32, t * 16, lane), scores, out[t]);
          }
        }
        const int i = at + own;  // the walk's token
        if (i < stop) {
          const int64_t row =
              ((run.first + (p.reverse ? run.length - 1 - i : i)) * a.heads + head) * p.value_width + col0;
          // (streamed: prompts 93 -> 88 us; the window kernels, whose blocks share more, lose 1 %)
          if (p.partial != nullptr)
            store_tiles<WHOLE, true>(p.partial + row, out, 1.0f / range, group, p.value_width - col0);
          else
            store_tiles<WHOLE, true>(p.out + row, out, 1.0f / range, group, p.value_width - col0);
        }
      }
      __syncthreads();
    }
    return;
  }

  // state rows (key columns) and columns (value columns) of this wave's tiles
  const int row_tile = wave * kTiles / kColTiles, col_tile = wave * kTiles % kColTiles;
  f32x4 state[kWaveRows][kWaveCols];
  const float* from = nullptr;
  if (!STATE_ONLY && a.segment_states != nullptr && (run.tile > 0 || a.state_in != nullptr))
    from = a.segment_states + ((pass_index * a.slots + slot) * a.heads + head) * state_size;
  else if (!STATE_ONLY && a.segment_states == nullptr && a.state_in != nullptr)
    from = a.state_in + (static_cast<int64_t>(run.sequence) * a.heads + head) * state_size;
#pragma unroll
  for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
    for (int j = 0; j < kWaveCols; ++j) state[i][j] = f32x4(0.0f);
  if (from != nullptr) {
    const int last_row = p.key_width - 1, last_col = p.value_width - 1;
#pragma unroll
    for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
      for (int j = 0; j < kWaveCols; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = (row_tile + i) * 16 + 4 * group + r, col = col0 + (col_tile + j) * 16 + column;
          const float value = from[min(row, last_row) * p.value_width + min(col, last_col)];
          state[i][j][r] = row <= last_row && col <= last_col ? value : 0.0f;
        }
  }
  const auto note_largest = [&] {
    if constexpr (kNarrow<T> && !STATE_ONLY) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
        for (int j = 0; j < kWaveCols; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(state[i][j][r]));
      for (int apart = 1; apart < 64; apart *= 2) most = fmaxf(most, __shfl_xor(most, apart));
      if (lane == 0) largest[wave] = most;
    }
  };
  note_largest();
  if constexpr (kNarrow<T> && !STATE_ONLY) __syncthreads();

  for (int at = start; at < stop; at += kChunk) {
    const int fill = fill_of(at);
    store_tiles_of(fill);
    if constexpr (!STATE_ONLY) {
      const float unit = kNarrow<T> ? unit_of_state() : 1.0f;
#pragma unroll
      for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
        for (int j = 0; j < kWaveCols; ++j) {
          float rounded[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) rounded[r] = state[i][j][r] * unit;
          store_row<T, SLICE, WIDTH>(state_rows, (col_tile + j) * 16 + column, (row_tile + i) * 16 + 4 * group,
                                     rounded);
        }
    }
    __syncthreads();
    if (at + kChunk < stop) fetch(at + kChunk);

    // the state behind the chunk
    const float decay = power_of(rate, fill);
#pragma unroll
    for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
      for (int j = 0; j < kWaveCols; ++j) state[i][j] *= decay;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 32 >= fill) break;
      // (a float16 key is the sum of two bfloat16)
      constexpr bool kPair = std::is_same_v<T, _Float16>;
      std::conditional_t<kPair, Frag<__bf16>, Operand<T>> key[kWaveRows], low[kPair ? kWaveRows : 1];
#pragma unroll
      for (int i = 0; i < kWaveRows; ++i) {
        const Operand<T> read = column_operand<T, kChunk, WIDTH>(keys, half * 32, (row_tile + i) * 16, lane);
        if constexpr (kPair) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            key[i][e] = static_cast<__bf16>(static_cast<float>(read[e]));
            low[i][e] = static_cast<__bf16>(static_cast<float>(read[e]) - static_cast<float>(key[i][e]));
          }
        } else {
          key[i] = read;
        }
      }
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int j = 0; j < kWaveCols; ++j) {
          const Operand<ST> value = column_operand<ST, kChunk, SLICE>(weighted + t * kTerm, half * 32,
                                                                      (col_tile + j) * 16, lane);
#pragma unroll
          for (int i = 0; i < kWaveRows; ++i) {
            state[i][j] = mma(key[i], value, state[i][j]);
            if constexpr (kPair)
              if (t == 0 || t + 1 < TERMS) state[i][j] = mma(low[i], value, state[i][j]);
          }
        }
    }
    note_largest();
    __syncthreads();
  }

  float* to = nullptr;
  if (STATE_ONLY)
    to = a.segment_states + ((pass_index * a.slots + slot) * a.heads + head) * state_size;
  else if (a.state_out != nullptr && stop == run.length)
    to = a.state_out + (static_cast<int64_t>(run.sequence) * a.heads + head) * state_size;
  if (to != nullptr) {
#pragma unroll
    for (int i = 0; i < kWaveRows; ++i)
#pragma unroll
      for (int j = 0; j < kWaveCols; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = (row_tile + i) * 16 + 4 * group + r, col = col0 + (col_tile + j) * 16 + column;
          if (row < p.key_width && col < p.value_width)
            to[static_cast<int64_t>(row) * p.value_width + col] = state[i][j][r];
        }
  }
}

// What every segment starts from: the segments' own sums, in their place, become the states before
// them, in the order of the segments; what a sequence starts from is only written where that is a
// given state (it may be overwritten by the last segment while the first still reads it).
// kPieceElements elements of a state to a block: 30 MB in and out in 8 us (2 x 4096 tokens, 32
// heads of 128, four segments).  Offsets are only looked at as far as this block's accesses go; the
// walk itself refuses the others.
constexpr int kPieceElements = 4 * kThreads;
template <typename T>
__global__ __launch_bounds__(kThreads) void decay_join_kernel(DecayArgs<T> a, int64_t state_size) {
  const uint32_t block = block_number();
  const uint32_t pieces = static_cast<uint32_t>((state_size + kPieceElements - 1) / kPieceElements),
                 row = block / pieces;
  const int head = static_cast<int>(row % a.heads);
  const int pass_index = static_cast<int>(row / a.heads % a.passes);
  const int sequence = static_cast<int>(row / a.heads / a.passes);
  if (sequence >= a.sequences.count) return;
  const Run run = run_of_sequence(a.sequences, sequence);
  const int segments = tiles_of(run.length, a.segment);  // (of length -1: no offsets to rely on)
  if (segments < (a.state_in == nullptr ? 2 : 1)) return;
  const int64_t slot = first_slot(a.sequences, run, a.segment);
  const float decay = power_of(a.log_decay[head] * 1.4426950408889634f, a.segment);
  const int64_t step = a.heads * state_size;
  constexpr int kAhead = 4;  // loads under way: a load behind each store took 16 us for 53 segments
  const int64_t begin = static_cast<int64_t>(block % pieces) * kPieceElements;
  const int64_t end = min(begin + kPieceElements, state_size);
  for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
    float state = a.state_in == nullptr
                      ? 0.0f
                      : a.state_in[(static_cast<int64_t>(sequence) * a.heads + head) * state_size + e];
    float* at = a.segment_states + ((pass_index * a.slots + slot) * a.heads + head) * state_size + e;
    for (int first = 0; first < segments; first += kAhead) {
      float own[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
        own[s] = first + s + 1 < segments ? at[(first + s) * step] : 0.0f;
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (first + s >= segments) break;
        at[(first + s) * step] = state;
        state = decay * state + own[s];
      }
    }
  }
}

// Gradients of a head of keys or values shared by `share` query heads: their sum, in order.  (Bound
// by the reads of the float32 parts.)
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_shared_kernel(const float* partial, T* out,
                                                              int64_t rows, int share, int width) {
  const int64_t e = static_cast<int64_t>(block_number()) * kThreads + threadIdx.x;
  if (e >= rows * width) return;
  const int64_t row = e / width, col = e % width;
  float sum = 0.0f;
  for (int s = 0; s < share; ++s) sum += partial[(row * share + s) * width + col];
  out[e] = static_cast<T>(sum);
}

// ---------------------------------------------------------------------------
// one token: the state is read, advanced, applied and written, once
// ---------------------------------------------------------------------------

template <typename T>
struct DecayTokenArgs {
  View<const T> query, key, value;
  const float* log_decay;
  const float* state_in;
  float* state_out;
  T* out;
  int slots, heads, share, key_width, value_width, slice;  // value columns of a block
  float scale;
};

// VEC neighbouring columns per thread, the rows dealt out to the threads that are left.  64 slots
// with 32 states of 128 x 128: 268 MB in and out in 50 us, 5.4 TB/s.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void decay_token_kernel(DecayTokenArgs<T> a) {
  __shared__ float query[kMostWidth], key[kMostWidth];
  __shared__ float sums[kThreads * VEC];
  const int tid = threadIdx.x;
  const int slices = (a.value_width + a.slice - 1) / a.slice;
  const uint32_t block = block_number();
  const int col0 = block % slices * a.slice;
  const int head = block / slices % a.heads, batch = block / slices / a.heads;
  if (batch >= a.slots) return;
  const int columns = min(a.slice, a.value_width - col0);
  if (tid < a.key_width) {
    query[tid] = static_cast<float>(a.query.row(batch, 0, head)[tid]);
    key[tid] = static_cast<float>(a.key.row(batch, 0, head / a.share)[tid]);
  }
  const int across = a.slice / VEC, rows = kThreads / across;
  const int col = tid % across * VEC, row0 = tid / across;
  const bool there = col < columns && row0 < rows;
  float value[VEC], sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    value[e] = there ? static_cast<float>(a.value.row(batch, 0, head / a.share)[col0 + col + e]) : 0.0f;
    sum[e] = 0.0f;
  }
  const float decay = power_of(a.log_decay[head] * 1.4426950408889634f, 1);
  __syncthreads();
  typedef float Piece __attribute__((ext_vector_type(VEC)));
  const int64_t at = (static_cast<int64_t>(batch) * a.heads + head) * a.key_width * a.value_width +
                     col0 + col;
  if (there) {
#pragma unroll 4
    for (int d = row0; d < a.key_width; d += rows) {
      const int64_t place = at + static_cast<int64_t>(d) * a.value_width;
      Piece state = *reinterpret_cast<const Piece*>(a.state_in + place);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        state[e] = decay * state[e] + key[d] * value[e];
        sum[e] += query[d] * state[e];
      }
      *reinterpret_cast<Piece*>(a.state_out + place) = state;
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[tid * VEC + e] = sum[e];
  __syncthreads();
  for (int c = tid; c < columns; c += kThreads) {
    float total = 0.0f;
    for (int r = 0; r < rows; ++r) total += sums[r * across * VEC + c];
    a.out[(static_cast<int64_t>(batch) * a.heads + head) * a.value_width + col0 + c] =
        static_cast<T>(total * a.scale);
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T, int WIDTH, int TERMS, bool WHOLE>
void decay_walk(DecayArgs<T>& args, const DecayPlan& plan, hipStream_t stream) {
  constexpr int kSlice = decay_slice(WIDTH);
  args.slices = 0;
  for (int i = 0; i < args.passes; ++i)
    args.slices += (args.pass[i].value_width + kSlice - 1) / kSlice;
  args.segment = plan.segment;
  args.slots = plan.slots;
  args.items = plan.slots * args.heads * args.slices;
  const dim3 grid = grid_of_items(args.items);
  if (plan.segmented) {
    decay_chunks_kernel<T, WIDTH, kSlice, TERMS, true, WHOLE>
        <<<grid, kDecayThreads<true>, 0, stream>>>(args);
    const int64_t size = static_cast<int64_t>(args.pass[0].key_width) * args.pass[0].value_width;
    const dim3 join = grid_of((size + kPieceElements - 1) / kPieceElements * args.heads * args.passes *
                              args.sequences.count);
    decay_join_kernel<T><<<join, kThreads, 0, stream>>>(args, size);
  } else {
    args.segment_states = nullptr;
  }
  decay_chunks_kernel<T, WIDTH, kSlice, TERMS, false, WHOLE>
      <<<grid, kDecayThreads<false>, 0, stream>>>(args);
}

template <typename T, int TERMS, bool WHOLE>
void decay_walk_width(DecayArgs<T>& args, const DecayPlan& plan, hipStream_t stream) {
  switch (plan.width) {
    case 32: return decay_walk<T, 32, TERMS, WHOLE>(args, plan, stream);
    case 64: return decay_walk<T, 64, TERMS, WHOLE>(args, plan, stream);
    default: return decay_walk<T, 128, TERMS, WHOLE>(args, plan, stream);
  }
}

template <typename T, int TERMS>
void decay_walk_any(DecayArgs<T>& args, const DecayPlan& plan, bool whole, hipStream_t stream) {
  if (whole)
    decay_walk_width<T, TERMS, true>(args, plan, stream);
  else
    decay_walk_width<T, TERMS, false>(args, plan, stream);
}

template <typename T>
bool whole_rows(const DecayCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  return whole_pieces<T>(*call.query, p.D) && whole_pieces<T>(*call.key, p.D) &&
         whole_pieces<T>(*call.value, p.Dv) &&
         (call.grad_output == nullptr || whole_pieces<T>(*call.grad_output, p.Dv)) &&
         whole_address(call.out) && whole_address(call.grad_query) && whole_address(call.grad_key) &&
         whole_address(call.grad_value);
}

template <typename T>
DecayArgs<T> decay_args(const DecayCall& call) {
  DecayArgs<T> args{};
  args.heads = call.problem->H;
  args.sequences = sequences_of(*call.problem);
  args.log_decay = call.log_decay;
  args.scale = call.problem->scale;
  return args;
}

template <typename T>
DecayPass<T> decay_forward_pass(const DecayCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  const int share = p.H / p.Hkv;
  return {view_of<T>(*call.query), view_of<T>(*call.key), view_of<T>(*call.value), 1, share, share,
          p.D, p.Dv, static_cast<T*>(call.out), nullptr, false};
}

// Two terms of a weighted value (2^-16) are enough where the state is only read through 16 bits.
template <typename T> constexpr int kTrainTerms = sizeof(T) == 4 ? 1 : 2;
template <typename T> constexpr int kUpdateTerms = sizeof(T) == 4 ? 1 : 3;

template <typename T>
void decay_forward(const DecayCall& call) {
  DecayArgs<T> args = decay_args<T>(call);
  const DecayPlan plan = decay_plan(*call.problem, 1);
  args.passes = 1;
  args.pass[0] = decay_forward_pass<T>(call);
  args.segment_states = reinterpret_cast<float*>(call.workspace);
  decay_walk_any<T, kTrainTerms<T>>(args, plan, whole_rows<T>(call), call.stream);
}

template <typename T>
void decay_backward(const DecayCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  const int share = p.H / p.Hkv;
  const DecayPlan plan = decay_plan(p, 3);
  DecayArgs<T> args = decay_args<T>(call);
  args.segment_states = reinterpret_cast<float*>(call.workspace);
  char* partial = call.workspace + plan.state_bytes;
  const View<const T> q = view_of<T>(*call.query), k = view_of<T>(*call.key),
                      v = view_of<T>(*call.value), go = view_of<T>(*call.grad_output);
  float *key_partial = nullptr, *value_partial = nullptr;
  args.passes = 0;
  if (call.grad_query)
    args.pass[args.passes++] = {go, v, k, 1, share, share, p.Dv, p.D,
                                static_cast<T*>(call.grad_query), nullptr, false};
  if (call.grad_key) {
    if (share > 1) key_partial = reinterpret_cast<float*>(partial);
    args.pass[args.passes++] = {v, go, q, share, 1, 1, p.Dv, p.D,
                                static_cast<T*>(call.grad_key), key_partial, true};
  }
  if (call.grad_value) {
    if (share > 1) value_partial = reinterpret_cast<float*>(partial + plan.key_partial_bytes);
    args.pass[args.passes++] = {k, q, go, share, 1, 1, p.D, p.Dv,
                                static_cast<T*>(call.grad_value), value_partial, true};
  }
  decay_walk_any<T, kTrainTerms<T>>(args, plan, whole_rows<T>(call), call.stream);
  const int64_t rows = static_cast<int64_t>(p.N) * p.Hkv;
  const auto blocks = [&](int width) {
    return grid_of((rows * width + kThreads - 1) / kThreads);
  };
  if (key_partial != nullptr)
    sum_shared_kernel<T><<<blocks(p.D), kThreads, 0, call.stream>>>(
        key_partial, static_cast<T*>(call.grad_key), rows, share, p.D);
  if (value_partial != nullptr)
    sum_shared_kernel<T><<<blocks(p.Dv), kThreads, 0, call.stream>>>(
        value_partial, static_cast<T*>(call.grad_value), rows, share, p.Dv);
}

template <typename T>
void decay_update(const DecayCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  if (p.cu_seqlens == nullptr && p.T == 1) {
    DecayTokenArgs<T> args{view_of<T>(*call.query), view_of<T>(*call.key), view_of<T>(*call.value),
                           call.log_decay, call.state_in, call.state_out,
                           static_cast<T*>(call.out), p.B, p.H, p.H / p.Hkv, p.D, p.Dv, 0, p.scale};
    const bool quads = p.Dv % 4 == 0 && reinterpret_cast<uintptr_t>(call.state_in) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(call.state_out) % 16 == 0;
    // whole rows of a state per block, or narrower slices until there are blocks for the chip
    args.slice = padded_width(p.Dv);
    while (args.slice > 16 && static_cast<int64_t>(p.B) * p.H * (p.Dv / args.slice + 1) < 512)
      args.slice /= 2;
    const dim3 grid = grid_of(static_cast<int64_t>((p.Dv + args.slice - 1) / args.slice) * p.H * p.B);
    if (quads)
      decay_token_kernel<T, 4><<<grid, kThreads, 0, call.stream>>>(args);
    else
      decay_token_kernel<T, 1><<<grid, kThreads, 0, call.stream>>>(args);
    return;
  }
  DecayArgs<T> args = decay_args<T>(call);
  const DecayPlan plan = decay_plan(p, 1);
  args.passes = 1;
  args.pass[0] = decay_forward_pass<T>(call);
  args.segment_states = reinterpret_cast<float*>(call.workspace);
  args.state_in = call.state_in;
  args.state_out = call.state_out;
  decay_walk_any<T, kUpdateTerms<T>>(args, plan, whole_rows<T>(call), call.stream);
}

}  // namespace rosa_mixer
