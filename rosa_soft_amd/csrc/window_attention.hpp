// Attention with a sliding window and sinks: token t sees token s <= t of its sequence when
// t - s < window or s < sinks.
//
//   p = softmax_s(scale q_t . k_s),  o_t = sum_s p_s v_s
//   backward: P again from the saved log-sum, dS = P (dO . v - dO . o),
//             dq = scale dS k, dk = scale dS^T q, dv = P^T dO
//
// Scores are formed transposed, keys down and the tokens of a wave across: the weights of a token
// then lie in the four lanes of its column, its maximum and sum are two lane exchanges away, and
// the weights are an operand of the product with the values as they stand.
#pragma once

#include "attention_device.hpp"
#include "mixer_calls.hpp"

namespace rosa_mixer {

template <typename T>
struct WindowArgs {
  View<const T> query, key, value, grad_output;
  const T* output;           // [tokens][heads][value_width]
  T* out;
  float *log_sum, *delta;    // [heads][tokens]
  T *grad_query, *grad_key, *grad_value;
  float* sink_sums;          // [sequence: sink_place][kv head][sink][key_width + value_width]
  float* sink_parts;         // [piece: sink_place][head][sink][key_width + value_width]
  int sink_rows, sink_far;   // tokens of a piece; longer sequences than sink_far have pieces
  const T *key_cache, *value_cache;
  const int32_t* lengths;
  int64_t capacity;
  Sequences sequences;
  int64_t slots, sink_slots, items;
  int heads, kv_heads, share, key_width, value_width, window, sinks;
  int key_block;             // keys of a block of window_grad_key_kernel
  int key_parts;             // blocks that share its walk
  bool exact_delta;          // delta of sequences whose tokens see few others is there already
  float *key_sums, *value_sums;  // [part][tokens][kv heads][width], where there is more than one
  float scale;
};

// Positions of a slot's cache: the sinks on rows of their own, the others in a ring behind them.
struct CacheRows {
  int sinks, ring;
  __device__ __forceinline__ int row(int position) const {
    return position < sinks ? position : sinks + (position - sinks) % ring;
  }
};

// Which elements of a column of scores are seen: e up to `last`, and from `first` on or below
// `sinks`; e counts from the lane's first row.  (Bitwise: no branch per element.)
struct Seen {
  int first, last, sinks;
  __device__ __forceinline__ bool operator()(int e) const {
    return (e <= last) & ((e >= first) | (e < sinks));
  }
};

// of token t, keys from `row` on (the lane's first of a tile) that end before `end`
__device__ __forceinline__ Seen seen_keys(int t, int row, int end, int window, int sinks) {
  asm volatile("" : "+v"(row));  // (stays on the path of the tiles that need it)
  return {t - window + 1 - row, min(t, end - 1) - row, sinks - row};
}

// The rows of keys or values of a head by position: those before `past` in the cache, the others
// among the new tokens.
template <typename T, bool CACHED>
struct History {
  const T* fresh;               // of the first new token
  int64_t stride;
  const T* cache;               // of row 0
  int width, past;
  CacheRows rows;
  __device__ __forceinline__ const T* row(int s) const {
    if (CACHED && s < past) return cache + static_cast<int64_t>(rows.row(s)) * width;
    return fresh + (CACHED ? s - past : s) * stride;
  }
  // Positions [begin, end), as rows that lie one behind the other.  Those of a cache do not where
  // the ring closes, nor where they end and the new tokens begin.
  __device__ __forceinline__ bool in_order(int begin, int end) const {
    if (!CACHED || begin >= past) return true;
    return end <= past && (begin < rows.sinks ? end <= rows.sinks
                                              : rows.row(begin) + (end - 1 - begin) < rows.sinks + rows.ring);
  }
  __device__ __forceinline__ Rows<T> span(int begin, int end) const {
    return {row(begin), CACHED && begin < past ? width : stride, end - 1 - begin};
  }
  template <typename Move>
  __device__ __forceinline__ void fetch(Move& move, int begin, int end, int tid) const {
    if (in_order(begin, end))
      move.fetch(span(begin, end), width, tid);
    else
      move.fetch_from([&](int i, int col) { return row(min(begin + i, end - 1)) + col; }, width, tid);
  }
};

template <bool CACHED, typename T>
__device__ __forceinline__ int tokens_before(const WindowArgs<T>& a, const Run& run) {
  if constexpr (!CACHED) return 0;
  return max(0, min(a.lengths[run.sequence], 0x7fffffff - run.length - 1024));
}

template <bool CACHED, typename T>
__device__ __forceinline__ History<T, CACHED> history_of(const WindowArgs<T>& a, const View<const T>& view,
                                                         const T* cache, int width, const Run& run,
                                                         int kv_head, int past) {
  History<T, CACHED> rows{};
  rows.fresh = view.row(run.batch, run.begin, kv_head);
  rows.stride = view.token_stride;
  rows.width = width;
  rows.past = past;
  if constexpr (CACHED) {
    rows.cache = cache + (static_cast<int64_t>(run.sequence) * a.kv_heads + kv_head) * a.capacity * width;
    rows.rows = {a.sinks, static_cast<int>(a.capacity) - a.sinks};
  }
  return rows;
}

// The key tiles of the tokens [first, last]: the sinks in front of the window, then the window.
struct KeyTiles {
  int window_begin, sinks_end, at, last;
  __device__ __forceinline__ KeyTiles(int first, int last_, int window, int sinks)
      : window_begin(max(0, first - window + 1)), sinks_end(min(sinks, window_begin)),
        at(sinks_end > 0 ? -1 : window_begin), last(last_) {}
  __device__ __forceinline__ bool more() const { return at <= last; }
  __device__ __forceinline__ int begin() const { return at < 0 ? 0 : at; }
  __device__ __forceinline__ int end() const { return at < 0 ? sinks_end : min(at + kKeys, last + 1); }
  __device__ __forceinline__ void next() { at = at < 0 ? window_begin : at + kKeys; }
};

// o (and the log-sums) of 64 QUERIES tokens of a query head, 16 QUERIES to a wave, over their key
// tiles: keys and values go through registers to LDS while the tile before is worked on, queries
// and sums stay in registers.  Weights are rounded to the inputs' type, as the operand of the
// product with the values, and summed as rounded.  Measured in bfloat16, 2 x 4096 tokens, 32 heads
// of 128 on 8, window 1024: 190 us, 635 TFLOP/s of visible pairs.  What bounds it: matrix and vector
// instructions of the two waves of a SIMD, of the second mostly exponentials and rounding (left
// out one at a time: scores 64 us, values' product 36, exponentials 17, loads 27).  One tile of
// tokens per wave instead of two: 227 us.  Wave priorities around the products and keys read ahead
// of them gained nothing.
template <typename T, int WIDTH, int QUERIES, bool CACHED, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWaves<T, WIDTH, WHOLE>))) void
window_forward_kernel(WindowArgs<T> a) {
  constexpr int kSteps = WIDTH / 32, kRows = 64 * QUERIES, kCols = WIDTH / 16;
  constexpr int kTile = kTileElements<T, kKeys, WIDTH>;
  __shared__ __attribute__((aligned(16))) Stored<T> key_tiles[kBuffers<T> * kTile];
  __shared__ __attribute__((aligned(16))) Stored<T> value_tiles[kBuffers<T> * kTile];

  const int64_t item = item_of_block(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the query heads that share keys and values are neighbours; late tiles, which see most, first
  const int64_t slot = a.slots - 1 - item / a.share % a.slots;
  const int kv_head = static_cast<int>(item / a.share / a.slots);
  const int head = kv_head * a.share + static_cast<int>(item % a.share);
  Run run;
  const Found found = find_run(a.sequences, slot, kRows, tid, &run);
  if (found != Found::kRun) {
    if (found == Found::kInvalid)
      fill_nan(a.out, slot * kRows, min((slot + 1) * kRows, static_cast<int64_t>(a.sequences.tokens)),
               a.heads, head, a.value_width, tid);
    return;
  }
  const int past = tokens_before<CACHED>(a, run);
  const int first = past + run.tile * kRows, last = min(first + kRows, past + run.length) - 1;
  const History<T, CACHED> key_rows = history_of<CACHED>(a, a.key, a.key_cache, a.key_width, run, kv_head, past);
  const History<T, CACHED> value_rows =
      history_of<CACHED>(a, a.value, a.value_cache, a.value_width, run, kv_head, past);

  // this wave's tokens, as the columns of operands
  const int wave_first = first + wave * 16 * QUERIES, wave_last = wave_first + 16 * QUERIES - 1;
  Operand<T> query[QUERIES][kSteps];
  const Rows<T> query_rows = a.query.rows(run.batch, run.begin + first - past, head, last - first + 1);
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int row = wave * 16 * QUERIES + i * 16 + column;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Frag<T> part = memory_operand<WHOLE>(query_rows, row, s * 32 + 8 * group, a.key_width);
      clear_operand<WHOLE>(part, s * 32, group, a.key_width);
      query[i][s] = as_operand<T>(part);
    }
  }
  f32x4 out[QUERIES][kCols];
  float most[QUERIES];
  // The sums of the weights: a product with ones, which adds what is rounded and takes no vector
  // instructions (every row of the result is the sum).
  f32x4 sum[QUERIES];
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    most[i] = -__builtin_inff();
    sum[i] = f32x4(0.0f);
#pragma unroll
    for (int d = 0; d < kCols; ++d) out[i][d] = f32x4(0.0f);
  }
  const float factor = a.scale * kLog2e;

  TileMove<T, kKeys, WIDTH, WHOLE> key_move, value_move;
  KeyTiles tiles(first, last, a.window, a.sinks);
  const auto fetch = [&] {
    const int begin = tiles.begin(), end = tiles.end();
    key_rows.fetch(key_move, begin, end, tid);
    value_rows.fetch(value_move, begin, end, tid);
  };
  fetch();
  for (int side = 0; tiles.more(); side = kBuffers<T> - 1 - side) {
    const int begin = tiles.begin(), end = tiles.end();
    tiles.next();
    Stored<T>*keys = key_tiles + side * kTile, *values = value_tiles + side * kTile;
    key_move.store(keys, a.key_width, tid);
    value_move.store(values, a.value_width, tid);
    __syncthreads();
    if (tiles.more()) fetch();
    // nothing of this tile is visible to the wave: behind it, or before its windows and no sink
    const bool none = begin > min(wave_last, last) || wave_first > last ||
                      (end - 1 <= wave_first - a.window && begin >= a.sinks);
    if (!none) {
      const bool all = end - begin == kKeys && end - 1 <= wave_first && wave_last - begin < a.window;
      f32x4 score[QUERIES][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < QUERIES; ++i) score[i][k] = f32x4(0.0f);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const Operand<T> key = row_operand<T, kKeys, WIDTH>(keys, k * 16, s * 32, lane);
#pragma unroll
          for (int i = 0; i < QUERIES; ++i) score[i][k] = mma(key, query[i][s], score[i][k]);
        }
      }
      Operand<T> weights[QUERIES][2];
      if (!all) {
#pragma unroll
        for (int i = 0; i < QUERIES; ++i) {
          const Seen seen = seen_keys(wave_first + i * 16 + column, begin + 4 * group, end, a.window,
                                      a.sinks);
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              score[i][k][r] = seen(k * 16 + r) ? score[i][k][r] : -__builtin_inff();
        }
      }
#pragma unroll
      for (int i = 0; i < QUERIES; ++i) {
        float here = score[i][0][0];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) here = fmaxf(here, score[i][k][r]);
        here = over_groups_max(here) * factor;
        if (__any(here > most[i] + kSlack)) {
          const float larger = fmaxf(here, most[i]);
          const float shrink = larger == -__builtin_inff() ? 1.0f : exp2_of(most[i] - larger);
          sum[i] *= shrink;
#pragma unroll
          for (int d = 0; d < kCols; ++d) out[i][d] *= shrink;
          most[i] = larger;
        }
        const float base = (most[i] == -__builtin_inff() ? 0.0f : most[i]) - kLift<T>;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            score[i][k][r] = exp2_of(score[i][k][r] * factor - base);
          }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          weights[i][half] = operand_of<T>(score[i][2 * half], score[i][2 * half + 1]);
          sum[i] = add_sums<T>(weights[i][half], sum[i]);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int d = 0; d < kCols; ++d) {
          const Operand<T> value = column_operand<T, kKeys, WIDTH>(values, half * 32, d * 16, lane);
#pragma unroll
          for (int i = 0; i < QUERIES; ++i) out[i][d] = mma(value, weights[i][half], out[i][d]);
        }
    }
    if constexpr (kBuffers<T> == 1) __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int t = wave_first + i * 16 + column;
    const float total = sum[i][0];
    if (t > last) continue;
    const int64_t token = run.first + t - past;
    T* to = a.out + (token * a.heads + head) * a.value_width;
    const float by = 1.0f / total;
    store_tiles<WHOLE, false>(to, out[i], by, group, a.value_width);
    if (a.log_sum != nullptr && group == 0)
      a.log_sum[static_cast<int64_t>(head) * a.sequences.tokens + token] = most[i] + log2_of(total) - kLift<T>;
  }
}

// dq, and the sums delta = dO . o = sum_s p_s dO . v_s that the gradients of keys need too.  The
// walk of the forward pass.  Where tokens see many others delta is taken from the output, whose
// rounding is small beside dO . v then.  Where they see kExactSpan or fewer (the window, or half
// of their sequence) it would add half as much error again (dq and dk of 50 tokens in
// bfloat16: 2.8e-3 of their norm instead of 2.4e-3), and a walk of its own sums delta over the
// keys first (DELTA: 27 us of 150, forward included, at 6 x 520 tokens, 22 heads, window 40).
// Packed calls go by their mean length when that walk is launched, and sequence by sequence in it.
// Slopes are rounded to the inputs' type, in float16 scaled to its upper range (follow_range).
// Measured as above: 245 us, 740 TFLOP/s.
constexpr int kExactSpan = 256;
__host__ __device__ __forceinline__ bool few_seen(int window, int length) {
  return window <= kExactSpan || length / 2 <= kExactSpan;
}

template <typename T, int WIDTH, int QUERIES, bool WHOLE, bool DELTA>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWaves<T, WIDTH, WHOLE>))) void
window_grad_query_kernel(WindowArgs<T> a) {
  constexpr int kSteps = WIDTH / 32, kRows = 64 * QUERIES, kCols = WIDTH / 16;
  constexpr int kTile = kTileElements<T, kKeys, WIDTH>;
  __shared__ __attribute__((aligned(16))) Stored<T> key_tiles[kBuffers<T> * kTile];
  __shared__ __attribute__((aligned(16))) Stored<T> value_tiles[kBuffers<T> * kTile];

  const int64_t item = item_of_block(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slot = a.slots - 1 - item / a.share % a.slots;
  const int kv_head = static_cast<int>(item / a.share / a.slots);
  const int head = kv_head * a.share + static_cast<int>(item % a.share);
  Run run;
  const Found found = find_run(a.sequences, slot, kRows, tid, &run);
  if (found != Found::kRun) {
    if (found == Found::kInvalid && !DELTA)
      fill_nan(a.grad_query, slot * kRows,
               min((slot + 1) * kRows, static_cast<int64_t>(a.sequences.tokens)), a.heads, head,
               a.key_width, tid);
    return;
  }
  const bool exact_delta = a.exact_delta && few_seen(a.window, run.length);
  if (DELTA && !exact_delta) return;
  const int first = run.tile * kRows, last = min(first + kRows, run.length) - 1;
  const History<T, false> key_rows = history_of<false>(a, a.key, a.key_cache, a.key_width, run, kv_head, 0);
  const History<T, false> value_rows =
      history_of<false>(a, a.value, a.value_cache, a.value_width, run, kv_head, 0);
  const int wave_first = first + wave * 16 * QUERIES, wave_last = wave_first + 16 * QUERIES - 1;

  Operand<T> query[QUERIES][kSteps], grad[QUERIES][kSteps];
  float log_sum[QUERIES], delta[QUERIES], unit[QUERIES];
  const int count = last - first + 1;
  const Rows<T> query_rows = a.query.rows(run.batch, run.begin + first, head, count);
  const Rows<T> grad_rows = a.grad_output.rows(run.batch, run.begin + first, head, count);
  const Rows<T> out_rows{a.output + ((run.first + first) * a.heads + head) * a.value_width,
                         static_cast<int64_t>(a.heads) * a.value_width, count - 1};
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int row = wave * 16 * QUERIES + i * 16 + column;
    const bool there = row < count;
    float dot = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Frag<T> part = memory_operand<WHOLE>(query_rows, row, s * 32 + 8 * group, a.key_width);
      Frag<T> grad_part = memory_operand<WHOLE>(grad_rows, row, s * 32 + 8 * group, a.value_width);
      Frag<T> out = memory_operand<WHOLE>(out_rows, row, s * 32 + 8 * group, a.value_width);
      clear_operand<WHOLE>(part, s * 32, group, a.key_width);
      clear_operand<WHOLE>(grad_part, s * 32, group, a.value_width);
      clear_operand<WHOLE>(out, s * 32, group, a.value_width);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot += static_cast<float>(grad_part[e]) * static_cast<float>(out[e]);
      query[i][s] = as_operand<T>(part);
      grad[i][s] = as_operand<T>(grad_part);
    }
    const int64_t at = static_cast<int64_t>(head) * a.sequences.tokens + run.first + first + min(row, count - 1);
    log_sum[i] = a.log_sum[at];
    if constexpr (DELTA) {
      delta[i] = 0.0f;
    } else if (exact_delta) {
      delta[i] = a.delta[at];
    } else {
      delta[i] = over_groups_sum(dot);
      if (there && group == 0) a.delta[at] = delta[i];
    }
    unit[i] = kNarrow<T> ? 0.0f : 1.0f;
  }
  if (!DELTA && a.grad_query == nullptr) return;
  float exact[QUERIES] = {};  // this lane's part of delta
  f32x4 out[QUERIES][kCols];
#pragma unroll
  for (int i = 0; i < QUERIES; ++i)
#pragma unroll
    for (int d = 0; d < kCols; ++d) out[i][d] = f32x4(0.0f);
  const float factor = a.scale * kLog2e;

  TileMove<T, kKeys, WIDTH, WHOLE> key_move, value_move;
  KeyTiles tiles(first, last, a.window, a.sinks);
  const auto fetch = [&] {
    const int begin = tiles.begin(), end = tiles.end();
    key_rows.fetch(key_move, begin, end, tid);
    value_rows.fetch(value_move, begin, end, tid);
  };
  fetch();
  for (int side = 0; tiles.more(); side = kBuffers<T> - 1 - side) {
    const int begin = tiles.begin(), end = tiles.end();
    tiles.next();
    Stored<T>*keys = key_tiles + side * kTile, *values = value_tiles + side * kTile;
    key_move.store(keys, a.key_width, tid);
    value_move.store(values, a.value_width, tid);
    __syncthreads();
    if (tiles.more()) fetch();
    const bool none = begin > min(wave_last, last) || wave_first > last ||
                      (end - 1 <= wave_first - a.window && begin >= a.sinks);
    if (!none) {
      const bool all = end - begin == kKeys && end - 1 <= wave_first && wave_last - begin < a.window;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x4 slope[QUERIES][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x4 score[QUERIES];
#pragma unroll
          for (int i = 0; i < QUERIES; ++i) score[i] = slope[i][k] = f32x4(0.0f);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const Operand<T> key = row_operand<T, kKeys, WIDTH>(keys, half * 32 + k * 16, s * 32, lane);
            const Operand<T> value = row_operand<T, kKeys, WIDTH>(values, half * 32 + k * 16, s * 32, lane);
#pragma unroll
            for (int i = 0; i < QUERIES; ++i) {
              score[i] = mma(key, query[i][s], score[i]);
              slope[i][k] = mma(value, grad[i][s], slope[i][k]);
            }
          }
#pragma unroll
          for (int i = 0; i < QUERIES; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float p = exp2_of(score[i][r] * factor - log_sum[i]);
              slope[i][k][r] = p * (slope[i][k][r] - delta[i]);
            }
            if (!all) {
              const Seen seen = seen_keys(wave_first + i * 16 + column,
                                          begin + half * 32 + k * 16 + 4 * group, end, a.window, a.sinks);
#pragma unroll
              for (int r = 0; r < 4; ++r) slope[i][k][r] = seen(r) ? slope[i][k][r] : 0.0f;
            }
            if constexpr (DELTA)
              exact[i] += slope[i][k][0] + slope[i][k][1] + slope[i][k][2] + slope[i][k][3];
          }
        }
        if constexpr (DELTA) continue;
        Operand<T> operand[QUERIES];
#pragma unroll
        for (int i = 0; i < QUERIES; ++i) {
          if constexpr (kNarrow<T>) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(slope[i][k][r]));
            const float by = follow_range(&unit[i], over_groups_max(most));
            if (__any(by != 1.0f)) {
#pragma unroll
              for (int d = 0; d < kCols; ++d) out[i][d] *= by;
            }
            slope[i][0] *= unit[i];
            slope[i][1] *= unit[i];
          }
          operand[i] = operand_of<T>(slope[i][0], slope[i][1]);
        }
#pragma unroll
        for (int d = 0; d < kCols; ++d) {
          const Operand<T> key = column_operand<T, kKeys, WIDTH>(keys, half * 32, d * 16, lane);
#pragma unroll
          for (int i = 0; i < QUERIES; ++i) out[i][d] = mma(key, operand[i], out[i][d]);
        }
      }
    }
    if constexpr (kBuffers<T> == 1) __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int t = wave_first + i * 16 + column;
    if constexpr (DELTA) exact[i] = over_groups_sum(exact[i]);
    if (t > last) continue;
    if constexpr (DELTA) {
      if (group == 0) a.delta[static_cast<int64_t>(head) * a.sequences.tokens + run.first + t] = exact[i];
      continue;
    }
    T* to = a.grad_query + ((run.first + t) * a.heads + head) * a.key_width;
    const float by = unit[i] == 0.0f ? a.scale : a.scale / unit[i];
    store_tiles<WHOLE, false>(to, out[i], by, group, a.key_width);
  }
}

// The tokens from here on see the sinks beyond their window: the first block of keys of a sequence
// walks the tokens before it, window_grad_sinks_kernel the others, or that block all of them where
// they are few (sequences of up to sink_far tokens).
__device__ __forceinline__ int64_t walk_end(int first, int keys, int window) {
  return static_cast<int64_t>(first) + keys - 1 + window;
}

// Where the sums of a sequence's sinks lie, and its first piece.  Packed sequences go by where they
// begin: of two with more than sink_far tokens the second begins more than sink_far behind the first,
// and n tokens are at most n / sink_rows + 1 pieces, so that no two share a place.
struct SinkPlace {
  int64_t sums, piece;
};
template <typename T>
__device__ __forceinline__ SinkPlace sink_place(const WindowArgs<T>& a, const Run& run) {
  if (a.sequences.offsets == nullptr) return {run.sequence, first_slot(a.sequences, run, a.sink_rows)};
  const int begin = static_cast<int>(run.begin);
  return {begin / a.sink_far, static_cast<int64_t>(begin / a.sink_rows) + begin / a.sink_far};
}

// dk and dv of the keys of a block, 16 KEYS to a wave, over the tokens that see them and the query
// heads that share them: scores have the tokens down and the wave's keys across.  Weights and slopes
// are rounded to the inputs' type.  Measured as above: 390 us, 620 TFLOP/s, one wave per SIMD (of 128
// columns, two key tiles take 377 registers): what bounds it is that nothing fills its waits.  One
// key tile per wave and two waves per SIMD instead: 402 us.
template <typename T, int WIDTH, int KEYS, bool WHOLE>
constexpr int kKeyWaves = WIDTH * sizeof(T) <= 128 || (sizeof(T) == 2 && KEYS == 1 && WHOLE) ? 2 : 1;
template <typename T, int WIDTH, int KEYS, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kKeyWaves<T, WIDTH, KEYS, WHOLE>))) void
window_grad_key_kernel(WindowArgs<T> a) {
  constexpr int kSteps = WIDTH / 32, kRows = 64 * KEYS, kCols = WIDTH / 16;
  constexpr int kQueries = sizeof(T) == 4 && WIDTH == 128 ? 32 : 64;  // (registers)
  constexpr int kTile = kTileElements<T, kQueries, WIDTH>;
  __shared__ __attribute__((aligned(16))) Stored<T> query_tiles[kBuffers<T> * kTile];
  __shared__ __attribute__((aligned(16))) Stored<T> grad_tiles[kBuffers<T> * kTile];
  __shared__ __attribute__((aligned(16))) float tile_sums[kBuffers<T>][2][kQueries];

  const int64_t item = item_of_block(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = static_cast<int>(item % a.key_parts);
  const int64_t slot = item / a.key_parts % a.slots;
  const int kv_head = static_cast<int>(item / a.key_parts / a.slots);
  const int64_t rows_of_parts = static_cast<int64_t>(part) * a.sequences.tokens * a.kv_heads;
  Run run;
  const Found found = find_run(a.sequences, slot, kRows, tid, &run);
  if (found != Found::kRun) {
    if (found == Found::kInvalid) {
      const int64_t first = slot * kRows;
      const int64_t last = min(first + kRows, static_cast<int64_t>(a.sequences.tokens));
      if (a.key_parts > 1) {  // (one part makes the sum NaN)
        if (part == 0) {
          fill_nan(a.key_sums, first, last, a.kv_heads, kv_head, a.key_width, tid);
          fill_nan(a.value_sums, first, last, a.kv_heads, kv_head, a.value_width, tid);
        }
      } else {
        fill_nan(a.grad_key, first, last, a.kv_heads, kv_head, a.key_width, tid);
        fill_nan(a.grad_value, first, last, a.kv_heads, kv_head, a.value_width, tid);
      }
    }
    return;
  }
  // keys of the block; the tokens [first, to) walked for them
  const int first = run.tile * kRows, behind = min(first + kRows, run.length);
  const bool all_tokens = run.tile == 0 && a.sinks > 0 && run.length <= a.sink_far;
  const int to = all_tokens ? run.length
                            : static_cast<int>(min<int64_t>(run.length, walk_end(first, kRows, a.window)));
  const int sums = a.key_width + a.value_width;

  const int wave_first = first + wave * 16 * KEYS;
  const Rows<T> key_rows = a.key.rows(run.batch, run.begin + first, kv_head, behind - first);
  const Rows<T> value_rows = a.value.rows(run.batch, run.begin + first, kv_head, behind - first);
  Operand<T> key[KEYS][kSteps], value[KEYS][kSteps];
  f32x4 grad_key[KEYS][kCols], grad_value[KEYS][kCols];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int row = wave * 16 * KEYS + i * 16 + column;
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      Frag<T> part = memory_operand<WHOLE>(key_rows, row, step * 32 + 8 * group, a.key_width);
      Frag<T> value_part = memory_operand<WHOLE>(value_rows, row, step * 32 + 8 * group, a.value_width);
      clear_operand<WHOLE>(part, step * 32, group, a.key_width);
      clear_operand<WHOLE>(value_part, step * 32, group, a.value_width);
      key[i][step] = as_operand<T>(part);
      value[i][step] = as_operand<T>(value_part);
    }
#pragma unroll
    for (int d = 0; d < kCols; ++d) grad_key[i][d] = grad_value[i][d] = f32x4(0.0f);
  }
  float unit[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) unit[i] = kNarrow<T> ? 0.0f : 1.0f;
  if (part == 0 && run.tile == 0 && a.sink_sums != nullptr && to < run.length) {
    const float* sinks = a.sink_sums + (sink_place(a, run).sums * a.kv_heads + kv_head) * a.sinks * sums;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int s = wave_first + i * 16 + column;
      if (s >= a.sinks) continue;
#pragma unroll
      for (int d = 0; d < kCols; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = d * 16 + 4 * group + r;
          if (col < a.key_width) grad_key[i][d][r] = sinks[s * sums + col];
          if (col < a.value_width) grad_value[i][d][r] = sinks[s * sums + a.key_width + col];
        }
    }
  }
  const float factor = a.scale * kLog2e;
  const bool idle = wave_first >= behind;

  TileMove<T, kQueries, WIDTH, WHOLE> query_move, grad_move;
  float next_log_sum = 0.0f, next_delta = 0.0f;
  const int walk = (to - first + kQueries - 1) / kQueries;
  const auto fetch = [&](int step) {
    const int head = kv_head * a.share + step / walk, begin = first + step % walk * kQueries;
    const int count = min(kQueries, to - begin);
    query_move.fetch(a.query.rows(run.batch, run.begin + begin, head, count), a.key_width, tid);
    grad_move.fetch(a.grad_output.rows(run.batch, run.begin + begin, head, count), a.value_width, tid);
    if (tid < kQueries) {
      const int64_t at =
          static_cast<int64_t>(head) * a.sequences.tokens + run.first + begin + min(tid, count - 1);
      next_log_sum = a.log_sum[at] - kLift<T>;
      next_delta = a.delta[at];
    }
  };
  // this part's steps (the last parts of a short walk have none)
  const int steps = (walk * a.share + a.key_parts - 1) / a.key_parts;
  const int step_end = min(walk * a.share, (part + 1) * steps);
  if (part * steps < step_end) fetch(part * steps);
  for (int step = part * steps, side = 0; step < step_end; ++step, side = kBuffers<T> - 1 - side) {
    const int begin = first + step % walk * kQueries;
    Stored<T>*queries = query_tiles + side * kTile, *grads = grad_tiles + side * kTile;
    float *log_sums = tile_sums[side][0], *deltas = tile_sums[side][1];
    query_move.store(queries, a.key_width, tid);
    grad_move.store(grads, a.value_width, tid);
    if (tid < kQueries) {
      log_sums[tid] = next_log_sum;
      deltas[tid] = next_delta;
    }
    __syncthreads();
    if (step + 1 < step_end) fetch(step + 1);
    const int wave_last = min(wave_first + 16 * KEYS, behind) - 1;
    const bool none = idle || begin + kQueries - 1 < wave_first ||
                      (begin - wave_last >= a.window && wave_first >= a.sinks);
    if (!none) {
      const bool all = wave_last - wave_first + 1 == 16 * KEYS && wave_last <= begin &&
                       begin + kQueries <= to && begin + kQueries - 1 - wave_first < a.window;
#pragma unroll
      for (int half = 0; half < kQueries / 32; ++half) {
        f32x4 weight[KEYS][2], slope[KEYS][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row0 = half * 32 + k * 16;
#pragma unroll
          for (int i = 0; i < KEYS; ++i) weight[i][k] = slope[i][k] = f32x4(0.0f);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const Operand<T> query = row_operand<T, kQueries, WIDTH>(queries, row0, s * 32, lane);
            const Operand<T> grad = row_operand<T, kQueries, WIDTH>(grads, row0, s * 32, lane);
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
              weight[i][k] = mma(query, key[i][s], weight[i][k]);
              slope[i][k] = mma(grad, value[i][s], slope[i][k]);
            }
          }
          const f32x4 log_sum = *reinterpret_cast<const f32x4*>(log_sums + row0 + 4 * group);
          const f32x4 delta = *reinterpret_cast<const f32x4*>(deltas + row0 + 4 * group);
#pragma unroll
          for (int i = 0; i < KEYS; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              weight[i][k][r] = exp2_of(weight[i][k][r] * factor - log_sum[r]);  // (lifted)
              slope[i][k][r] = weight[i][k][r] * (slope[i][k][r] - delta[r]);
            }
          }
        }
        if (!all) {  // tokens t from this row on that see key s: s <= t < to, t - s < window
#pragma unroll
          for (int i = 0; i < KEYS; ++i) {
            const int s = wave_first + i * 16 + column, row = begin + half * 32 + 4 * group;
            const int64_t end = s >= behind ? 0 : s < a.sinks ? to : min<int64_t>(to, int64_t{s} + a.window);
            const int first_seen = s - row, last_seen = static_cast<int>(end) - 1 - row;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const bool seen = (k * 16 + r >= first_seen) & (k * 16 + r <= last_seen);
                weight[i][k][r] = seen ? weight[i][k][r] : 0.0f;
                slope[i][k][r] = seen ? slope[i][k][r] : 0.0f;
              }
          }
        }
        Operand<T> weights[KEYS], slopes[KEYS];
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
          if constexpr (kNarrow<T>) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(slope[i][k][r]));
            const float by = follow_range(&unit[i], over_groups_max(most));
            if (__any(by != 1.0f)) {
#pragma unroll
              for (int d = 0; d < kCols; ++d) grad_key[i][d] *= by;
            }
            slope[i][0] *= unit[i];
            slope[i][1] *= unit[i];
          }
          weights[i] = operand_of<T>(weight[i][0], weight[i][1]);
          slopes[i] = operand_of<T>(slope[i][0], slope[i][1]);
        }
#pragma unroll
        for (int d = 0; d < kCols; ++d) {
          const Operand<T> grad = column_operand<T, kQueries, WIDTH>(grads, half * 32, d * 16, lane);
          const Operand<T> query = column_operand<T, kQueries, WIDTH>(queries, half * 32, d * 16, lane);
#pragma unroll
          for (int i = 0; i < KEYS; ++i) {
            grad_value[i][d] = mma(grad, weights[i], grad_value[i][d]);
            grad_key[i][d] = mma(query, slopes[i], grad_key[i][d]);
          }
        }
      }
    }
    if constexpr (kBuffers<T> == 1) __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int s = wave_first + i * 16 + column;
    if (s >= behind) continue;
    const float back = unit[i] == 0.0f ? 1.0f : 1.0f / unit[i];
    const int64_t row = (run.first + s) * a.kv_heads + kv_head;
    const float key_by = a.scale * back * kUnlift<T>;
    if (a.key_parts > 1) {
      float* key_to = a.key_sums + (rows_of_parts + row) * a.key_width;
      float* value_to = a.value_sums + (rows_of_parts + row) * a.value_width;
      store_tiles<WHOLE, false>(key_to, grad_key[i], key_by, group, a.key_width);
      store_tiles<WHOLE, false>(value_to, grad_value[i], kUnlift<T>, group, a.value_width);
      continue;
    }
    if (a.grad_key != nullptr)
      store_tiles<WHOLE, false>(a.grad_key + row * a.key_width, grad_key[i], key_by, group, a.key_width);
    if (a.grad_value != nullptr)
      store_tiles<WHOLE, false>(a.grad_value + row * a.value_width, grad_value[i], kUnlift<T>, group,
                                a.value_width);
  }
}

// The sum of the parts of a walk, in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_join_keys_kernel(const float* parts, T* out, int count,
                                                                    int64_t elements) {
  const int64_t e = static_cast<int64_t>(block_number()) * kThreads + threadIdx.x;
  if (e >= elements) return;
  float sum = 0.0f;
  for (int part = 0; part < count; ++part) sum += parts[part * elements + e];
  out[e] = static_cast<T>(sum);
}

// The gradients of the sinks from the tokens beyond the first block's walk: every block takes a
// piece of sink_rows tokens of one query head and 16 sinks, every wave 32 tokens of a tile.  (One
// block walking all of them would be the last to finish by far.)  Measured as above, 4 sinks:
// 28 us, most of it the reads of q and dO (98 MB, 3.5 TB/s).
template <typename T, int WIDTH, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1))) void
window_grad_sinks_kernel(WindowArgs<T> a) {
  constexpr int kSteps = WIDTH / 32, kCols = WIDTH / 16;
  constexpr int kRows = sizeof(T) == 4 ? 64 : 128, kTeams = kRows / 32;  // waves with tokens
  constexpr int kSumPitch = WIDTH + 4;
  constexpr size_t kTileBytes = sizeof(Stored<T>) * kTileElements<T, kRows, WIDTH>;
  static_assert(2 * kTileBytes >= sizeof(float) * kTeams * 2 * 16 * kSumPitch, "sums lie over the tiles");
  __shared__ __attribute__((aligned(16))) char shared[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) float log_sums[kRows], deltas[kRows];
  Stored<T>* queries = reinterpret_cast<Stored<T>*>(shared);
  Stored<T>* grads = reinterpret_cast<Stored<T>*>(shared + kTileBytes);

  const int64_t item = item_of_block(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int parts = (a.sinks + 15) / 16;
  const int first = static_cast<int>(item % parts) * 16;
  const int head = static_cast<int>(item / parts % a.heads), kv_head = head / a.share;
  const int64_t slot = item / parts / a.heads;
  Run run;
  if (find_run(a.sequences, slot, a.sink_rows, tid, &run) != Found::kRun) return;
  if (run.length <= a.sink_far) return;  // (sink_far is no less than where the first block's walk ends)
  const int from = max(run.tile * a.sink_rows, static_cast<int>(walk_end(0, a.key_block, a.window)));
  const int to = run.tile * a.sink_rows + min(a.sink_rows, run.length - run.tile * a.sink_rows);
  if (from >= to) return;  // (nor are its sums read)

  // these tokens see all sinks
  Operand<T> key[kSteps], value[kSteps];
  f32x4 grad_key[kCols], grad_value[kCols];
  const Rows<T> key_rows = a.key.rows(run.batch, run.begin + first, kv_head, a.sinks - first);
  const Rows<T> value_rows = a.value.rows(run.batch, run.begin + first, kv_head, a.sinks - first);
#pragma unroll
  for (int step = 0; step < kSteps; ++step) {
    Frag<T> part = memory_operand<WHOLE>(key_rows, column, step * 32 + 8 * group, a.key_width);
    Frag<T> value_part = memory_operand<WHOLE>(value_rows, column, step * 32 + 8 * group, a.value_width);
    clear_operand<WHOLE>(part, step * 32, group, a.key_width);
    clear_operand<WHOLE>(value_part, step * 32, group, a.value_width);
    key[step] = as_operand<T>(part);
    value[step] = as_operand<T>(value_part);
  }
#pragma unroll
  for (int d = 0; d < kCols; ++d) grad_key[d] = grad_value[d] = f32x4(0.0f);
  float unit = kNarrow<T> ? 0.0f : 1.0f;
  const float factor = a.scale * kLog2e;

  TileMove<T, kRows, WIDTH, WHOLE> query_move, grad_move;
  for (int begin = from; begin < to; begin += kRows) {
    const int count = min(kRows, to - begin);
    query_move.fetch(a.query.rows(run.batch, run.begin + begin, head, count), a.key_width, tid);
    grad_move.fetch(a.grad_output.rows(run.batch, run.begin + begin, head, count), a.value_width, tid);
    __syncthreads();
    if (tid < kRows) {
      const int64_t at =
          static_cast<int64_t>(head) * a.sequences.tokens + run.first + begin + min(tid, count - 1);
      log_sums[tid] = a.log_sum[at] - kLift<T>;
      deltas[tid] = a.delta[at];
    }
    query_move.store(queries, a.key_width, tid);
    grad_move.store(grads, a.value_width, tid);
    __syncthreads();
    const int row0 = wave * 32;
    if (wave >= kTeams || row0 >= count) continue;
    f32x4 weight[2], slope[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      weight[k] = slope[k] = f32x4(0.0f);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        weight[k] = mma(row_operand<T, kRows, WIDTH>(queries, row0 + k * 16, s * 32, lane), key[s], weight[k]);
        slope[k] = mma(row_operand<T, kRows, WIDTH>(grads, row0 + k * 16, s * 32, lane), value[s], slope[k]);
      }
      const int row = row0 + k * 16 + 4 * group;
      const f32x4 log_sum = *reinterpret_cast<const f32x4*>(log_sums + row);
      const f32x4 delta = *reinterpret_cast<const f32x4*>(deltas + row);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool there = row + r < count;
        weight[k][r] = there ? exp2_of(weight[k][r] * factor - log_sum[r]) : 0.0f;
        slope[k][r] = there ? weight[k][r] * (slope[k][r] - delta[r]) : 0.0f;
      }
    }
    if constexpr (kNarrow<T>) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(slope[k][r]));
      const float by = follow_range(&unit, over_groups_max(most));
#pragma unroll
      for (int d = 0; d < kCols; ++d) grad_key[d] *= by;
      slope[0] *= unit;
      slope[1] *= unit;
    }
    const Operand<T> weights = operand_of<T>(weight[0], weight[1]);
    const Operand<T> slopes = operand_of<T>(slope[0], slope[1]);
#pragma unroll
    for (int d = 0; d < kCols; ++d) {
      grad_value[d] = mma(column_operand<T, kRows, WIDTH>(grads, row0, d * 16, lane), weights, grad_value[d]);
      grad_key[d] = mma(column_operand<T, kRows, WIDTH>(queries, row0, d * 16, lane), slopes, grad_key[d]);
    }
  }

  // the waves' sums, in their order
  __syncthreads();
  float* sums = reinterpret_cast<float*>(shared);
  const float back = unit == 0.0f ? 1.0f : 1.0f / unit;
  if (wave < kTeams) {
#pragma unroll
    for (int d = 0; d < kCols; ++d) {
      float* at = sums + (wave * 32 + column) * kSumPitch + d * 16 + 4 * group;
      *reinterpret_cast<f32x4*>(at) = grad_key[d] * back;
      *reinterpret_cast<f32x4*>(at + 16 * kSumPitch) = grad_value[d];
    }
  }
  __syncthreads();
  const int columns = a.key_width + a.value_width, there = min(16, a.sinks - first);
  float* piece =
      a.sink_parts + (((sink_place(a, run).piece + run.tile) * a.heads + head) * a.sinks + first) * columns;
  for (int e = tid; e < there * columns; e += kThreads) {
    const int s = e / columns, col = e % columns;
    const int at = col < a.key_width ? s * kSumPitch + col : (16 + s) * kSumPitch + col - a.key_width;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeams; ++w) sum += sums[w * 32 * kSumPitch + at];
    piece[e] = sum;
  }
}

// The pieces of window_grad_sinks_kernel, and the query heads of a group, added up in their order:
// [sequence: sink_place][kv head][sink][key_width + value_width].
template <typename T>
__global__ __launch_bounds__(kThreads) void window_join_sinks_kernel(WindowArgs<T> a) {
  const int tid = threadIdx.x, size = a.sinks * (a.key_width + a.value_width);
  const int blocks = (size + kThreads - 1) / kThreads;
  const uint32_t block = block_number();
  const int sequence = static_cast<int>(block / blocks / a.kv_heads);
  const int kv_head = static_cast<int>(block / blocks % a.kv_heads);
  if (sequence >= a.sequences.count) return;
  const Run run = run_of_sequence(a.sequences, sequence);
  if (run.length <= a.sink_far) return;  // (of length -1: no offsets to rely on)
  const int e = static_cast<int>(block % blocks) * kThreads + tid;
  if (e >= size) return;
  const int first = static_cast<int>(walk_end(0, a.key_block, a.window)) / a.sink_rows;
  const int pieces = tiles_of(run.length, a.sink_rows);
  const SinkPlace place = sink_place(a, run);
  const int64_t slot = place.piece + first;
  const float* part = a.sink_parts + (slot * a.heads + kv_head * a.share) * size + e;
  float sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < (pieces - first) * a.share; ++i)
    sum += part[(static_cast<int64_t>(i / a.share) * a.heads + i % a.share) * size];
  a.sink_sums[(place.sums * a.kv_heads + kv_head) * size + e] = sum;
}

// ---------------------------------------------------------------------------
// serving
// ---------------------------------------------------------------------------

// The new tokens that a cache keeps, each on its row: the sinks and the newest `ring` others.
// Blocks of 64 tokens of one head of keys: 67 MB in and out in 11 us at 4 x 2048 tokens, 8 heads of
// 128, bfloat16.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void window_append_kernel(WindowArgs<T> a, T* key_cache,
                                                                 T* value_cache) {
  const int tid = threadIdx.x;
  const uint32_t block = block_number();
  const int64_t slot = block / a.kv_heads;
  const int kv_head = static_cast<int>(block % a.kv_heads);
  if (slot >= slots_of(a.sequences, 64)) return;
  Run run;
  if (find_run(a.sequences, slot, 64, tid, &run) != Found::kRun) return;
  const int past = tokens_before<true>(a, run);
  const History<T, true> key_rows = history_of<true>(a, a.key, a.key_cache, a.key_width, run, kv_head, past);
  const History<T, true> value_rows =
      history_of<true>(a, a.value, a.value_cache, a.value_width, run, kv_head, past);
  const int begin = past + run.tile * 64, end = min(begin + 64, past + run.length);
  const int64_t oldest = static_cast<int64_t>(past) + run.length - key_rows.rows.ring;
  const int64_t at = (static_cast<int64_t>(run.sequence) * a.kv_heads + kv_head) * a.capacity;
  const auto copy = [&](T* cache, int width, auto&& from) {
    constexpr int kElements = 16 / static_cast<int>(sizeof(T));
    typedef T Piece __attribute__((ext_vector_type(kElements)));
    const int pieces = (width + kElements - 1) / kElements;
    for (int e = tid; e < (end - begin) * pieces; e += kThreads) {
      const int s = begin + e / pieces, col = e % pieces * kElements;
      if (s >= a.sinks && s < oldest) continue;
      T* to = cache + (at + key_rows.rows.row(s)) * width + col;
      const T* source = from(s) + col;
      if constexpr (WHOLE)
        *reinterpret_cast<Piece*>(to) = *reinterpret_cast<const Piece*>(source);
      else
        for (int i = 0; i < kElements && col + i < width; ++i) to[i] = source[i];
    }
  };
  copy(key_cache, a.key_width, [&](int s) { return key_rows.row(s); });
  copy(value_cache, a.value_width, [&](int s) { return value_rows.row(s); });
}

// One new token of every slot against its cache, which is shared out to the blocks of a head of
// keys and, in tiles of 32 keys, to their waves: every wave has a softmax of its own over its
// tiles, with the query heads of the group (up to 16) across; the waves are joined at the end and
// the blocks by window_token_join_kernel.  Bound by the reads of the cache: 64 slots, 8 heads of
// 128, window 4096, bfloat16: 1.07 GB in 175 us, 6.1 TB/s; 1 slot, 2 heads of 64, window 65536: 34 MB
// in 10 us, of which the launch and the first loads are half, and 6 us for the join.
template <typename T>
struct TokenArgs {
  WindowArgs<T> window;
  T *key_cache, *value_cache;
  int splits, head_blocks;
  float* partial;   // [slot][head][split][2 + value_width]: maximum, sum, outputs
};

template <typename T, int WIDTH, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWaves<T, WIDTH, WHOLE>))) void
window_token_kernel(TokenArgs<T> args) {
  constexpr int kSteps = WIDTH / 32, kCols = WIDTH / 16, kTile = 32;
  constexpr int kElements = 16 / static_cast<int>(sizeof(T)), kPerRow = WIDTH / kElements;
  constexpr int kPieces = kTile * kPerRow / 64;
  typedef T Piece __attribute__((ext_vector_type(kElements)));
  const WindowArgs<T>& a = args.window;
  constexpr size_t kTileBytes = sizeof(Stored<T>) * kTileElements<T, kTile, WIDTH>;
  constexpr size_t kJoinBytes = sizeof(float) * 16 * (WIDTH + 4);
  __shared__ __attribute__((aligned(16))) char shared[4 * (kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes)];
  __shared__ float tops[4][16], totals[4][16];

  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Stored<T>* values = reinterpret_cast<Stored<T>*>(shared) + wave * kTileElements<T, kTile, WIDTH>;
  const uint32_t block = block_number();
  const int split = block % args.splits;
  const int head_block = block / args.splits % args.head_blocks;
  const int kv_head = block / args.splits / args.head_blocks % a.kv_heads;
  const int slot = block / args.splits / args.head_blocks / a.kv_heads;
  if (slot >= a.sequences.count) return;
  const Run run{slot, 1, 0, slot, 0, slot};
  const int past = tokens_before<true>(a, run);
  const History<T, true> key_rows = history_of<true>(a, a.key, a.key_cache, a.key_width, run, kv_head, past);
  const History<T, true> value_rows =
      history_of<true>(a, a.value, a.value_cache, a.value_width, run, kv_head, past);

  if (split == 0 && head_block == 0) {  // (the row that it takes is one that nobody sees any more)
    const int64_t at = (static_cast<int64_t>(slot) * a.kv_heads + kv_head) * a.capacity + key_rows.rows.row(past);
    for (int d = tid; d < a.key_width; d += kThreads) args.key_cache[at * a.key_width + d] = key_rows.fresh[d];
    for (int d = tid; d < a.value_width; d += kThreads)
      args.value_cache[at * a.value_width + d] = value_rows.fresh[d];
  }
  // what the token sees, in order: sinks, window, itself
  const int window_begin = max(0, past - a.window + 1), sinks_end = min(a.sinks, window_begin);
  const int seen = sinks_end + past - window_begin + 1;
  const int tiles = (seen + kTile - 1) / kTile;
  const int share = (tiles + args.splits - 1) / args.splits;
  const int tile_end = min(tiles, (split + 1) * share);
  const auto position = [&](int u) { return u < sinks_end ? u : window_begin + u - sinks_end; };

  // this column's member of the group of query heads (the last one again beyond it)
  const int head = kv_head * a.share + min(head_block * 16 + column, a.share - 1);
  const Rows<T> query_row = {a.query.row(slot, 0, head), 0, 0};
  Operand<T> query[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    Frag<T> part = memory_operand<WHOLE>(query_row, 0, s * 32 + 8 * group, a.key_width);
    clear_operand<WHOLE>(part, s * 32, group, a.key_width);
    query[s] = as_operand<T>(part);
  }
  f32x4 out[kCols];
#pragma unroll
  for (int d = 0; d < kCols; ++d) out[d] = f32x4(0.0f);
  float most = -__builtin_inff(), sum = 0.0f;
  const float factor = a.scale * kLog2e;

  Frag<T> key[2][kSteps];
  Piece held[kPieces];
  const auto fetch = [&](int tile) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Rows<T> row = {key_rows.row(position(min(tile * kTile + k * 16 + column, seen - 1))), 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        key[k][s] = memory_operand<WHOLE>(row, 0, s * 32 + 8 * group, a.key_width);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * 64 + lane, col = piece % kPerRow * kElements;
      const T* row = value_rows.row(position(min(tile * kTile + piece / kPerRow, seen - 1)));
      if constexpr (WHOLE) {
        held[i] = *reinterpret_cast<const Piece*>(row + min(col, a.value_width - kElements));
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e) held[i][e] = row[min(col + e, a.value_width - 1)];
      }
    }
  };
  int tile = split * share + wave;
  if (tile < tile_end) fetch(tile);
  for (; tile < tile_end; tile += 4) {
    f32x4 score[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      score[k] = f32x4(0.0f);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        clear_operand<WHOLE>(key[k][s], s * 32, group, a.key_width);
        score[k] = mma(as_operand<T>(key[k][s]), query[s], score[k]);
      }
    }
    // (LDS accesses of one wave are carried out in order: its tile needs no barrier)
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * 64 + lane;
      float part[kElements];
#pragma unroll
      for (int e = 0; e < kElements; ++e) part[e] = static_cast<float>(held[i][e]);
      store_row<T, kTile, WIDTH>(values, piece / kPerRow, piece % kPerRow * kElements, part);
    }
    asm volatile("" ::: "memory");
    if (tile + 4 < tile_end) fetch(tile + 4);
    float here = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (tile * kTile + k * 16 + 4 * group + r >= seen) score[k][r] = -__builtin_inff();
        here = fmaxf(here, score[k][r]);
      }
    here = over_groups_max(here) * factor;
    if (__any(here > most)) {
      const float larger = fmaxf(here, most);
      const float shrink = larger == -__builtin_inff() ? 1.0f : exp2_of(most - larger);
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < kCols; ++d) out[d] *= shrink;
      most = larger;
    }
    const float base = (most == -__builtin_inff() ? 0.0f : most) - kLift<T>;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        score[k][r] = exp2_of(score[k][r] * factor - base);
        sum += score[k][r];
      }
    const Operand<T> weights = operand_of<T>(score[0], score[1]);
#pragma unroll
    for (int d = 0; d < kCols; ++d)
      out[d] = mma(column_operand<T, kTile, WIDTH>(values, 0, d * 16, lane), weights, out[d]);
    asm volatile("" ::: "memory");
  }
  sum = over_groups_sum(sum);

  // the waves of the block
  __syncthreads();
  float* outs = reinterpret_cast<float*>(shared) + wave * 16 * (WIDTH + 4);
#pragma unroll
  for (int d = 0; d < kCols; ++d)
    *reinterpret_cast<f32x4*>(outs + column * (WIDTH + 4) + d * 16 + 4 * group) = out[d];
  if (group == 0) {
    tops[wave][column] = most;
    totals[wave][column] = sum;
  }
  __syncthreads();
  const int members = min(16, a.share - head_block * 16);
  for (int e = tid; e < members * a.value_width; e += kThreads) {
    const int m = e / a.value_width, d = e % a.value_width;
    const float top = fmaxf(fmaxf(tops[0][m], tops[1][m]), fmaxf(tops[2][m], tops[3][m]));
    float total = 0.0f, value = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = top == -__builtin_inff() ? 1.0f : exp2_of(tops[w][m] - top);
      total += by * totals[w][m];
      value += by * (reinterpret_cast<float*>(shared) + w * 16 * (WIDTH + 4))[m * (WIDTH + 4) + d];
    }
    const int64_t row = static_cast<int64_t>(slot) * a.heads + kv_head * a.share + head_block * 16 + m;
    if (args.splits == 1) {
      a.out[row * a.value_width + d] = static_cast<T>(value / total);
    } else {
      float* to = args.partial + (row * args.splits + split) * (2 + a.value_width);
      if (d == 0) {
        to[0] = top;
        to[1] = total;
      }
      to[2 + d] = value;
    }
  }
}

// One block per slot and head: the parts of window_token_kernel, whose weights a thread each forms
// and whose outputs the waves add up in turn.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_token_join_kernel(const float* partial, T* out,
                                                                     int splits, int width) {
  __shared__ float weights[kMostSplits], sums[kThreads], tops[4], totals[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const float* parts = partial + row * splits * (2 + width);
  float top = -__builtin_inff();
  for (int s = tid; s < splits; s += kThreads) {
    weights[s] = parts[static_cast<int64_t>(s) * (2 + width)];
    top = fmaxf(top, weights[s]);
  }
  for (int apart = 1; apart < 64; apart *= 2) top = fmaxf(top, __shfl_xor(top, apart));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float total = 0.0f;
  for (int s = tid; s < splits; s += kThreads) {
    const float by = top == -__builtin_inff() ? 1.0f : exp2_of(weights[s] - top);
    weights[s] = by;
    total += by * parts[static_cast<int64_t>(s) * (2 + width) + 1];
  }
  for (int apart = 1; apart < 64; apart *= 2) total += __shfl_xor(total, apart);
  if (lane == 0) totals[wave] = total;
  __syncthreads();
  total = totals[0] + totals[1] + totals[2] + totals[3];
  for (int col0 = 0; col0 < width; col0 += 64) {
    const int col = col0 + lane;
    float value = 0.0f;
    if (col < width) {
#pragma unroll 8
      for (int s = wave; s < splits; s += 4)
        value += weights[s] * parts[static_cast<int64_t>(s) * (2 + width) + 2 + col];
    }
    sums[tid] = value;
    __syncthreads();
    if (wave == 0 && col < width)
      out[row * width + col] = static_cast<T>((sums[lane] + sums[64 + lane] + sums[128 + lane] +
                                               sums[192 + lane]) / total);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T>
WindowArgs<T> window_args(const WindowCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  WindowArgs<T> args{};
  args.query = view_of<T>(*call.query);
  args.key = view_of<T>(*call.key);
  args.value = view_of<T>(*call.value);
  args.sequences = sequences_of(p);
  args.heads = p.H;
  args.kv_heads = p.Hkv;
  args.share = p.H / p.Hkv;
  args.key_width = p.D;
  args.value_width = p.Dv;
  args.window = call.window;
  args.sinks = call.sinks;
  args.scale = p.scale;
  args.out = static_cast<T*>(call.out);
  args.log_sum = call.log_sum;
  return args;
}

// Tokens (in sixteens) of a wave: two, so that an operand read from LDS serves two products; one
// where two make fewer than kFull blocks, which two rounds of the chip's take (o and dq of 664
// blocks of two: 26.5 and 32.6 us, of 1192 of one: 24.5 and 29.2; of 712: 43 and 64 us, of 1344: 44.6
// and 62.6; of 2048: 195 and 250 us, of 4096 of one: 227 and 296), and where two do not fit the
// registers (float32, 128 columns).
constexpr int64_t kFull = 1024;

template <typename T>
bool whole_rows(const WindowCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  return whole_pieces<T>(*call.query, p.D) && whole_pieces<T>(*call.key, p.D) &&
         whole_pieces<T>(*call.value, p.Dv) &&
         (call.grad_output == nullptr || (whole_pieces<T>(*call.grad_output, p.Dv) &&
                                          whole_stride<T>(static_cast<int64_t>(p.H) * p.Dv))) &&
         whole_address(call.output) && whole_address(call.key_cache) && whole_address(call.value_cache) &&
         whole_address(call.out) && whole_address(call.grad_query) && whole_address(call.grad_key) &&
         whole_address(call.grad_value);
}

template <typename T, int WIDTH, int QUERIES, bool CACHED, bool WHOLE>
void window_forward_launch(WindowArgs<T>& args, hipStream_t stream) {
  args.slots = slots_of(args.sequences, 64 * QUERIES);
  args.items = args.slots * args.heads;
  window_forward_kernel<T, WIDTH, QUERIES, CACHED, WHOLE>
      <<<grid_of_items(args.items), kThreads, 0, stream>>>(args);
}

template <typename T, int WIDTH, bool CACHED, bool WHOLE>
void window_forward_rows(WindowArgs<T>& args, hipStream_t stream) {
  if constexpr (kPairs<T, WIDTH>) {
    if (slots_of(args.sequences, 128) * args.heads >= kFull)
      return window_forward_launch<T, WIDTH, 2, CACHED, WHOLE>(args, stream);
  }
  window_forward_launch<T, WIDTH, 1, CACHED, WHOLE>(args, stream);
}

template <typename T, bool WHOLE>
void window_forward_width(const WindowCall& call) {
  WindowArgs<T> args = window_args<T>(call);
  const rosa_mixer_problem& p = *call.problem;
  switch (padded_width(p.D > p.Dv ? p.D : p.Dv)) {
    case 32: return window_forward_rows<T, 32, false, WHOLE>(args, call.stream);
    case 64: return window_forward_rows<T, 64, false, WHOLE>(args, call.stream);
    default: return window_forward_rows<T, 128, false, WHOLE>(args, call.stream);
  }
}

template <typename T>
void window_forward(const WindowCall& call) {
  if (whole_rows<T>(call))
    window_forward_width<T, true>(call);
  else
    window_forward_width<T, false>(call);
}

template <typename T, int WIDTH, int QUERIES, bool WHOLE, bool DELTA>
void window_grad_query_launch(WindowArgs<T>& args, hipStream_t stream) {
  args.slots = slots_of(args.sequences, 64 * QUERIES);
  args.items = args.slots * args.heads;
  window_grad_query_kernel<T, WIDTH, QUERIES, WHOLE, DELTA>
      <<<grid_of_items(args.items), kThreads, 0, stream>>>(args);
}

template <typename T, int WIDTH, int KEYS, bool WHOLE>
void window_grad_key_launch(WindowArgs<T>& args, hipStream_t stream) {
  if (args.sink_slots > 0) {
    args.items = args.sink_slots * args.heads * ((args.sinks + 15) / 16);
    window_grad_sinks_kernel<T, WIDTH, WHOLE>
        <<<grid_of_items(args.items), kThreads, 0, stream>>>(args);
    const int size = args.sinks * (args.key_width + args.value_width);
    window_join_sinks_kernel<T>
        <<<grid_of(static_cast<int64_t>((size + kThreads - 1) / kThreads) * args.kv_heads *
                   args.sequences.count),
           kThreads, 0, stream>>>(args);
  }
  args.slots = slots_of(args.sequences, args.key_block);
  args.items = args.slots * args.kv_heads * args.key_parts;
  window_grad_key_kernel<T, WIDTH, KEYS, WHOLE>
      <<<grid_of_items(args.items), kThreads, 0, stream>>>(args);
  if (args.key_parts == 1) return;
  const auto join = [&](const float* parts, T* out, int width) {
    if (out == nullptr) return;
    const int64_t elements = static_cast<int64_t>(args.sequences.tokens) * args.kv_heads * width;
    window_join_keys_kernel<T><<<grid_of((elements + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
        parts, out, args.key_parts, elements);
  };
  join(args.key_sums, args.grad_key, args.key_width);
  join(args.value_sums, args.grad_value, args.value_width);
}

template <typename T, int WIDTH, bool WHOLE>
void window_backward_launch(WindowArgs<T>& args, hipStream_t stream) {
  constexpr int kMost = kPairs<T, WIDTH> ? 2 : 1;
  const bool pairs = slots_of(args.sequences, 128) * args.heads >= kFull;
  if constexpr (sizeof(T) == 2) {
    if (args.exact_delta && pairs)
      window_grad_query_launch<T, WIDTH, 2, WHOLE, true>(args, stream);
    else if (args.exact_delta)
      window_grad_query_launch<T, WIDTH, 1, WHOLE, true>(args, stream);
  }
  if (kMost == 2 && pairs)
    window_grad_query_launch<T, WIDTH, kMost, WHOLE, false>(args, stream);
  else
    window_grad_query_launch<T, WIDTH, 1, WHOLE, false>(args, stream);
  if (args.grad_key == nullptr && args.grad_value == nullptr) return;
  if (kPairs<T, WIDTH> && args.key_block == 128)
    window_grad_key_launch<T, WIDTH, kPairs<T, WIDTH> ? 2 : 1, WHOLE>(args, stream);
  else
    window_grad_key_launch<T, WIDTH, 1, WHOLE>(args, stream);
}

template <typename T, bool WHOLE>
void window_backward_width(const WindowCall& call) {
  WindowArgs<T> args = window_args<T>(call);
  const rosa_mixer_problem& p = *call.problem;
  const WindowPlan plan = window_plan(p, call.window, call.sinks);
  args.grad_output = view_of<T>(*call.grad_output);
  args.output = static_cast<const T*>(call.output);
  args.delta = reinterpret_cast<float*>(call.workspace);
  args.grad_query = static_cast<T*>(call.grad_query);
  args.grad_key = static_cast<T*>(call.grad_key);
  args.grad_value = static_cast<T*>(call.grad_value);
  args.sink_slots = plan.sink_slots;
  args.sink_rows = plan.sink_rows;
  args.sink_far = plan.sink_far;
  args.exact_delta = sizeof(T) == 2 && few_seen(call.window, p.cu_seqlens == nullptr ? p.T : p.N / p.S);
  args.key_block = plan.key_block;
  args.key_parts = plan.key_parts;
  if (plan.key_parts > 1) {
    char* sums = call.workspace + plan.delta_bytes + plan.sink_bytes + plan.sink_part_bytes;
    args.key_sums = reinterpret_cast<float*>(sums);
    args.value_sums = reinterpret_cast<float*>(sums + plan.key_sum_bytes);
  }
  if (plan.sink_slots > 0) {
    args.sink_sums = reinterpret_cast<float*>(call.workspace + plan.delta_bytes);
    args.sink_parts = reinterpret_cast<float*>(call.workspace + plan.delta_bytes + plan.sink_bytes);
  }
  switch (padded_width(p.D > p.Dv ? p.D : p.Dv)) {
    case 32: return window_backward_launch<T, 32, WHOLE>(args, call.stream);
    case 64: return window_backward_launch<T, 64, WHOLE>(args, call.stream);
    default: return window_backward_launch<T, 128, WHOLE>(args, call.stream);
  }
}

template <typename T>
void window_backward(const WindowCall& call) {
  if (whole_rows<T>(call))
    window_backward_width<T, true>(call);
  else
    window_backward_width<T, false>(call);
}

template <typename T, int WIDTH, bool WHOLE>
void window_update_launch(WindowArgs<T>& args, const WindowCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  T* key_cache = static_cast<T*>(call.key_cache);
  T* value_cache = static_cast<T*>(call.value_cache);
  if (p.cu_seqlens == nullptr && p.T == 1) {
    const TokenPlan plan = token_plan(p, call.capacity);
    TokenArgs<T> token{args, key_cache, value_cache, plan.splits, plan.head_blocks,
                       reinterpret_cast<float*>(call.workspace)};
    const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * plan.head_blocks * plan.splits;
    window_token_kernel<T, WIDTH, WHOLE><<<grid_of(blocks), kThreads, 0, call.stream>>>(token);
    if (plan.splits > 1)  // (of few slots)
      window_token_join_kernel<T><<<dim3(static_cast<unsigned>(p.B) * p.H), kThreads, 0, call.stream>>>(
          token.partial, args.out, plan.splits, p.Dv);
    return;
  }
  window_forward_rows<T, WIDTH, true, WHOLE>(args, call.stream);
  const int64_t blocks = slots_of(args.sequences, 64) * p.Hkv;
  window_append_kernel<T, WHOLE>
      <<<grid_of(blocks), kThreads, 0, call.stream>>>(args, key_cache, value_cache);
}

template <typename T, bool WHOLE>
void window_update_width(const WindowCall& call) {
  WindowArgs<T> args = window_args<T>(call);
  const rosa_mixer_problem& p = *call.problem;
  args.key_cache = static_cast<const T*>(call.key_cache);
  args.value_cache = static_cast<const T*>(call.value_cache);
  args.lengths = call.lengths;
  args.capacity = call.capacity;
  switch (padded_width(p.D > p.Dv ? p.D : p.Dv)) {
    case 32: return window_update_launch<T, 32, WHOLE>(args, call);
    case 64: return window_update_launch<T, 64, WHOLE>(args, call);
    default: return window_update_launch<T, 128, WHOLE>(args, call);
  }
}

template <typename T>
void window_update(const WindowCall& call) {
  if (whole_rows<T>(call))
    window_update_width<T, true>(call);
  else
    window_update_width<T, false>(call);
}

}  // namespace rosa_mixer
