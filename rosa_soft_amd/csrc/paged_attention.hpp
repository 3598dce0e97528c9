// Attention of new tokens over a paged cache: position p of a slot lies on row p mod P of page
// table[p / P], with P a power of two from 16 on, so that 16 neighbouring positions from a multiple of
// 16 on are 16 neighbouring rows.
//
//   p = softmax_s(scale q_t . k_s) over s <= t (or those of them on selected pages),  o_t = sum_s p_s v_s
//
// The query heads of a group share keys and values: the rows of a slot are its (token, member of the
// group) pairs, member fastest, whatever the number of either.  Slots of up to 16 rows (single tokens,
// short drafts) are bound by the reads of the cache and have paged_token_kernel, in which the waves
// of a block share out keys; the others are bound by matrix products and have paged_chunk_kernel, in
// which they share out rows and keys go through LDS.
//
// Neither the host nor a launch knows the slots' lengths.  Every block reads all of them and works out
// by itself how the call is cut into portions of about the same number of keys, and which is its own
// (portion_of); tiles that are cut leave partial sums to the paged_join kernels.
#pragma once

#include "attention_device.hpp"
#include "paged_calls.hpp"

#include <algorithm>

namespace rosa_mixer {

// A tile of rows whose keys are shared out to several portions.
struct PagedTask {
  int64_t first;              // token of the slot's first row
  int row, rows, part, splits;
};

struct PagedDivision {
  int target, least, most_few, round;
  int64_t parts;              // of a head of keys: what two of them are apart in `partial`
  float* partial;             // [kv head][part][row][width + 4]: outputs, maximum, sum
  PagedTask* tasks;
  int* task_count;
};

template <typename T>
struct PagedArgs {
  View<const T> query, key, value;
  T* out;                     // [tokens][heads][value_width]
  T *key_pages, *value_pages, *key_bounds;
  const int32_t *tables, *lengths;
  const int64_t* rows;
  Sequences sequences;
  int pages, columns, page_shift;
  int heads, kv_heads, share, key_width, value_width;
  float scale;
  bool fused;                 // the kernels that attend put new tokens on their rows
  PagedDivision division;
  // selected pages
  double* scores;             // [token of the slab][kv head][column]
  int32_t *lists, *seen;      // [token][kv head][count + 1], [token][kv head]
  int count, list_splits;
  int64_t slab_first, slab_tokens;

  __device__ __forceinline__ int64_t capacity() const { return static_cast<int64_t>(columns) << page_shift; }
  __device__ __forceinline__ bool is_page(int id) const { return static_cast<uint32_t>(id) < static_cast<uint32_t>(pages); }
  // row of a page's head in the pools
  __device__ __forceinline__ int64_t place(int id, int kv_head, int offset) const {
    return ((static_cast<int64_t>(id) * kv_heads + kv_head) << page_shift) + offset;
  }
  // the row that a new token is put on, or -1
  __device__ __forceinline__ int64_t row_of(int64_t token) const {
    const int64_t row = rows[token];
    return row >= 0 && row < static_cast<int64_t>(pages) << page_shift ? row : -1;
  }
};

// ---------------------------------------------------------------------------
// sharing out
// ---------------------------------------------------------------------------

struct SlotWork {
  int begin, fresh, past, tiles, walk;  // first new token, new ones, earlier ones; tiles of rows, of keys
};

// ROWS, KEYS: of a tile.  FEW: slots of up to `most_few` rows, or the others.
template <int ROWS, int KEYS, bool FEW, typename T>
__device__ __forceinline__ SlotWork slot_work(const PagedArgs<T>& a, int s, int* bad) {
  SlotWork w;
  const Sequences& q = a.sequences;
  if (q.offsets == nullptr) {
    w.begin = 0;
    w.fresh = q.length;
  } else {
    const int end = q.offsets[s + 1];
    w.begin = q.offsets[s];
    *bad |= w.begin > end || (s == 0 && w.begin != 0) || (s == q.count - 1 && end != q.tokens);
    w.fresh = w.begin < 0 || end > q.tokens ? 0 : max(0, end - w.begin);
  }
  w.past = max(0, min(a.lengths[s], 0x7fffffff - 1024 - w.fresh));
  const int rows = w.fresh * a.share;
  w.tiles = w.fresh > 0 && (rows <= a.division.most_few) == FEW ? (rows - 1) / ROWS + 1 : 0;
  const int64_t end = min(static_cast<int64_t>(w.past) + w.fresh, a.capacity());
  w.walk = static_cast<int>((end + KEYS - 1) / KEYS);
  return w;
}

struct Portion {
  SlotWork work;
  int slot, kv_head, tile, split, splits, part, task;
};

// Inclusive sum over the lanes of a wave: within rows of 16 lanes, then the last lane of a row to the
// next one, and that of the first half to the second.
__device__ __forceinline__ int scan_wave(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // from 1 lane before
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);  // 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);  // 4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);  // 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);  // lane 15 of rows 0 and 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);  // lane 31
  return x;
}
// The sum over a wave of numbers below 2^62.
__device__ __forceinline__ int64_t over_wave_sum(int64_t x) {
  int64_t sum = 0;
#pragma unroll
  for (int shift = 0; shift < 64; shift += 24)  // (64 of 24 bits fit 32)
    sum += static_cast<int64_t>(__builtin_amdgcn_readlane(scan_wave(static_cast<int>(x >> shift & 0xffffff)), 63))
           << shift;
  return sum;
}

// Which head and which of its `total` portions a block works on; -1: none.  FEW: neighbouring blocks
// have neighbouring heads, which lie side by side on a page.  Otherwise blocks of the same keys, which
// are neighbours among a head's portions, go to the same XCD.
template <bool FEW>
__device__ __forceinline__ int64_t portion_number(int64_t total, int kv_heads, int* kv_head) {
  const uint32_t block = block_number();
  if constexpr (FEW) {
    *kv_head = static_cast<int>(block % kv_heads);
    const int64_t item = block / kv_heads;
    return item < total ? item : -1;
  } else {
    const int64_t item = item_of_block(total * kv_heads);
    if (item >= total * kv_heads) return -1;
    *kv_head = static_cast<int>(item / total);
    return item % total;
  }
}

// Number `at` among the portions of a slot.
template <bool FEW>
__device__ __forceinline__ void place_portion(Portion* p, int at, int parts_before, int tasks_before) {
  const int tiles = p->work.tiles;
  if constexpr (FEW) {
    p->split = at % p->splits;
    p->tile = at / p->splits;
  } else {  // late tiles, which see most, first
    p->split = at / tiles;
    p->tile = tiles - 1 - at % tiles;
  }
  p->part = parts_before + p->tile * p->splits + p->split;
  p->task = tasks_before + p->tile;
}

// The portion of a block.  All portions of a call together have `all` = sum over its slots of (tiles of
// rows) (tiles of keys); one has at most all / target of them, or `least`, so that a head of keys has
// about `target` portions more than tiles of rows, however the slots' lengths differ.  Up to 64 slots
// every wave looks at all of them by itself, a slot to a lane; beyond, the threads of the block have
// neighbouring slots each.
template <int ROWS, int KEYS, bool FEW, typename T>
__device__ __forceinline__ Found portion_of(const PagedArgs<T>& a, int tid, Portion* p) {
  const PagedDivision& d = a.division;
  const int count = a.sequences.count, lane = tid & 63, wave = tid >> 6;
  // (no walk is as long as 2^27 tiles)
  const auto portion_length = [&](int64_t all) {
    return static_cast<int>(min(max(static_cast<int64_t>(d.least), (all + d.target - 1) / d.target), int64_t{1} << 27));
  };
  const auto splits_of = [&](const SlotWork& w, int length) {
    return w.tiles > 0 ? max(1, (w.walk + length * d.round / 8) / length) : 0;
  };
  const auto note_tasks = [&](int tasks) {
    if (block_number() == 0 && tid == 0 && d.task_count != nullptr) *d.task_count = tasks;
  };
  if (count <= 64) {
    int bad = 0;
    SlotWork w{};
    if (lane < count) w = slot_work<ROWS, KEYS, FEW>(a, lane, &bad);
    if (__any(bad)) {
      note_tasks(0);
      return Found::kInvalid;
    }
    const int length = portion_length(over_wave_sum(static_cast<int64_t>(w.tiles) * w.walk));
    const int splits = splits_of(w, length), items = w.tiles * splits;
    const int upto = scan_wave(items), total = __builtin_amdgcn_readlane(upto, 63);
    const int parts = scan_wave(splits > 1 ? items : 0);
    const int tasks = scan_wave(splits > 1 ? w.tiles : 0);
    note_tasks(__builtin_amdgcn_readlane(tasks, 63));
    const int64_t item = portion_number<FEW>(total, a.kv_heads, &p->kv_head);
    if (item < 0) return Found::kNothing;
    const int slot = __popcll(__ballot(upto <= item));
    const auto of_slot = [&](int x) { return __builtin_amdgcn_readlane(x, slot); };
    p->slot = slot;
    p->work = {of_slot(w.begin), of_slot(w.fresh), of_slot(w.past), of_slot(w.tiles), of_slot(w.walk)};
    p->splits = of_slot(splits);
    const bool cut = p->splits > 1;
    const int all = of_slot(items);
    place_portion<FEW>(p, static_cast<int>(item) - (of_slot(upto) - all),
                       of_slot(parts) - (cut ? all : 0), of_slot(tasks) - (cut ? p->work.tiles : 0));
    return Found::kRun;
  }
  constexpr int kAll = kThreads / 64;
  __shared__ int64_t sums[kAll];
  __shared__ int ends[3][kAll];
  __shared__ Portion found;
  const int per = (count + kThreads - 1) / kThreads;
  const int from = min(count, tid * per), to = min(count, from + per);
  int bad = 0;
  int64_t all = 0;
  for (int s = from; s < to; ++s) {
    const SlotWork w = slot_work<ROWS, KEYS, FEW>(a, s, &bad);
    all += static_cast<int64_t>(w.tiles) * w.walk;
  }
  all = over_wave_sum(all);
  if (lane == 0) sums[wave] = all;
  if (__syncthreads_or(bad)) {
    note_tasks(0);
    return Found::kInvalid;
  }
  all = 0;
  for (int w = 0; w < kAll; ++w) all += sums[w];
  const int length = portion_length(all);
  int mine[3] = {0, 0, 0};
  for (int s = from; s < to; ++s) {
    const SlotWork w = slot_work<ROWS, KEYS, FEW>(a, s, &bad);
    const int splits = splits_of(w, length), items = w.tiles * splits;
    mine[0] += items;
    mine[1] += splits > 1 ? items : 0;
    mine[2] += splits > 1 ? w.tiles : 0;
  }
  int before[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int upto = scan_wave(mine[i]);
    if (lane == 63) ends[i][wave] = upto;
    before[i] = upto - mine[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    total[i] = 0;
    for (int w = 0; w < kAll; ++w) {
      if (w == wave) before[i] += total[i];
      total[i] += ends[i][w];
    }
  }
  note_tasks(total[2]);
  int kv_head = 0;
  const int64_t item = portion_number<FEW>(total[0], a.kv_heads, &kv_head);
  if (item < 0) return Found::kNothing;
  if (item >= before[0] && item < before[0] + mine[0]) {
    for (int s = from; s < to; ++s) {
      const SlotWork w = slot_work<ROWS, KEYS, FEW>(a, s, &bad);
      const int splits = splits_of(w, length), items = w.tiles * splits;
      if (item < before[0] + items) {
        Portion here;
        here.work = w;
        here.slot = s;
        here.kv_head = kv_head;
        here.splits = splits;
        place_portion<FEW>(&here, static_cast<int>(item - before[0]), before[1], before[2]);
        found = here;
        break;
      }
      before[0] += items;
      before[1] += splits > 1 ? items : 0;
      before[2] += splits > 1 ? w.tiles : 0;
    }
  }
  __syncthreads();
  *p = found;
  return Found::kRun;
}

// The last of `count` slots that `begins` is true of, from slot 0 on, of which it is: among 64 times as many
// with every look at them.
template <typename Begins>
__device__ __forceinline__ int last_slot(int count, int lane, Begins&& begins) {
  int slot = 0, left = count;  // it is one of [slot, slot + left)
  while (left > 1) {
    const int step = (left + 63) / 64, end = (lane + 1) * step;
    const int before = __popcll(__ballot(end < left && begins(slot + end)));
    slot += before * step;
    left = min(step, left - before * step);
  }
  return slot;
}
// The slot of a new token.  (Offsets that decrease make it some slot.)
template <typename T>
__device__ __forceinline__ int slot_of_token(const PagedArgs<T>& a, int token, int lane) {
  const Sequences& q = a.sequences;
  if (q.offsets == nullptr) return token / q.length;
  return last_slot(q.count, lane, [&](int s) { return q.offsets[s] <= token; });
}
template <typename T>
__device__ __forceinline__ int past_of(const PagedArgs<T>& a, int slot, int fresh) {
  return max(0, min(a.lengths[slot], 0x7fffffff - 1024 - fresh));
}
template <typename T>
__device__ __forceinline__ int position_of(const PagedArgs<T>& a, int token, int slot) {
  const Sequences& q = a.sequences;
  const int begin = q.offsets == nullptr ? slot * q.length : q.offsets[slot];
  const int fresh = q.offsets == nullptr ? q.length : q.offsets[slot + 1] - begin;
  return past_of(a, slot, max(0, min(fresh, q.tokens))) + max(0, token - begin);
}

template <int THREADS = kThreads, typename T>
__device__ __forceinline__ bool offsets_valid(const PagedArgs<T>& a, int tid) {
  const Sequences& q = a.sequences;
  if (q.offsets == nullptr) return true;
  int bad = 0;
  for (int s = tid; s < q.count; s += THREADS) {
    const int begin = q.offsets[s], end = q.offsets[s + 1];
    bad |= begin > end || (s == 0 && begin != 0) || (s == q.count - 1 && end != q.tokens);
  }
  return !__syncthreads_or(bad);
}

// ---------------------------------------------------------------------------
// new tokens
// ---------------------------------------------------------------------------

// The least and the largest of what they are, or NaN where any of it is.
__device__ __forceinline__ float lower_of(float a, float b) { return b < a || b != b ? b : a; }
__device__ __forceinline__ float higher_of(float a, float b) { return b > a || b != b ? b : a; }

// Pages that a chunk touches for a head, at most: `each` of a slot, or in the order of packed slots, whose
// pages begin at as many as the tokens before them fill whole, and two for each slot before.  (Blocks are
// limited so that those of all heads are below 2^28.)
__host__ __device__ __forceinline__ uint32_t pages_of_slot(int tokens, int page_shift) {
  return static_cast<uint32_t>((tokens - 1) >> page_shift) + 2;
}
template <typename T>
__host__ __device__ __forceinline__ uint32_t pages_touched(const PagedArgs<T>& a) {
  const Sequences& q = a.sequences;
  const auto count = static_cast<uint32_t>(q.count);
  return q.offsets == nullptr ? count * pages_of_slot(q.length, a.page_shift)
                              : static_cast<uint32_t>(q.tokens >> a.page_shift) + 2 * count;
}

// The new tokens on their rows, and the bounds of the pages that they lie on.  A block has one page of
// one slot and head at a time: no other one changes its bounds.  Only where bounds are kept, or pages
// selected, of several tokens or packed ones: otherwise the kernels that attend (for groups of up to 16
// members where there are bounds) or that score (for more columns than are selected) put tokens on
// their rows, which spares a launch (64 slots' single tokens: 294 us before, 281 since).  Latency is all of
// it: 173 packed tokens of 6 slots, 4 heads of 96 columns, 9.0 us.  Blocks by what is touched, which go on to
// further pages: with a block for each slot, head and page that all tokens together may touch, 1024 packed
// single tokens took 1350 us with their attention, 460 since.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedArgs<T> a) {
  __shared__ float lows[kMostWidth], highs[kMostWidth];
  __shared__ uint64_t stored[kThreads / 64];  // which tokens of the page have a row
  __shared__ int number_of_page;
  const int tid = threadIdx.x, page = 1 << a.page_shift;
  if (!offsets_valid(a, tid)) return;
  constexpr int kElements = 16 / static_cast<int>(sizeof(T));
  typedef T Piece __attribute__((ext_vector_type(kElements)));
  const Sequences& q = a.sequences;
  const uint32_t heads = static_cast<uint32_t>(a.kv_heads), items = pages_touched(a) * heads;
  const uint32_t each = q.offsets == nullptr ? pages_of_slot(q.length, a.page_shift) : 1;
  for (uint32_t at = blockIdx.x; at < items; at += gridDim.x) {
    const uint32_t item = at / heads;
    const int kv_head = static_cast<int>(at % heads);
    const int slot = q.offsets == nullptr
                         ? static_cast<int>(item / each)
                         : last_slot(q.count, tid & 63, [&](int s) {
                             return static_cast<uint32_t>(q.offsets[s] >> a.page_shift) + 2 * s <= item;
                           });
    const Run run = run_of_sequence(q, slot);
    if (run.length < 1) continue;
    // of a page among those that the slot's new tokens touch
    const int64_t number = q.offsets == nullptr ? item % each : item - (run.begin >> a.page_shift) - 2 * slot;
    const int past = past_of(a, slot, run.length);
    const T* keys = a.key.row(run.batch, run.begin, kv_head);
    const T* values = a.value.row(run.batch, run.begin, kv_head);
    const int64_t start = ((static_cast<int64_t>(past) >> a.page_shift) + number) << a.page_shift;
    if (start >= static_cast<int64_t>(past) + run.length) continue;
    // new tokens [begin, end) of the slot
    const int begin = static_cast<int>(max(start - past, int64_t{0}));
    const int end = static_cast<int>(min(start + page - past, static_cast<int64_t>(run.length)));
    const auto copy = [&](T* pages, int width, const T* from, int64_t stride) {
      const int pieces = (width + kElements - 1) / kElements;
      for (int e = tid; e < (end - begin) * pieces; e += kThreads) {
        const int token = begin + e / pieces, col = e % pieces * kElements;
        const int64_t row = a.row_of(run.first + token);
        if (row < 0) continue;
        const int id = static_cast<int>(row >> a.page_shift), offset = static_cast<int>(row & (page - 1));
        T* to = pages + a.place(id, kv_head, offset) * width + col;
        const T* source = from + token * stride + col;
        if constexpr (WHOLE)
          *reinterpret_cast<Piece*>(to) = *reinterpret_cast<const Piece*>(source);
        else
          for (int i = 0; i < kElements && col + i < width; ++i) to[i] = source[i];
      }
    };
    copy(a.key_pages, a.key_width, keys, a.key.token_stride);
    copy(a.value_pages, a.value_width, values, a.value.token_stride);
    // (padding is on no page, and has no part in its bounds; a page has at most as many as threads)
    const int64_t row = tid < end - begin ? a.row_of(run.first + begin + tid) : -1;
    const uint64_t put = __ballot(row >= 0);
    if ((tid & 63) == 0) stored[tid >> 6] = put;
    if (row >= 0) number_of_page = static_cast<int>(row >> a.page_shift);
    if (!__syncthreads_or(row >= 0)) continue;
    T* bounds = a.key_bounds + (static_cast<int64_t>(number_of_page) * a.kv_heads + kv_head) * 2 * a.key_width;
    const int d = tid & (kMostWidth - 1), half = tid / kMostWidth;
    float low = __builtin_inff(), high = -__builtin_inff();
    if (d < a.key_width) {
#pragma unroll 4
      for (int token = begin + half; token < end; token += 2) {
        const float x = static_cast<float>(keys[token * a.key.token_stride + d]);
        if (stored[(token - begin) >> 6] >> (token - begin & 63) & 1) {
          low = lower_of(low, x);
          high = higher_of(high, x);
        }
      }
      if (half == 1) {
        lows[d] = low;
        highs[d] = high;
      }
    }
    __syncthreads();
    if (half == 0 && d < a.key_width) {
      low = lower_of(low, lows[d]);
      high = higher_of(high, highs[d]);
      if (start < past) {
        low = lower_of(low, static_cast<float>(bounds[d]));
        high = higher_of(high, static_cast<float>(bounds[a.key_width + d]));
      }
      bounds[d] = static_cast<T>(low);
      bounds[a.key_width + d] = static_cast<T>(high);
    }
    __syncthreads();
  }
}

// The tokens whose first row is among [row0, row0 + rows) of a slot, on their rows.  (What a call reads
// of the pages are earlier tokens: no other block waits for these.)
template <bool WHOLE, typename T>
__device__ __forceinline__ void put_tokens(const PagedArgs<T>& a, const T* keys, const T* values, int64_t first,
                                           int kv_head, int row0, int rows, int tid) {
  constexpr int kElements = 16 / static_cast<int>(sizeof(T));
  typedef T Piece __attribute__((ext_vector_type(kElements)));
  const int begin = (row0 + a.share - 1) / a.share, end = (row0 + rows + a.share - 1) / a.share;
  const int key_pieces = (a.key_width + kElements - 1) / kElements;
  const int pieces = key_pieces + (a.value_width + kElements - 1) / kElements;
  for (int e = tid; e < (end - begin) * pieces; e += kThreads) {
    const int token = begin + e / pieces, piece = e % pieces;
    const int64_t row = a.row_of(first + token);
    if (row < 0) continue;
    const bool is_key = piece < key_pieces;
    const int width = is_key ? a.key_width : a.value_width;
    const int col = (is_key ? piece : piece - key_pieces) * kElements;
    T* to = (is_key ? a.key_pages : a.value_pages) + col +
            a.place(static_cast<int>(row >> a.page_shift), kv_head,
                    static_cast<int>(row & ((1 << a.page_shift) - 1))) * width;
    const T* from = is_key ? keys + token * a.key.token_stride : values + token * a.value.token_stride;
    if constexpr (WHOLE)
      *reinterpret_cast<Piece*>(to) = *reinterpret_cast<const Piece*>(from + col);
    else
      for (int i = 0; i < kElements && col + i < width; ++i) to[i] = from[col + i];
  }
}

// Clears 16 bytes of a value that are not all finite; whether they were not.  A weight of zero would make
// NaN of them, in rows that do not see them as well: in tiles that not all rows see they are cleared, and
// rows from their position on become NaN.  (Paid once a block, by the tiles on the diagonal.  Numbers
// without their sign rank like whole ones: one comparison for all of them.)  The first of a float32's
// three bfloat16 parts is infinite from 2^128 - 2^119 on, the middle between bfloat16's largest number
// and 2^128, and the others are no numbers: float32 counts from there on.
template <typename T, typename Piece>
__device__ __forceinline__ bool clear_wild(Piece& piece) {
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  const Words words = __builtin_bit_cast(Words, piece);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most = max(most, words[i] & 0x7fffffff);
    if constexpr (sizeof(T) == 2) most = max(most, words[i] << 16 & 0x7fffffff);
  }
  const bool wild = most >= (std::is_same_v<T, _Float16> ? 0x7c000000u : sizeof(T) == 4 ? 0x7f7f8000u : 0x7f800000u);
  if (wild) piece = Piece(static_cast<T>(0.0f));
  return wild;
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

// A tile of 16 rows of a slot and head of keys over a portion of its keys, in tiles of 32 that
// the waves take in turn; every wave has a softmax of its own, and the waves are joined at the end.
// Keys go from memory to the operands of the products, values through LDS, which transposes them.
// With `lists` the keys are those of the pages in a token's list, one behind the other.
//
// Every key and value is read once for all members of the group, a tile ahead of its use, and reads are
// what bounds it (2 GiB are read at 5.8 TB/s, copied at 4.9): 64 slots of up to 9000 tokens, 8 heads of
// 128, bf16, 1395 MB in 264 us, 5.3 TB/s; two slots of up to 200000, 2 heads of 64, fp16, 197 MB in 34 us,
// 5.9 TB/s; 33 pages of 64 for each of 32 slots, 8 heads of 128, 274 MB in 45 us, 6.1 TB/s.  In float32,
// whose operands are split in registers, 64 slots of up to 4500 tokens take 386 us (3.6 TB/s, one wave to a
// SIMD), of 9000 with 64 columns 303 (4.6 TB/s).  One slot of 512 tokens in float32 takes 8.6 us: the way
// from the lengths to the table, the page and through the waves' softmaxes.
// Weights are summed in float32 as they are, and rounded to the inputs' type as operands of the product with
// the values: a result is off by half a step of them at most.  (paged_chunk_kernel sums them as rounded, a
// product with ones: by a whole one at most, and by none where one weight is all.)
// Waves have keys of their own because 16 rows are one operand: sharing rows out would leave three of
// them without work.  Two sixteens of rows (drafts of 5 tokens, 4 heads on one) took 62 us, and the
// kernel for many rows takes 49.
template <typename T, int WIDTH, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWaves<T, WIDTH, WHOLE>))) void
paged_token_kernel(PagedArgs<T> a) {
  constexpr int kSteps = WIDTH / 32, kCols = WIDTH / 16, kTile = 32, kRows = 16;
  constexpr int kElements = 16 / static_cast<int>(sizeof(T)), kPerRow = WIDTH / kElements;
  constexpr int kPieces = kTile * kPerRow / 64, kPieceRows = 64 / kPerRow;
  constexpr int kOuts = WIDTH + 4;
  typedef T Piece __attribute__((ext_vector_type(kElements)));
  constexpr size_t kTileBytes = sizeof(Stored<T>) * kTileElements<T, kTile, WIDTH>;
  constexpr size_t kJoinBytes = sizeof(float) * kRows * kOuts;
  __shared__ __attribute__((aligned(16))) char shared[4 * (kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes)];
  __shared__ float tops[4][kRows], totals[4][kRows];
  __shared__ int wild_from[4];  // position of a wave's first value that is not finite, where keys are masked

  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Stored<T>* tile_values = reinterpret_cast<Stored<T>*>(shared) + wave * kTileElements<T, kTile, WIDTH>;

  // what the block works on: rows [row0, row0 + rows) of the tokens behind `first`
  int kv_head, row0, rows, split, splits, part, task, past, last;
  int64_t first, batch, begin;
  const int32_t* table;
  bool void_rows = false;  // nothing can be said of these tokens
  if (a.lists != nullptr) {
    const uint32_t block = block_number();
    const int tiles = (a.share + kRows - 1) / kRows;
    kv_head = static_cast<int>(block % a.kv_heads);
    const int64_t item = block / a.kv_heads;
    split = static_cast<int>(item % a.list_splits);
    splits = a.list_splits;
    const int tile = static_cast<int>(item / splits % tiles);
    first = item / splits / tiles;
    if (first >= a.sequences.tokens) return;
    if (block == 0 && tid == 0 && splits > 1) *a.division.task_count = a.sequences.tokens * tiles;
    task = static_cast<int>(first) * tiles + tile;
    part = task * splits + split;
    row0 = tile * kRows;
    rows = min(kRows, a.share - row0);
    const bool packed = a.sequences.offsets != nullptr;
    batch = packed ? 0 : first / a.sequences.length;
    begin = packed ? first : first % a.sequences.length;
    const int64_t at = first * a.kv_heads + kv_head;
    table = a.lists + at * (a.count + 1);
    last = a.seen[at] - 1;
    void_rows = last < 0;
    past = last;
  } else {
    Portion p;
    const Found found = portion_of<kRows, kTile, true>(a, tid, &p);
    if (found != Found::kRun) return;  // (invalid offsets: paged_chunk_kernel says so)
    kv_head = p.kv_head;
    row0 = p.tile * kRows;
    rows = min(kRows, p.work.fresh * a.share - row0);
    split = p.split;
    splits = p.splits;
    part = p.part;
    task = p.task;
    past = p.work.past;
    const bool packed = a.sequences.offsets != nullptr;
    batch = packed ? 0 : p.slot;
    begin = p.work.begin;
    first = packed ? p.work.begin : static_cast<int64_t>(p.slot) * a.sequences.length;
    table = a.tables + static_cast<int64_t>(p.slot) * a.columns;
    last = static_cast<int>(min(static_cast<int64_t>(past) + (row0 + rows - 1) / a.share, a.capacity() - 1));
  }
  const bool single = a.lists != nullptr;
  if (splits > 1 && split == 0 && kv_head == 0 && tid == 0)
    a.division.tasks[task] = {first, row0, rows, part, splits};

  const T* fresh_key = a.key.row(batch, begin, kv_head);
  const T* fresh_value = a.value.row(batch, begin, kv_head);
  // (in lists every key is on a page: no token sees one behind its own)
  const int fresh_from = single ? 0x7fffffff : past;
  if (a.fused && split == 0) {
    put_tokens<WHOLE>(a, fresh_key, fresh_value, first, kv_head, row0, rows, tid);
    if (a.key_bounds != nullptr && row0 == 0) {  // (of single tokens)
      const int64_t row = a.row_of(first);
      if (row >= 0) {
        T* low = a.key_bounds + ((row >> a.page_shift) * a.kv_heads + kv_head) * 2 * a.key_width;
        T* high = low + a.key_width;
        const bool alone = (past & ((1 << a.page_shift) - 1)) == 0;
        for (int d = tid; d < a.key_width; d += kThreads) {
          const float x = static_cast<float>(fresh_key[d]);
          low[d] = static_cast<T>(alone ? x : lower_of(x, static_cast<float>(low[d])));
          high[d] = static_cast<T>(alone ? x : higher_of(x, static_cast<float>(high[d])));
        }
      }
    }
  }

  const int tiles = last >> 5;  // number of the last one
  const int share = (tiles + splits) / splits;
  const int tile_end = void_rows ? 0 : min(tiles + 1, (split + 1) * share);
  const int first_limit = single ? last : past + row0 / a.share;

  // this wave's rows, as the columns of operands (the last one again beyond it)
  Operand<T> query[kSteps];
  const int my_row = row0 + min(column, rows - 1), my_token = my_row / a.share;
  const int limit = single ? last : past + my_token;
  const Rows<T> query_row = {
      a.query.row(batch, begin + my_token, kv_head * a.share + my_row - my_token * a.share), 0, 0};
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    Frag<T> part_of_row = memory_operand<WHOLE>(query_row, 0, s * 32 + 8 * group, a.key_width);
    clear_operand<WHOLE>(part_of_row, s * 32, group, a.key_width);
    query[s] = as_operand<T>(part_of_row);
  }
  f32x4 out[kCols];
#pragma unroll
  for (int d = 0; d < kCols; ++d) out[d] = f32x4(0.0f);
  float most = -__builtin_inff(), sum = 0.0f;
  const float factor = a.scale * kLog2e;

  Frag<T> key[2][kSteps];
  Piece held[kPieces];
  // A half of a tile lies on one page.  Halves behind the last key are its half again, rows behind it
  // its row: nothing that no token wrote is read.
  const auto half_begin = [&](int tile, int h) { return min(tile * kTile + h * 16, last & ~15); };
  const auto look_up = [&](int tile, int (&id)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      id[h] = __builtin_amdgcn_readfirstlane(table[half_begin(tile, h) >> a.page_shift]);
  };
  const auto fetch = [&](int tile, const int (&id)[2]) {
    int bad = 0;
    const T *keys[2], *values[2];
    int rows_left[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = half_begin(tile, h);
      const bool there = a.is_page(id[h]);
      bad |= there ? 0 : 1 << h;
      const int64_t row = a.place(there ? id[h] : 0, kv_head, at & ((1 << a.page_shift) - 1));
      keys[h] = a.key_pages + row * a.key_width;
      values[h] = a.value_pages + row * a.value_width;
      rows_left[h] = min(15, last - at);
    }
    if (tile * kTile + kTile <= fresh_from) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Rows<T> source = {keys[h], a.key_width, rows_left[h]};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          key[h][s] = memory_operand<WHOLE>(source, column, s * 32 + 8 * group, a.key_width);
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int h = i * kPieceRows / 16, row = i * kPieceRows - 16 * h + lane / kPerRow;
        const int col = lane % kPerRow * kElements;
        const Rows<T> source = {values[h], a.value_width, rows_left[h]};
        if constexpr (WHOLE) {
          held[i] = *reinterpret_cast<const Piece*>(
              place_of<WHOLE>(source, min(row, source.last), min(col, a.value_width - kElements)));
        } else {
          const T* from = place_of<WHOLE>(source, min(row, source.last), 0);
#pragma unroll
          for (int e = 0; e < kElements; ++e) held[i][e] = from[min(col + e, a.value_width - 1)];
        }
      }
      return bad;
    }
    // new tokens are taken from the inputs, whether they have a row or not
    const auto source_of = [&](const T* row_zero, int h, int row, int width, const T* fresh, int64_t stride) {
      const int token = half_begin(tile, h) + row - fresh_from;
      return token >= 0 ? fresh + token * stride : row_zero + row * width;
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Rows<T> source = {source_of(keys[h], h, min(column, rows_left[h]), a.key_width, fresh_key,
                                        a.key.token_stride), 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        key[h][s] = memory_operand<WHOLE>(source, 0, s * 32 + 8 * group, a.key_width);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int h = i * kPieceRows / 16;
      const int row = min(i * kPieceRows - 16 * h + lane / kPerRow, rows_left[h]);
      const int col = lane % kPerRow * kElements;
      const T* from = source_of(values[h], h, row, a.value_width, fresh_value, a.value.token_stride);
      if constexpr (WHOLE) {
        held[i] = *reinterpret_cast<const Piece*>(from + min(col, a.value_width - kElements));
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e) held[i][e] = from[min(col + e, a.value_width - 1)];
      }
    }
    return bad;
  };
  int tile = split * share + wave, bad = 0, id[2] = {0, 0};
  if (lane == 0) wild_from[wave] = 0x7fffffff;
  if (tile < tile_end) {
    look_up(tile, id);
    bad = fetch(tile, id);
    look_up(tile + 4, id);
  }
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
    const int missing = bad;
    if (missing != 0) {  // what is on no page makes NaN of the rows that see it, and nothing of others
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (missing >> (i * kPieceRows / 16) & 1) held[i] = Piece(static_cast<T>(0.0f));
    }
    const bool masked = tile * kTile + kTile - 1 > first_limit;
    if (masked && first_limit < last) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (clear_wild<T>(held[i])) atomicMin(&wild_from[wave], tile * kTile + i * kPieceRows + lane / kPerRow);
    }
    // (LDS accesses of one wave are carried out in order: its tile needs no barrier)
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int col = lane % kPerRow * kElements;
      float part_of_row[kElements];
#pragma unroll
      for (int e = 0; e < kElements; ++e) part_of_row[e] = static_cast<float>(held[i][e]);
      store_row<T, kTile, WIDTH>(tile_values, i * kPieceRows + lane / kPerRow, col, part_of_row);
    }
    asm volatile("" ::: "memory");
    if (tile + 4 < tile_end) {
      bad = fetch(tile + 4, id);
      look_up(tile + 8, id);
    }
    if (missing != 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (missing >> k & 1) score[k] = f32x4(__builtin_nanf(""));
    }
    if (masked) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (tile * kTile + k * 16 + 4 * group + r > min(limit, last)) score[k][r] = -__builtin_inff();
    }
    float here = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) here = fmaxf(here, score[k][r]);
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
      out[d] = mma(column_operand<T, kTile, WIDTH>(tile_values, 0, d * 16, lane), weights, out[d]);
    asm volatile("" ::: "memory");
  }

  // the waves of the block
  __syncthreads();
  float* outs = reinterpret_cast<float*>(shared) + wave * kRows * kOuts;
  sum = over_groups_sum(sum);
#pragma unroll
  for (int d = 0; d < kCols; ++d)
    *reinterpret_cast<f32x4*>(outs + column * kOuts + d * 16 + 4 * group) = out[d];
  if (group == 0) {
    // tokens behind the table have a key that is on no page
    const bool lost = void_rows || (!single && limit >= a.capacity()) || limit >= wild_from[wave];
    tops[wave][column] = most;
    totals[wave][column] = lost ? __builtin_nanf("") : sum;
  }
  __syncthreads();
  float* partial = a.division.partial + (static_cast<int64_t>(kv_head) * a.division.parts + part) * kRows * kOuts;
  for (int e = tid; e < rows * a.value_width; e += kThreads) {
    const int m = e / a.value_width, d = e % a.value_width;
    const float top = fmaxf(fmaxf(tops[0][m], tops[1][m]), fmaxf(tops[2][m], tops[3][m]));
    float total = 0.0f, value = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = top == -__builtin_inff() ? 1.0f : exp2_of(tops[w][m] - top);
      total += by * totals[w][m];
      value += by * (reinterpret_cast<float*>(shared) + w * kRows * kOuts)[m * kOuts + d];
    }
    if (splits == 1) {
      const int row = row0 + m, token = row / a.share;
      const int64_t at = (first + token) * a.heads + kv_head * a.share + row - token * a.share;
      a.out[at * a.value_width + d] = static_cast<T>(value / total);
    } else {
      float* to = partial + m * kOuts;
      to[d] = value;
      if (d == 0) {
        to[WIDTH] = top;
        to[WIDTH + 1] = total;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

// 64 QUERIES rows of a slot and head of keys, 16 QUERIES to a wave, over a portion of its keys in tiles
// of 64, which go through registers to LDS while the tile before is worked on; queries and sums stay in
// registers.  USED: the columns that keys and values have at most (tiles have WIDTH).  Weights are
// rounded to the inputs' type, as the operand of the product with the values, and summed as rounded.
//
// Four prompts of 2048 tokens behind up to 2500, 32 heads on 8 of 128 columns, bf16 (399 GFLOP): 445 us on
// a chip at work, 900 TFLOP/s (a product of 8192 x 8192 x 8192 by the library: 1400), 556 after it was idle
// (1130).  No pipe is full: matrix ones are busy for 39 % of the time, vector ones issue for 45 %, LDS works
// for 27 % (a wave reads all of both tiles, 32 KB, for its 32 rows); the registers hold two waves to a SIMD,
// and waves wait for 32 % of their time.  With operands read ahead of their products 476 us became 470.
// Tried and not kept: the next half tile's scores among the exponentials of this one, 588; eight waves for
// 256 rows in two teams, one with matrix instructions while the other has vector ones, 497 to 669, as all
// eight read as much of LDS again.
// Drafts of 5 tokens for 16 slots of up to 4096 (64 rows): 181 MB in 33 us, 5.7 TB/s.  Packed prompts of
// 1 to 2047 tokens behind up to 3001 (12 heads on 4 of 80 columns, fp16, 38 GFLOP): 120 us.  Portions
// of unequal length (of 512 places for blocks the one that ends last has 1.4 times the mean), columns padded
// from 80 to 96 and the prompts' distance from the library's rate make 70 of them; what the others are spent
// on is not known.  In float32 drafts
// take 136 us, prompts of 1024 tokens 112 TFLOP/s (176 with 64 columns); columns that are not whole pieces
// of 16 bytes are moved one by one: 100 and 33 of them, 16 prompts of 200 tokens, 62 TFLOP/s.
template <typename T, int WIDTH, int USED, int QUERIES, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWaves<T, WIDTH, WHOLE>))) void
paged_chunk_kernel(PagedArgs<T> a) {
  constexpr int kSteps = USED / 32, kRows = 64 * QUERIES, kCols = USED / 16;
  constexpr int kTile = kTileElements<T, kKeys, WIDTH>;
  using Move = TileMove<T, kKeys, WIDTH, WHOLE>;
  __shared__ __attribute__((aligned(16))) Stored<T> key_tiles[kBuffers<T> * kTile];
  __shared__ __attribute__((aligned(16))) Stored<T> value_tiles[kBuffers<T> * kTile];
  __shared__ int wild_from[4];  // position of a wave's first value that is not finite, where keys are masked

  const int tid = threadIdx.x, lane = tid & 63, group = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Portion p;
  const Found found = portion_of<kRows, kKeys, false>(a, tid, &p);
  if (found != Found::kRun) {
    if (found == Found::kInvalid) {
      const int64_t elements = static_cast<int64_t>(a.sequences.tokens) * a.heads * a.value_width;
      const int64_t blocks = static_cast<int64_t>(gridDim.x) * gridDim.y;
      for (int64_t e = static_cast<int64_t>(blockIdx.y * gridDim.x + blockIdx.x) * kThreads + tid;
           e < elements; e += blocks * kThreads)
        a.out[e] = static_cast<T>(__builtin_nanf(""));
    }
    return;
  }
  const int kv_head = p.kv_head, past = p.work.past, row0 = p.tile * kRows;
  const int rows = min(kRows, p.work.fresh * a.share - row0);
  const bool packed = a.sequences.offsets != nullptr;
  const int64_t batch = packed ? 0 : p.slot, begin_token = p.work.begin;
  const int64_t first_token = packed ? p.work.begin : static_cast<int64_t>(p.slot) * a.sequences.length;
  const int32_t* table = a.tables + static_cast<int64_t>(p.slot) * a.columns;
  const int64_t capacity = a.capacity();
  const int last = static_cast<int>(min(static_cast<int64_t>(past) + (row0 + rows - 1) / a.share, capacity - 1));
  if (p.splits > 1 && p.split == 0 && kv_head == 0 && tid == 0)
    a.division.tasks[p.task] = {first_token, row0, rows, p.part, p.splits};

  // this wave's rows, as the columns of operands (the last one again beyond it)
  const int wave_row = row0 + wave * 16 * QUERIES;
  const int wave_first = past + min(wave_row, row0 + rows - 1) / a.share;
  // no row of the wave sees a key from here on
  const int wave_end = wave_row < row0 + rows ? past + (min(wave_row + 16 * QUERIES, row0 + rows) - 1) / a.share + 1 : 0;
  Operand<T> query[QUERIES][kSteps];
  int limit[QUERIES];
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int row = min(wave_row + i * 16 + column, row0 + rows - 1), token = row / a.share;
    limit[i] = past + token;
    const Rows<T> query_row = {
        a.query.row(batch, begin_token + token, kv_head * a.share + row - token * a.share), 0, 0};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Frag<T> part = memory_operand<WHOLE>(query_row, 0, s * 32 + 8 * group, a.key_width);
      clear_operand<WHOLE>(part, s * 32, group, a.key_width);
      query[i][s] = as_operand<T>(part);
    }
  }
  f32x4 out[QUERIES][kCols];
  float most[QUERIES];
  f32x4 sum[QUERIES];  // (a product with ones: every row of the result is the sum)
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    most[i] = -__builtin_inff();
    sum[i] = f32x4(0.0f);
#pragma unroll
    for (int d = 0; d < kCols; ++d) out[i][d] = f32x4(0.0f);
  }
  const float factor = a.scale * kLog2e;

  // A quarter of a tile lies on one page, whose number a lane of the wave's first four holds.
  // Quarters and rows behind the last key are the last one's again.
  Move key_move, value_move;
  const Rows<T> fresh_keys = a.key.rows(batch, begin_token, kv_head, p.work.fresh);
  const Rows<T> fresh_values = a.value.rows(batch, begin_token, kv_head, p.work.fresh);
  const int page_mask = (1 << a.page_shift) - 1;
  const auto look_up = [&](int tile) {
    return table[min(tile * kKeys + 16 * (lane & 3), last & ~15) >> a.page_shift];
  };
  const auto missing_of = [&](int ids) {
    return static_cast<int>(__ballot(lane < 4 && !a.is_page(ids)));
  };
  const auto fetch = [&](Move& move, const T* pages, int width, const Rows<T>& fresh, int tile, int ids) {
    const int begin = tile * kKeys, left = min(kKeys - 1, last - begin);
    ids = a.is_page(ids) ? ids : 0;
    // new tokens are taken from the inputs, whether they have a row or not
    const bool fresh_only = begin >= past, one_page = begin + left < past && a.page_shift >= 6;
    if (fresh_only || one_page) {
      const Rows<T> held = {pages + a.place(__builtin_amdgcn_readlane(ids, 0), kv_head, begin & page_mask) * width,
                            width, left};
      move.fetch(fresh_only ? rows_from(fresh, begin - past, left + 1) : held, width, tid);
      return;
    }
    if (WHOLE && begin + kKeys <= past && left == kKeys - 1) {
      // (a base that the wave shares and an offset of 32 bits)
      const uint32_t col = min(Move::col_of(tid), width - Move::kElements);
#pragma unroll
      for (int i = 0; i < Move::kPieces; ++i) {
        const int quarter = (i * (kThreads / Move::kPerRow) + wave * (64 / Move::kPerRow)) >> 4;
        const int id = __builtin_amdgcn_readlane(ids, quarter);
        const T* base = pages + a.place(id, kv_head, (begin + 16 * quarter) & page_mask) * width;
        const uint32_t offset = ((Move::row_of(i, tid) & 15) * static_cast<uint32_t>(width) + col) *
                                static_cast<uint32_t>(sizeof(T));
        move.held[i] = *reinterpret_cast<const typename Move::Piece*>(reinterpret_cast<const char*>(base) + offset);
      }
      return;
    }
    move.fetch_from(
        [&](int row, int col) {
          row = min(row, left);
          const int quarter = __builtin_amdgcn_readfirstlane(row >> 4);
          const int id = __builtin_amdgcn_readlane(ids, quarter);
          const T* held = pages + (a.place(id, kv_head, (begin + 16 * quarter) & page_mask) + (row & 15)) * width;
          const int token = begin + row - past;
          return (token >= 0 ? fresh.base + token * fresh.stride : held) + col;
        },
        width, tid);
  };
  const auto fetch_keys = [&](int tile, int ids) {
    fetch(key_move, a.key_pages, a.key_width, fresh_keys, tile, ids);
  };
  const auto fetch_values = [&](int tile, int ids) {
    fetch(value_move, a.value_pages, a.value_width, fresh_values, tile, ids);
  };
  // what is on no page makes NaN of the rows that see it, and nothing of others
  const auto clear_missing = [&](int missing) {
    if (missing == 0) return;
#pragma unroll
    for (int i = 0; i < Move::kPieces; ++i)
      if (missing >> (Move::row_of(i, tid) >> 4) & 1)
        value_move.held[i] = typename Move::Piece(static_cast<T>(0.0f));
  };

  if (lane == 0) wild_from[wave] = 0x7fffffff;
  int wild = 0x7fffffff;
  const int first_limit = past + row0 / a.share;

  const int tiles = last / kKeys + 1, share = (tiles + p.splits - 1) / p.splits;
  const int tile_end = min(tiles, (p.split + 1) * share);
  int tile = p.split * share;
  int ids = 0, missing = 0;  // (looked up a tile before their pages are)
  if (tile < tile_end) {
    ids = look_up(tile);
    missing = missing_of(ids);
    fetch_keys(tile, ids);
    fetch_values(tile, ids);
    ids = look_up(tile + 1);
  }
  if (a.fused && p.split == 0)
    put_tokens<WHOLE>(a, fresh_keys.base, fresh_values.base, first_token, kv_head, row0, rows, tid);
  for (int side = 0; tile < tile_end; ++tile, side = kBuffers<T> - 1 - side) {
    const int begin = tile * kKeys, here_missing = missing;
    Stored<T>*keys = key_tiles + side * kTile, *values = value_tiles + side * kTile;
    clear_missing(missing);
    const bool diagonal = begin + kKeys - 1 > first_limit && first_limit < last;
    if (diagonal) {
#pragma unroll
      for (int i = 0; i < Move::kPieces; ++i)
        if (clear_wild<T>(value_move.held[i])) atomicMin(&wild_from[wave], begin + Move::row_of(i, tid));
    }
    key_move.store(keys, a.key_width, tid);
    value_move.store(values, a.value_width, tid);
    __syncthreads();
    if (diagonal)
      for (int w = 0; w < 4; ++w) wild = min(wild, wild_from[w]);
    if (tile + 1 < tile_end) {
      missing = missing_of(ids);
      fetch_keys(tile + 1, ids);
      fetch_values(tile + 1, ids);
      ids = look_up(tile + 2);
    }
    if (begin < wave_end) {
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
      if constexpr (sizeof(T) == 2) {
        // operands are read from LDS some products ahead of their own
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int j = 0; j < 4 * kSteps - 6; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, QUERIES, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6 * QUERIES, 0);
      }
      if (here_missing != 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (here_missing >> k & 1)
#pragma unroll
            for (int i = 0; i < QUERIES; ++i) score[i][k] = f32x4(__builtin_nanf(""));
      }
      if (begin + kKeys - 1 > min(wave_first, last)) {
#pragma unroll
        for (int i = 0; i < QUERIES; ++i) {
          const int upto = min(limit[i], last) - begin - 4 * group;
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              score[i][k][r] = k * 16 + r <= upto ? score[i][k][r] : -__builtin_inff();
        }
      }
      Operand<T> weights[QUERIES][2];
#pragma unroll
      for (int i = 0; i < QUERIES; ++i) {
        float here = score[i][0][0];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) here = fmaxf(here, score[i][k][r]);
        here = over_groups_max(here) * factor;
        // (every row by its own scores: what it does not see leaves its roundings as they are)
        const bool passed = here > most[i] + kSlack;
        if (__any(passed)) {
          const float larger = passed ? here : most[i];
          const float shrink = passed ? exp2_of(most[i] - larger) : 1.0f;
          sum[i] *= shrink;
#pragma unroll
          for (int d = 0; d < kCols; ++d) out[i][d] *= shrink;
          most[i] = larger;
        }
        const float base = (most[i] == -__builtin_inff() ? 0.0f : most[i]) - kLift<T>;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) score[i][k][r] = exp2_of(score[i][k][r] * factor - base);
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
      if constexpr (sizeof(T) == 2) {
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
        for (int j = 0; j < 2 * kCols - 4; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, QUERIES, 1);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6 * QUERIES, 1);
      }
    }
    if constexpr (kBuffers<T> == 1) __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int row = wave_row + i * 16 + column;
    if (row >= row0 + rows) continue;
    // tokens behind the table have a key that is on no page
    const float total = limit[i] >= capacity || limit[i] >= wild ? __builtin_nanf("") : sum[i][0];
    const int token = row / a.share;
    if (p.splits == 1) {
      const int64_t at = (first_token + token) * a.heads + kv_head * a.share + row - token * a.share;
      store_tiles<WHOLE, false>(a.out + at * a.value_width, out[i], 1.0f / total, group, a.value_width);
    } else {
      constexpr int kOuts = WIDTH + 4;
      float* to = a.division.partial +
                  ((static_cast<int64_t>(kv_head) * a.division.parts + p.part) * kRows + row - row0) * kOuts;
#pragma unroll
      for (int d = 0; d < kCols; ++d) *reinterpret_cast<f32x4*>(to + d * 16 + 4 * group) = out[i][d];
      if (group == 0) {
        to[WIDTH] = most[i];
        to[WIDTH + 1] = total;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// tiles that were cut
// ---------------------------------------------------------------------------

// What a thread has of parts first, first + STEP, ... of a row: its four columns, relative to the maximum.
struct PartSum {
  f32x4 value;
  float top, total;
};
// Four parts at once, so that their loads are under way together.  Columns from `used` on are left out.
template <int STEP>
__device__ __forceinline__ PartSum join_parts(const float* parts, int64_t apart, int first, int splits, int width,
                                              int col, int used) {
  constexpr int kAtOnce = 4;
  PartSum sum = {f32x4(0.0f), -__builtin_inff(), 0.0f};
  col = min(col, (used - 1) & ~3);
  for (; first < splits; first += kAtOnce * STEP) {
    float tops[kAtOnce], totals[kAtOnce];
    f32x4 values[kAtOnce];
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) {
      const float* part = parts + min(first + s * STEP, splits - 1) * apart;
      tops[s] = part[width];
      totals[s] = part[width + 1];
      values[s] = *reinterpret_cast<const f32x4*>(part + col);
    }
    float larger = sum.top;
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) larger = fmaxf(larger, tops[s]);
    const float base = larger == -__builtin_inff() ? 0.0f : larger, shrink = exp2_of(sum.top - base);
    sum.top = larger;
    sum.total *= shrink;
    sum.value *= shrink;
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s)
      if (first + s * STEP < splits) {
        const float by = exp2_of(tops[s] - base);
        sum.total += by * totals[s];
        sum.value += by * values[s];
      }
  }
  return sum;
}

// The parts of the first `unit_rows` rows of every tile.  Of few rows there may be many parts: a block
// has a row, and its threads four columns of some parts each.  Latency: 3.4 us for one slot, 5.1 us for 64
// slots with 2048 rows, 5.9 for 32 rows of 380 parts each (8.4 with the parts' maxima read before the rest).
template <typename T, int WIDTH>
__global__ __launch_bounds__(kThreads) void paged_join_few_kernel(PagedArgs<T> a, int tile_rows, int unit_rows) {
  constexpr int kOuts = WIDTH + 4, kLanes = WIDTH / 4, kTeams = kThreads / kLanes;
  __shared__ __attribute__((aligned(16))) float sums[kTeams][WIDTH];
  __shared__ float tops[kTeams], totals[kTeams];
  const int tid = threadIdx.x, col = tid % kLanes * 4, team = tid / kLanes;
  const int64_t units = static_cast<int64_t>(*a.division.task_count) * a.kv_heads * unit_rows;
  const int64_t apart = static_cast<int64_t>(tile_rows) * kOuts;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const PagedTask task = a.division.tasks[unit / unit_rows / a.kv_heads];
    const int kv_head = static_cast<int>(unit / unit_rows % a.kv_heads), r = static_cast<int>(unit % unit_rows);
    if (r >= task.rows) continue;
    const float* parts = a.division.partial +
                         ((static_cast<int64_t>(kv_head) * a.division.parts + task.part) * tile_rows + r) * kOuts;
    const PartSum sum = join_parts<kTeams>(parts, apart, team, task.splits, WIDTH, col, a.value_width);
    *reinterpret_cast<f32x4*>(&sums[team][col]) = sum.value;
    if (col == 0) {
      tops[team] = sum.top;
      totals[team] = sum.total;
    }
    __syncthreads();
    if (tid < a.value_width) {
      float top = tops[0], total = 0.0f, value = 0.0f;
      for (int t = 1; t < kTeams; ++t) top = fmaxf(top, tops[t]);
      const float base = top == -__builtin_inff() ? 0.0f : top;
      for (int t = 0; t < kTeams; ++t) {
        const float by = exp2_of(tops[t] - base);
        total += by * totals[t];
        value += by * sums[t][tid];
      }
      const int row = task.row + r, token = row / a.share;
      const int64_t at = (task.first + token) * a.heads + kv_head * a.share + row - token * a.share;
      a.out[at * a.value_width + tid] = static_cast<T>(value / total);
    }
    __syncthreads();
  }
}

// The same of many rows, which have few parts each: a thread has four columns of a row.  5 us for 16
// slots of 20 rows and 8 heads, 14 us for 51 MB of parts of packed prompts, which come from memory (4 TB/s).
template <typename T, int WIDTH>
__global__ __launch_bounds__(kThreads) void paged_join_many_kernel(PagedArgs<T> a, int tile_rows, int unit_rows) {
  constexpr int kOuts = WIDTH + 4, kLanes = WIDTH / 4, kTeams = kThreads / kLanes;
  const int col = threadIdx.x % kLanes * 4, team = threadIdx.x / kLanes;
  const int64_t units = static_cast<int64_t>(*a.division.task_count) * a.kv_heads * unit_rows;
  const int64_t apart = static_cast<int64_t>(tile_rows) * kOuts;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kTeams + team; unit < units;
       unit += static_cast<int64_t>(gridDim.x) * kTeams) {
    const int64_t tile = unit / unit_rows;
    const PagedTask task = a.division.tasks[tile / a.kv_heads];
    const int kv_head = static_cast<int>(tile % a.kv_heads), r = static_cast<int>(unit % unit_rows);
    if (r >= task.rows || col >= a.value_width) continue;
    const float* parts = a.division.partial +
                         ((static_cast<int64_t>(kv_head) * a.division.parts + task.part) * tile_rows + r) * kOuts;
    const PartSum sum = join_parts<1>(parts, apart, 0, task.splits, WIDTH, col, a.value_width);
    const int row = task.row + r, token = row / a.share;
    T* out = a.out + ((task.first + token) * a.heads + kv_head * a.share + row - token * a.share) * a.value_width;
    store4(out, col, sum.value * (1.0f / sum.total), a.value_width,
           a.value_width % 4 == 0 && reinterpret_cast<uintptr_t>(out) % sizeof(Quad<T>) == 0);
  }
}

// ---------------------------------------------------------------------------
// selected pages
// ---------------------------------------------------------------------------

// A single new token and the bounds of its page, which no token of the call has to know.
template <typename T>
__device__ __forceinline__ void put_single(const PagedArgs<T>& a, int64_t token, int slot, int kv_head, int past,
                                           int tid) {
  const int64_t row = a.row_of(token);
  if (row < 0) return;
  const int id = static_cast<int>(row >> a.page_shift), mask = (1 << a.page_shift) - 1;
  const int64_t to = a.place(id, kv_head, static_cast<int>(row & mask));
  const T* key = a.key.row(slot, 0, kv_head);
  const T* value = a.value.row(slot, 0, kv_head);
  T* low = a.key_bounds + (static_cast<int64_t>(id) * a.kv_heads + kv_head) * 2 * a.key_width;
  T* high = low + a.key_width;
  for (int d = tid; d < a.key_width; d += kThreads) {
    const float x = static_cast<float>(key[d]);
    const bool alone = (past & mask) == 0;
    a.key_pages[to * a.key_width + d] = key[d];
    low[d] = static_cast<T>(alone ? x : lower_of(x, static_cast<float>(low[d])));
    high[d] = static_cast<T>(alone ? x : higher_of(x, static_cast<float>(high[d])));
  }
  for (int d = tid; d < a.value_width; d += kThreads) a.value_pages[to * a.value_width + d] = value[d];
}

// x of the lane that a pattern within 16 lanes names
template <int PATTERN>
__device__ __forceinline__ double from_lane(double x) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), PATTERN, 0xf, 0xf, true);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), PATTERN, 0xf, 0xf, true);
  return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}
// The sum over groups of LANES lanes, 16 or 32 of them: within two, four, eight (mirrored, so that a
// lane meets one of the other four), sixteen, and the next sixteen.
template <int LANES>
__device__ __forceinline__ double over_lanes_sum(double x) {
  x += from_lane<0xb1>(x);
  x += from_lane<0x4e>(x);
  x += from_lane<0x141>(x);
  x += from_lane<0x140>(x);
  if constexpr (LANES == 32) x += __shfl_xor(x, 16);
  return x;
}

// Whether 16 bytes of numbers have infinity among them, or NaN: as whole numbers with a sign, of which
// the largest is taken, they lie above all that is finite, and what is below zero below it.
template <typename T, typename Piece>
__device__ __forceinline__ bool reaches_infinity(const Piece& piece) {
  if constexpr (sizeof(T) == 4) {
    typedef int Words __attribute__((ext_vector_type(4)));
    const Words words = __builtin_bit_cast(Words, piece);
    return max(max(words[0], words[1]), max(words[2], words[3])) >= 0x7f800000;
  } else {
    typedef short Pair __attribute__((ext_vector_type(2)));
    struct Pairs {
      Pair of[4];
    };
    const Pairs pairs = __builtin_bit_cast(Pairs, piece);
    const Pair most = __builtin_elementwise_max(__builtin_elementwise_max(pairs.of[0], pairs.of[1]),
                                                __builtin_elementwise_max(pairs.of[2], pairs.of[3]));
    return max(most[0], most[1]) >= (std::is_same_v<T, _Float16> ? 0x7c00 : 0x7f80);
  }
}

// The largest product that a key within a page's bounds can have with a query of the group, in 64 bits,
// in which the products are exact: pages are ranked as their bounds rank, to the rounding of a sum of 64 bits
// (2^-53 of its largest part sum for each of up to 127 additions), whose order is the same in every run.
// A lane has the queries' elements of its columns in registers for all pages; the lanes of a page add up.
// Vector instructions in 64 bits bound it, and the latency of a page's number and bounds, which four pages
// at once hide: 32 slots of up to 256 pages, 32 heads on 8 of 128 columns, bf16, 15.7 us (one page at
// once 19; a page to a lane with queries in LDS 13.5 to 19, and far slower for few pages; a lane for some
// columns of all heads 26; three waves to a SIMD 17.5); 173 packed tokens of up to 188 pages 18.3 us.
// ONE: the group has at most four members, whose queries are loaded once.  More are loaded again for
// every turn of pages, whose bounds and best scores stay in registers: two slots of 3125 pages, 16 heads
// on 2, 9.7 us (11.8 with best scores in memory from one four to the next).
template <typename T, bool WHOLE, bool ONE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(ONE && WHOLE ? 4 : 2))) void
paged_score_kernel(PagedArgs<T> a, int blocks_of_token) {
  constexpr int kElements = 16 / static_cast<int>(sizeof(T)), kMembers = 4;
  constexpr int kLanes = kMostWidth / kElements, kPages = kThreads / kLanes, kTurns = 4;  // of a page; at once
  typedef T Piece __attribute__((ext_vector_type(kElements)));
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t block = block_number();
  const int64_t at = block / blocks_of_token;
  const int64_t number = at / a.kv_heads;
  const int kv_head = static_cast<int>(at % a.kv_heads);
  if (number >= a.slab_tokens) return;
  const int token = static_cast<int>(a.slab_first + number);
  const int slot = slot_of_token(a, token, lane);
  const int position = position_of(a, token, slot);
  const int earlier = min(position >> a.page_shift, a.columns);
  const bool puts = a.fused && block % blocks_of_token == 0;
  if (earlier <= a.count) {  // all of them are selected
    if (puts) put_single(a, token, slot, kv_head, position, tid);
    return;
  }
  const bool packed = a.sequences.offsets != nullptr;
  const int32_t* table = a.tables + static_cast<int64_t>(slot) * a.columns;
  double* scores = a.scores + at * a.columns;
  const int col = tid % kLanes * kElements;
  // (lanes behind the last column have queries of zero, some other bounds, and sums that are left out)
  const int from = min(col, WHOLE ? a.key_width - kElements : a.key_width - 1);
  double queries[kMembers][kElements];
  const auto fetch_queries = [&](int member0) {
    const int members = min(kMembers, a.share - member0);
#pragma unroll
    for (int m = 0; m < kMembers; ++m) {
      const int head = kv_head * a.share + member0 + min(m, members - 1);
      const T* query = packed ? a.query.row(0, token, head)
                              : a.query.row(slot, token - slot * a.sequences.length, head);
      Piece part;
      if constexpr (WHOLE) {
        part = *reinterpret_cast<const Piece*>(query + from);
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e) part[e] = query[min(col + e, a.key_width - 1)];
      }
#pragma unroll
      for (int e = 0; e < kElements; ++e)
        queries[m][e] = col + e < a.key_width ? static_cast<double>(static_cast<float>(part[e])) : 0.0;
    }
  };
  const int step = blocks_of_token * kPages * kTurns;
  const int start = static_cast<int>(block % blocks_of_token) * kPages * kTurns;
  fetch_queries(0);
  for (int base = start; base < earlier; base += step) {
    int id[kTurns];
    Piece lows[kTurns], highs[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) id[i] = table[min(base + i * kPages + tid / kLanes, earlier - 1)];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const T* low = a.key_bounds +
                     (static_cast<int64_t>(a.is_page(id[i]) ? id[i] : 0) * a.kv_heads + kv_head) * 2 * a.key_width;
      const T* high = low + a.key_width;
      if constexpr (WHOLE) {
        lows[i] = *reinterpret_cast<const Piece*>(low + from);
        highs[i] = *reinterpret_cast<const Piece*>(high + from);
      } else {
#pragma unroll
        for (int e = 0; e < kElements; ++e) {
          const bool there = from + e < a.key_width;
          lows[i][e] = there ? low[from + e] : static_cast<T>(0.0f);
          highs[i][e] = there ? high[from + e] : static_cast<T>(0.0f);
        }
      }
    }
    double best[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) best[i] = -__builtin_inf();
    uint32_t no_number = 0;  // turns in which a sum is none after all
    for (int member0 = 0; member0 < (ONE ? 1 : a.share); member0 += kMembers) {
      if (!ONE && (base > start || member0 > 0)) fetch_queries(member0);
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        if (base + i * kPages >= earlier) break;
        double sum[kMembers] = {};
#pragma unroll
        for (int e = 0; e < kElements; ++e) {
          const double least = static_cast<float>(lows[i][e]), largest = static_cast<float>(highs[i][e]);
#pragma unroll
          for (int m = 0; m < kMembers; ++m)
            sum[m] = fma(queries[m][e], queries[m][e] > 0.0 ? largest : least, sum[m]);
        }
#pragma unroll
        for (int m = 0; m < kMembers; ++m)  // (zero times infinity is no number)
          sum[m] = over_lanes_sum<kLanes>(col < a.key_width ? sum[m] : 0.0);
#pragma unroll
        for (int m = 0; m < kMembers; ++m) best[i] = sum[m] > best[i] || sum[m] != sum[m] ? sum[m] : best[i];
        const int page = base + i * kPages + tid / kLanes;
        if ((ONE || member0 + kMembers >= a.share) && tid % kLanes == 0 && page < earlier)
          scores[page] = a.is_page(id[i]) ? best[i] : __builtin_nan("");
      }
      // A query of zero took the lower bound, and is no number times the upper one either if that is
      // infinite.  (Apart from the sums, and looked at last, so that nothing waits for it.)
      bool infinite = false;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) infinite |= reaches_infinity<T>(highs[i]);
      if (__any(infinite))
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          // (converted in this branch: else all of them are held in registers for it)
          typedef uint32_t Words __attribute__((ext_vector_type(4)));
          Words words = __builtin_bit_cast(Words, highs[i]);
          asm volatile("" : "+v"(words));
          const Piece upper = __builtin_bit_cast(Piece, words);
#pragma unroll
          for (int e = 0; e < kElements; ++e) {
            const double largest = static_cast<float>(upper[e]);
#pragma unroll
            for (int m = 0; m < kMembers; ++m) {
              const double other = queries[m][e] * largest;
              if (other != other) no_number |= 1u << i;
            }
          }
        }
    }
    if (__any(no_number != 0)) {
      const uint64_t lanes = ((uint64_t{1} << kLanes) - 1) << (lane & -kLanes);
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const uint64_t those = __ballot(col < a.key_width && (no_number >> i & 1) != 0);
        const int page = base + i * kPages + tid / kLanes;
        if ((those & lanes) != 0 && tid % kLanes == 0 && page < earlier) scores[page] = __builtin_nan("");
      }
    }
  }
  if (puts) put_single(a, token, slot, kv_head, position, tid);
}

// A score as a whole number that ranks alike; what is no number ranks first.
__device__ __forceinline__ uint64_t rank_of(double score) {
  if (score != score) return ~uint64_t{0};
  const uint64_t bits = __builtin_bit_cast(uint64_t, score + 0.0);  // (no zero below zero)
  return bits >> 63 ? ~bits : bits | uint64_t{1} << 63;
}

// The pages of a token and head of keys: the `count` with the largest scores, in the order of the
// slot's table, and its own; and how many positions it sees on them.  A block finds the score of the
// last one that is selected eight bits at a time, by counting, from the first bit on in which scores
// differ (before it all of them would count in one place), and keeps four scores a thread in registers.
// Barriers bound it: 256 lists of up to 256 pages 6 us; 4 lists of 3125 pages, by 1024 threads, 11.7 us
// (13.2 where every pass read the scores).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_select_kernel(PagedArgs<T> a) {
  constexpr int kAll = THREADS / 64;
  __shared__ int counts[256], ends[kAll], equal_ends[kAll], chosen[2];
  __shared__ uint64_t lowest[kAll], highest[kAll];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t at = block_number(), number = at / a.kv_heads;
  if (number >= a.slab_tokens) return;
  const int token = static_cast<int>(a.slab_first + number);
  const int64_t to = static_cast<int64_t>(token) * a.kv_heads + at % a.kv_heads;
  int32_t* list = a.lists + to * (a.count + 1);
  if (!offsets_valid<THREADS>(a, tid)) {
    if (tid == 0) a.seen[to] = 0;
    return;
  }
  const int slot = slot_of_token(a, token, lane), position = position_of(a, token, slot);
  const int32_t* table = a.tables + static_cast<int64_t>(slot) * a.columns;
  const int own = position >> a.page_shift, earlier = min(own, a.columns);
  const int selected = min(earlier, a.count);
  if (tid == 0) {
    list[selected] = own < a.columns ? table[own] : -1;
    a.seen[to] = (selected << a.page_shift) + (position & ((1 << a.page_shift) - 1)) + 1;
  }
  if (earlier <= a.count) {
    for (int j = tid; j < earlier; j += THREADS) list[j] = table[j];
    return;
  }
  const double* scores = a.scores + at * a.columns;
  // the pages in turns of a block's threads, for all threads; a few turns stay in registers
  constexpr int kHeld = 4;
  uint64_t held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = rank_of(scores[min(i * THREADS + tid, earlier - 1)]);
  const auto for_each = [&](auto&& visit) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i * THREADS < earlier) visit(i * THREADS + tid, held[i]);
    for (int base = kHeld * THREADS; base < earlier; base += THREADS)
      visit(base + tid, rank_of(scores[min(base + tid, earlier - 1)]));
  };
  uint64_t low = ~uint64_t{0}, high = 0;
  for_each([&](int j, uint64_t rank) {
    if (j < earlier) {
      low = min(low, rank);
      high = max(high, rank);
    }
  });
  for (int away = 1; away < 64; away *= 2) {
    low = min(low, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(low), away)));
    high = max(high, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(high), away)));
  }
  if (lane == 0) {
    lowest[wave] = low;
    highest[wave] = high;
  }
  __syncthreads();
  for (int w = 0; w < kAll; ++w) {
    low = min(low, lowest[w]);
    high = max(high, highest[w]);
  }
  // those above `prefix` in the bits of `mask` are selected, and the first `need` of those equal to it
  int bits = low == high ? 0 : 64 - __clzll(low ^ high);  // that are not yet known
  uint64_t mask = bits == 64 ? 0 : ~uint64_t{0} << bits, prefix = low & mask;
  int need = a.count;
  while (bits > 0) {
    const int shift = max(bits - 8, 0), digits = (1 << (bits - shift)) - 1;
    if (tid < 256) counts[tid] = 0;
    __syncthreads();
    for_each([&](int j, uint64_t rank) {
      if (j < earlier && (rank & mask) == prefix) atomicAdd(&counts[rank >> shift & digits], 1);
    });
    __syncthreads();
    const int mine = tid < 256 ? counts[255 - tid] : 0, upto = scan_wave(mine);
    if (lane == 63) ends[wave] = upto;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < wave; ++w) before += ends[w];
    if (before < need && need <= before + mine) {
      chosen[0] = 255 - tid;
      chosen[1] = before;
    }
    __syncthreads();
    const int digit = chosen[0];
    need -= chosen[1];
    prefix |= static_cast<uint64_t>(digit) << shift;
    mask = ~uint64_t{0} << shift;
    bits = shift;
    const bool all = counts[digit] == need;
    __syncthreads();
    if (all) break;
  }
  int above = 0, equal = 0;  // of the pages so far
  for_each([&](int j, uint64_t rank) {
    rank &= mask;
    const bool more = j < earlier && rank > prefix, same = j < earlier && rank == prefix;
    const uint64_t more_mask = __ballot(more), same_mask = __ballot(same);
    if (lane == 0) {
      ends[wave] = __popcll(more_mask);
      equal_ends[wave] = __popcll(same_mask);
    }
    __syncthreads();
    const uint64_t below = (uint64_t{1} << lane) - 1;
    int above_me = above + __popcll(more_mask & below), equal_me = equal + __popcll(same_mask & below);
    for (int w = 0; w < kAll; ++w) {
      if (w < wave) {
        above_me += ends[w];
        equal_me += equal_ends[w];
      }
      above += ends[w];
      equal += equal_ends[w];
    }
    if (more || (same && equal_me < need)) list[above_me + min(equal_me, need)] = table[j];
    __syncthreads();
  });
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T>
PagedArgs<T> paged_args(const PagedCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  const rosa_paged_cache& c = *call.cache;
  PagedArgs<T> args{};
  args.query = view_of<T>(*call.query);
  args.key = view_of<T>(*call.key);
  args.value = view_of<T>(*call.value);
  args.out = static_cast<T*>(call.out);
  args.key_pages = static_cast<T*>(c.key_pages);
  args.value_pages = static_cast<T*>(c.value_pages);
  args.key_bounds = static_cast<T*>(c.key_bounds);
  args.tables = c.tables;
  args.lengths = c.lengths;
  args.rows = c.rows;
  args.sequences = sequences_of(p);
  args.pages = c.pages;
  args.columns = c.columns;
  args.page_shift = __builtin_ctz(static_cast<unsigned>(c.page));
  args.heads = p.H;
  args.kv_heads = p.Hkv;
  args.share = p.H / p.Hkv;
  args.key_width = p.D;
  args.value_width = p.Dv;
  args.scale = p.scale;
  args.count = call.count;
  return args;
}

template <typename T>
PagedDivision division_of(const PagedShare& share, int most_few, char* at) {
  PagedDivision d{};
  d.target = share.target;
  d.least = share.least;
  d.most_few = most_few;
  d.round = share.round;
  d.parts = share.parts;
  if (share.parts > 0) {
    d.partial = reinterpret_cast<float*>(at);
    d.task_count = reinterpret_cast<int*>(at + share.part_bytes);
    d.tasks = reinterpret_cast<PagedTask*>(at + share.part_bytes + 256);
  }
  return d;
}

// Blocks that go on to further work: a thousand more take the chip 4 us to begin, whatever they do.  Those
// of a join are as many as it can hold at once (51 MB of parts: 1024 of them 17 us, 2048 14, 4096 14).
constexpr int64_t kJoinBlocks = 2048;
// And those that put tokens on their rows: each looks at all offsets once.
constexpr int64_t kAppendBlocks = 2048;
constexpr int64_t kScoreBlocks = 1024;

template <typename T, int WIDTH, bool WHOLE>
void paged_token_launch(PagedArgs<T>& args, const PagedShare& share, hipStream_t stream) {
  const dim3 grid = grid_of(share.items * args.kv_heads);
  paged_token_kernel<T, WIDTH, WHOLE><<<grid, kThreads, 0, stream>>>(args);
  if (share.parts == 0) return;
  const int64_t units = share.cut() * args.kv_heads * share.unit_rows;
  paged_join_few_kernel<T, WIDTH>
      <<<dim3(static_cast<unsigned>(std::min<int64_t>(units, kJoinBlocks))), kThreads, 0, stream>>>(
          args, share.rows, share.unit_rows);
}

template <typename T, int WIDTH, int USED, bool WHOLE>
void paged_chunk_rows(PagedArgs<T>& args, const PagedShare& share, hipStream_t stream) {
  const dim3 grid = grid_of_items(share.items * args.kv_heads);
  if constexpr (kPairs<T, WIDTH>) {
    if (share.rows == 128) paged_chunk_kernel<T, WIDTH, USED, 2, WHOLE><<<grid, kThreads, 0, stream>>>(args);
  }
  if (share.rows == 64) paged_chunk_kernel<T, WIDTH, USED, 1, WHOLE><<<grid, kThreads, 0, stream>>>(args);
}

template <typename T, int WIDTH, bool WHOLE>
void paged_chunk_launch(PagedArgs<T>& args, const PagedShare& share, hipStream_t stream) {
  // (columns that no head has are left out where that is a quarter of them)
  if constexpr (WIDTH == 128) {
    if (args.key_width <= 96 && args.value_width <= 96)
      paged_chunk_rows<T, WIDTH, 96, WHOLE>(args, share, stream);
    else
      paged_chunk_rows<T, WIDTH, WIDTH, WHOLE>(args, share, stream);
  } else {
    paged_chunk_rows<T, WIDTH, WIDTH, WHOLE>(args, share, stream);
  }
  if (share.parts == 0) return;
  const int64_t blocks = (share.cut() * args.kv_heads * share.unit_rows * (WIDTH / 4) - 1) / kThreads + 1;
  paged_join_many_kernel<T, WIDTH>
      <<<dim3(static_cast<unsigned>(std::min<int64_t>(blocks, kJoinBlocks))), kThreads, 0, stream>>>(
          args, share.rows, share.unit_rows);
}

template <typename T, bool WHOLE>
void paged_append_launch(PagedArgs<T>& args, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(pages_touched(args)) * args.kv_heads;
  paged_append_kernel<T, WHOLE>
      <<<dim3(static_cast<unsigned>(std::min<int64_t>(items, kAppendBlocks))), kThreads, 0, stream>>>(args);
}

// Scores of a slab of tokens take at most this much memory, or one token's.
template <typename T, bool WHOLE>
void paged_select_launch(PagedArgs<T>& args, const PagedPlan& plan, hipStream_t stream) {
  const int64_t row = static_cast<int64_t>(args.kv_heads) * args.columns * 8;
  const int64_t slab = static_cast<int64_t>(plan.score_bytes) / row;
  for (int64_t first = 0; first < args.sequences.tokens; first += slab) {
    args.slab_first = first;
    args.slab_tokens = std::min<int64_t>(slab, args.sequences.tokens - first);
    const int64_t pairs = args.slab_tokens * args.kv_heads;
    if (args.columns > args.count) {
      const int64_t at_once = 4 * kThreads / (kMostWidth * sizeof(T) / 16);
      const int64_t most = (args.columns + at_once - 1) / at_once;
      const int blocks = static_cast<int>(std::max<int64_t>(1, std::min(most, kScoreBlocks / pairs)));
      if (args.share <= 4)
        paged_score_kernel<T, WHOLE, true><<<grid_of(pairs * blocks), kThreads, 0, stream>>>(args, blocks);
      else
        paged_score_kernel<T, WHOLE, false><<<grid_of(pairs * blocks), kThreads, 0, stream>>>(args, blocks);
    }
    // (few long lists: all the threads that a block can have)
    if (pairs <= 256 && args.columns > 1024)
      paged_select_kernel<T, 1024><<<grid_of(pairs), 1024, 0, stream>>>(args);
    else
      paged_select_kernel<T, kThreads><<<grid_of(pairs), kThreads, 0, stream>>>(args);
  }
}

template <typename T, int WIDTH, bool WHOLE>
void paged_update_launch(const PagedCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  const PagedPlan plan = paged_plan(p, *call.cache, call.count);
  PagedArgs<T> args = paged_args<T>(call);
  char* at = call.workspace;
  const PagedDivision few = division_of<T>(plan.few, plan.most_few, at);
  at += plan.few.bytes();
  const PagedDivision many = division_of<T>(plan.many, plan.most_few, at);
  at += plan.many.bytes();
  if (call.count > 0) {
    // (single tokens are put on their rows by the kernel of the scores, where it runs)
    args.fused = p.cu_seqlens == nullptr && p.T == 1 && args.columns > args.count;
    if (!args.fused) paged_append_launch<T, WHOLE>(args, call.stream);
    args.lists = reinterpret_cast<int32_t*>(at);
    args.seen = reinterpret_cast<int32_t*>(at + plan.list_bytes);
    args.scores = reinterpret_cast<double*>(at + plan.list_bytes + plan.seen_bytes);
    paged_select_launch<T, WHOLE>(args, plan, call.stream);
    args.fused = false;
    args.division = few;
    args.list_splits = plan.few.target;
    return paged_token_launch<T, WIDTH, WHOLE>(args, plan.few, call.stream);
  }
  // (bounds of a page that several tokens are put on have a kernel of their own)
  args.fused = args.key_bounds == nullptr || (p.cu_seqlens == nullptr && p.T == 1 && !plan.many.used);
  if (!args.fused) paged_append_launch<T, WHOLE>(args, call.stream);
  if (plan.few.used) {
    args.division = few;
    paged_token_launch<T, WIDTH, WHOLE>(args, plan.few, call.stream);
  }
  if (plan.many.used) {
    args.division = many;
    paged_chunk_launch<T, WIDTH, WHOLE>(args, plan.many, call.stream);
  }
}

template <typename T, bool WHOLE>
void paged_update_width(const PagedCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  switch (padded_width(p.D > p.Dv ? p.D : p.Dv)) {
    case 32: return paged_update_launch<T, 32, WHOLE>(call);
    case 64: return paged_update_launch<T, 64, WHOLE>(call);
    default: return paged_update_launch<T, 128, WHOLE>(call);
  }
}

template <typename T>
void paged_update(const PagedCall& call) {
  const rosa_mixer_problem& p = *call.problem;
  const rosa_paged_cache& c = *call.cache;
  const bool whole = whole_pieces<T>(*call.query, p.D) && whole_pieces<T>(*call.key, p.D) &&
                     whole_pieces<T>(*call.value, p.Dv) && whole_address(call.out) &&
                     whole_address(c.key_pages) && whole_address(c.value_pages) &&
                     whole_address(c.key_bounds);
  if (whole)
    paged_update_width<T, true>(call);
  else
    paged_update_width<T, false>(call);
}

}  // namespace rosa_mixer
