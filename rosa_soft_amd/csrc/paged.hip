// C entry points of the paged cache: checks, work division and workspace in host arithmetic, and the
// kernels that hand pages out and take them back.  The attention is in paged_attention.hpp, one
// translation unit per element type.
#include "paged_calls.hpp"
#include "mixer_device.hpp"

#include <algorithm>
#include <cmath>

namespace rosa_mixer {

namespace {

constexpr int64_t kBlocks = 512;                        // two for a compute unit
constexpr int kFewRows = 16;                            // of a slot, that paged_token_kernel takes
constexpr int64_t kMostScoreBytes = int64_t{1} << 28;   // of a slab of tokens
constexpr int kTableThreads = 1024;
// Tokens whose rows the block that hands out pages writes by itself; more have a launch of their own.
constexpr int kTokensOfBlock = 16384;
// Pages that a block can mark at a time, a bit of LDS each (64 KB): a larger pool is looked at in parts.
constexpr int kMarkedPages = 1 << 19;
constexpr int kRun = 512;  // columns of a slot that a wave looks through at a time

}  // namespace

// Portions of a call, beside one for each tile of rows, and from which part of a portion on a walk has
// one more.  More share ragged slots out more evenly, and make more partial sums.  Few rows (reads bound
// them; 64 slots of up to 9000 tokens, 8 heads of 128): 512 portions 296 us, 768 279, 1024 281, 2048 278;
// two slots of up to 200000, 2 heads of 64: 43, 44, 46 and 50 us.  Many rows, dense (512 tokens behind
// 60000, 32 heads on 8; 64 behind up to 8000 for each of 8 slots; one prompt of 2048): 512 portions, one
// more from 3/8 on: 641, 76 and 69 us, from 7/8 on: 641, 98 and 68; 768: 694, 88 and 80.  Packed (a step of
// 1 to 2047 tokens for 10 slots; 15 single ones and 1024): 139 and 281 us, 141 and 296, 116 and 247.
constexpr int kFewPortions = 768, kManyPortions = 512, kPackedPortions = 768;

PagedPlan paged_plan(const rosa_mixer_problem& p, const rosa_paged_cache& cache, int count) {
  PagedPlan plan{};
  plan.width = padded_width(std::max(p.D, p.Dv));
  const int share = p.H / p.Hkv;
  const bool packed = p.cu_seqlens != nullptr;
  const int64_t sequences = packed ? p.S : p.B;
  const int64_t capacity = static_cast<int64_t>(cache.columns) * cache.page;
  const int outs = plan.width + 4;
  const auto finish = [&](PagedShare* s) {
    if (s->parts > 0) {
      s->part_bytes = aligned(static_cast<size_t>(s->parts) * p.Hkv * s->rows * outs * 4);
      s->task_bytes = 256 + aligned(static_cast<size_t>(s->parts) * 32);
    }
  };
  PagedShare& few = plan.few;
  few.rows = kFewRows;
  if (count > 0) {
    // Tokens on their own, which see about as many keys each: until there are two blocks for a compute
    // unit or a wave has but two tiles.
    few.used = true;
    const int64_t tiles = static_cast<int64_t>(p.N) * ((share + few.rows - 1) / few.rows);
    const int64_t walk = (std::min<int64_t>(count + 1, cache.columns) * cache.page + 31) / 32;
    const int64_t blocks = tiles * p.Hkv;
    few.target = static_cast<int>(
        std::max<int64_t>(1, std::min((kBlocks + blocks - 1) / blocks, walk / 8)));
    few.tiles = tiles;
    few.items = tiles * few.target;
    few.parts = few.target > 1 ? few.items : 0;
    few.unit_rows = std::min(few.rows, share);
    finish(&few);
    plan.list_bytes = aligned(static_cast<size_t>(p.N) * p.Hkv * (count + 1) * 4);
    plan.seen_bytes = aligned(static_cast<size_t>(p.N) * p.Hkv * 4);
    const int64_t row = static_cast<int64_t>(p.Hkv) * cache.columns * 8;
    plan.score_bytes = static_cast<size_t>(
        row * std::min<int64_t>(p.N, std::max<int64_t>(1, kMostScoreBytes / row)));
    return plan;
  }
  // A packed call's single tokens have the kernel for few rows beside the other one, unless prompts are
  // most of the work: 63 single tokens behind up to 8000, 32 heads on 8, with 5 more tokens of another
  // slot: 279 us with both, 305 with one; 15 with 1024 more: 269 and 280; 5 rows of single tokens and
  // 1200 tokens of prompts: 126 and 116.  Of 20 rows (5 tokens, 4 heads on one) the other kernel is
  // faster as well, 51 us and 62 in two sixteens for 16 slots of up to 4096 tokens.
  const int64_t rows = packed ? share : static_cast<int64_t>(p.T) * share;  // of a slot, at least
  few.used = rows <= kFewRows && !(packed && static_cast<int64_t>(p.N) * share >= 64 * sequences);
  plan.most_few = few.used ? kFewRows : 0;
  if (few.used) {
    few.target = (kFewPortions + p.Hkv - 1) / p.Hkv;
    few.least = 4;
    few.round = 7;
    few.unit_rows = packed ? few.rows : static_cast<int>(rows);
    few.tiles = sequences;
    few.items = sequences + few.target;
    few.parts = (capacity + 31) / 32 > few.least ? 2 * few.target : 0;
    finish(&few);
  }
  PagedShare& many = plan.many;
  many.used = packed || !few.used;
  if (many.used) {
    // 128 rows, so that an operand read from LDS serves two products, where a slot may have as many and
    // they fit the registers (float32, 128 columns: they do not).
    const bool pairs = p.dtype != ROSA_DTYPE_F32 || plan.width < 128;
    many.rows = pairs && (packed || rows > 64) ? 128 : 64;
    const int64_t tiles = packed ? static_cast<int64_t>(p.N) * share / many.rows + sequences
                                 : sequences * ((rows + many.rows - 1) / many.rows);
    many.target = ((packed ? kPackedPortions : kManyPortions) + p.Hkv - 1) / p.Hkv;
    many.least = 4;
    many.round = packed ? 7 : 3;
    many.unit_rows = packed ? many.rows : static_cast<int>(std::min<int64_t>(many.rows, rows));
    many.tiles = tiles;
    many.items = tiles + many.target;
    many.parts = (capacity + 63) / 64 > many.least ? 2 * many.target : 0;
    finish(&many);
  }
  return plan;
}

// ---------------------------------------------------------------------------
// tables
// ---------------------------------------------------------------------------

namespace {

struct TableArgs {
  int32_t *tables, *pool;
  const int32_t *lengths, *keep, *offsets;
  int64_t* rows;
  int slots, columns, pages, page_shift, T, N;
  __device__ __forceinline__ int64_t held(int64_t tokens) const {  // columns of that many tokens
    return min((tokens + (1 << page_shift) - 1) >> page_shift, static_cast<int64_t>(columns));
  }
  __device__ __forceinline__ int64_t length(int s) const { return max(lengths[s], 0); }
  __device__ __forceinline__ int64_t kept(int s) const {  // columns that a release leaves to a slot
    return held(min(static_cast<int64_t>(max(keep[s], 0)), length(s)));
  }
  __device__ __forceinline__ int64_t row_at(int s, int64_t position) const {
    const int64_t column = position >> page_shift;
    const int id = column < columns ? tables[static_cast<int64_t>(s) * columns + column] : -1;
    return id >= 0 && id < pages ? (static_cast<int64_t>(id) << page_shift) + (position & ((1 << page_shift) - 1))
                                 : -1;
  }
};

// Inclusive sum over the threads of a block, and its total.
__device__ __forceinline__ int64_t scan_block(int64_t x, int tid, int64_t* ends, int64_t* total) {
  const int lane = tid & 63, wave = tid >> 6;
  for (int apart = 1; apart < 64; apart *= 2) {
    const int64_t before = __shfl_up(static_cast<long long>(x), apart);
    if (lane >= apart) x += before;
  }
  if (lane == 63) ends[wave] = x;
  __syncthreads();
  int64_t all = 0;
  for (int w = 0; w < kTableThreads / 64; ++w) {
    if (w < wave) x += ends[w];
    all += ends[w];
  }
  __syncthreads();
  *total = all;
  return x;
}

// The last slot whose first item is `item` or one before it: the one that has it.
__device__ __forceinline__ int slot_of_item(const int* first, int slots, int item) {
  int low = 0, high = slots;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    (first[middle] <= item ? low : high) = middle;
  }
  return low;
}

__device__ __forceinline__ int64_t row_of_token(const TableArgs& a, const int32_t* offsets, int token) {
  if (offsets == nullptr) {
    const int s = token / a.T;
    return a.row_at(s, a.length(s) + token - s * a.T);
  }
  const int s = slot_of_item(offsets, a.slots, token);
  return a.row_at(s, a.length(s) + token - offsets[s]);
}

// One block, since every page that is handed out depends on those before it: the items of a call (new
// pages of slots, in order) are numbered by a sum over the slots, and every thread takes some of them.
// Latency is all of it: 3.8 us for 64 slots with 8 tokens each; a call that releases and one that hands
// out, with the rows, 16 us in all.
__global__ __launch_bounds__(kTableThreads) void page_tables_update_kernel(TableArgs a, bool all_rows) {
  extern __shared__ int first[];  // [slots] items, [slots + 1] tokens
  __shared__ int64_t ends[kTableThreads / 64];
  const int tid = threadIdx.x;
  int* offsets = first + a.slots;
  const int free = max(0, min(a.pool[0], a.pages));
  int bad = 0;
  if (a.offsets != nullptr) {
    for (int s = tid; s < a.slots; s += kTableThreads) {
      const int begin = a.offsets[s], end = a.offsets[s + 1];
      bad |= begin > end || (s == 0 && begin != 0) || (s == a.slots - 1 && end != a.N);
      offsets[s] = begin;
    }
    if (__syncthreads_or(bad)) {
      if (all_rows)
        for (int64_t n = tid; n < a.N; n += kTableThreads) a.rows[n] = -1;
      return;
    }
  }
  int64_t items = 0;
  for (int base = 0; base < a.slots; base += kTableThreads) {
    const int s = base + tid;
    int64_t mine = 0, total;
    if (s < a.slots) {
      const int fresh = a.offsets == nullptr ? a.T : a.offsets[s + 1] - a.offsets[s];
      mine = a.held(a.length(s) + fresh) - a.held(a.length(s));
    }
    const int64_t upto = items + scan_block(mine, tid, ends, &total);
    if (s < a.slots) first[s] = static_cast<int>(upto - mine);
    items += total;
  }
  __syncthreads();
  for (int64_t k = tid; k < items; k += kTableThreads) {
    const int s = slot_of_item(first, a.slots, static_cast<int>(k));
    const int64_t column = a.held(a.length(s)) + k - first[s];
    a.tables[static_cast<int64_t>(s) * a.columns + column] = k < free ? a.pool[free - k] : -1;
  }
  if (tid == 0) a.pool[0] = static_cast<int>(max(int64_t{0}, free - items));
  if (!all_rows) return;
  __syncthreads();
  for (int64_t n = tid; n < a.N; n += kTableThreads)
    a.rows[n] = row_of_token(a, a.offsets == nullptr ? nullptr : offsets, static_cast<int>(n));
}

// The rows of many tokens, once the tables are made: one block would write them at 8 bytes a thread and turn.
__global__ __launch_bounds__(kThreads) void page_rows_kernel(TableArgs a) {
  int bad = 0;
  if (a.offsets != nullptr) {
    for (int s = threadIdx.x; s < a.slots; s += kThreads) {
      const int begin = a.offsets[s], end = a.offsets[s + 1];
      bad |= begin > end || (s == 0 && begin != 0) || (s == a.slots - 1 && end != a.N);
    }
    bad = __syncthreads_or(bad);
  }
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (n < a.N) a.rows[n] = bad ? -1 : row_of_token(a, a.offsets, static_cast<int>(n));
}

// The entries that a release takes from the slots, in order: `first[s]` is the number of a slot's first one.
struct Released {
  const TableArgs& a;
  const int* first;
  int64_t count;
  bool all;  // no slot keeps any
  __device__ __forceinline__ int32_t* operator[](int64_t k) const {
    const int s = slot_of_item(first, a.slots, static_cast<int>(k));
    return a.tables + static_cast<int64_t>(s) * a.columns + a.kept(s) + k - first[s];
  }
};
__device__ __forceinline__ Released released_entries(const TableArgs& a, int* first, int64_t* ends, int tid) {
  int64_t items = 0;
  int keeps = 0;
  for (int base = 0; base < a.slots; base += kTableThreads) {
    const int s = base + tid;
    int64_t mine = 0, total;
    if (s < a.slots) {
      const int64_t kept = a.kept(s);
      mine = a.held(a.length(s)) - kept;
      keeps |= kept > 0;
    }
    const int64_t upto = items + scan_block(mine, tid, ends, &total);
    if (s < a.slots) first[s] = static_cast<int>(upto - mine);
    items += total;
  }
  const bool some = __syncthreads_or(keeps);
  return {a, first, items, !some};
}

// A bit for each page from `low` on.
struct Marks {
  uint32_t* words;
  int64_t low;
  int pages;
  __device__ __forceinline__ bool covers(int id) const { return id >= low && id - low < pages; }
  __device__ __forceinline__ uint32_t bit(int id) const { return 1u << ((id - low) & 31); }
  __device__ __forceinline__ uint32_t* word(int id) const { return words + (id - low) / 32; }
  __device__ __forceinline__ bool has(int id) const { return *word(id) & bit(id); }
  // whether it was there before
  __device__ __forceinline__ bool add(int id) const { return atomicOr(word(id), bit(id)) & bit(id); }
  __device__ __forceinline__ void remove(int id) const { atomicAnd(word(id), ~bit(id)); }
};
__device__ __forceinline__ Marks no_marks(const TableArgs& a, uint32_t* words, int64_t low, int tid) {
  const int pages = static_cast<int>(min(a.pages - low, static_cast<int64_t>(kMarkedPages)));
  for (int i = tid; i < (pages + 31) / 32; i += kTableThreads) words[i] = 0;
  __syncthreads();
  return {words, low, pages};
}

// A page may be in several tables (a prompt in common): ahead of a release, entries that it would take
// from a slot become -1 where some slot keeps their page.  Every block marks the pages that are to go
// back, looks for them among its share of the entries that stay, and has an entry dropped if it found
// its page; blocks that read an entry which another one has dropped pass it over.  Latency again: 7.2 us
// for 64 slots of up to 9000 tokens on pages of 16, of which eight each are taken back, 7.7 for 256 slots;
// with the release 23 us for 512 slots of 20000 (8 without this look at 640000 entries).
__global__ __launch_bounds__(kTableThreads) void page_tables_keep_kernel(TableArgs a) {
  extern __shared__ int first[];
  __shared__ int64_t ends[kTableThreads / 64];
  __shared__ uint32_t words[kMarkedPages / 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Released released = released_entries(a, first, ends, tid);
  if (released.count == 0 || released.all) return;
  const int per = (a.columns + kRun - 1) / kRun;
  const int64_t runs = static_cast<int64_t>(a.slots) * per;
  for (int64_t low = 0; low < a.pages; low += kMarkedPages) {
    const Marks marks = no_marks(a, words, low, tid);
    int any = 0;
    for (int64_t k = tid; k < released.count; k += kTableThreads) {
      const int id = *released[k];
      if (!marks.covers(id)) continue;
      marks.add(id);
      any = 1;
    }
    if (!__syncthreads_or(any)) continue;
    int found = 0;
    for (int64_t run = static_cast<int64_t>(blockIdx.x) * (kTableThreads / 64) + wave; run < runs;
         run += static_cast<int64_t>(gridDim.x) * (kTableThreads / 64)) {
      const int s = static_cast<int>(run / per), begin = static_cast<int>(run % per) * kRun;
      const int end = static_cast<int>(min(a.kept(s), static_cast<int64_t>(begin) + kRun));
      if (begin >= end) continue;
      const int32_t* entries = a.tables + static_cast<int64_t>(s) * a.columns;
      int ids[kRun / 64];  // (all loads under way before the first look)
#pragma unroll
      for (int i = 0; i < kRun / 64; ++i) ids[i] = entries[min(begin + i * 64 + lane, end - 1)];
#pragma unroll
      for (int i = 0; i < kRun / 64; ++i)
        if (marks.covers(ids[i]) && marks.has(ids[i])) {
          marks.remove(ids[i]);
          found = 1;
        }
    }
    if (__syncthreads_or(found))
      for (int64_t k = tid; k < released.count; k += kTableThreads) {
        int32_t* entry = released[k];
        const int id = *entry;
        if (marks.covers(id) && !marks.has(id)) *entry = -1;
      }
    __syncthreads();
  }
}

// Whether the page of a thread's entry is marked already, or a thread before it has the same one: those
// of one turn of a block are compared with one another, which is rare.  Marks it.
__device__ __forceinline__ bool taken_before(const Marks& marks, int id, int* ids, int tid) {
  const bool covered = marks.covers(id);
  bool again = covered && marks.has(id);
  __syncthreads();
  const bool twice = covered && marks.add(id) && !again;
  if (__syncthreads_or(twice)) {
    ids[tid] = covered ? id : -1;
    __syncthreads();
#pragma unroll 8
    for (int t = 0; t < tid; ++t) again |= ids[t] == id;
    __syncthreads();
  }
  return covered && again;
}

// Numbering backwards: from the last entry to the first, each valid page goes on top of those before
// it.  A page that several slots give back goes with the first of its entries in that order; the others
// are passed over, those of pages beyond the first window in a look ahead of this one.  5.7 us for 64
// slots with 8 tokens each; each 1024 entries more take 3 us.
__global__ __launch_bounds__(kTableThreads) void page_tables_release_kernel(TableArgs a) {
  extern __shared__ int first[];
  __shared__ int64_t ends[kTableThreads / 64];
  __shared__ uint32_t words[kMarkedPages / 32];
  __shared__ int ids[kTableThreads];
  const int tid = threadIdx.x;
  const Released released = released_entries(a, first, ends, tid);
  for (int64_t low = kMarkedPages; low < a.pages && released.count > 0; low += kMarkedPages) {
    const Marks marks = no_marks(a, words, low, tid);
    for (int64_t base = released.count - 1; base >= 0; base -= kTableThreads) {
      int32_t* entry = base >= tid ? released[base - tid] : nullptr;
      if (taken_before(marks, entry != nullptr ? *entry : -1, ids, tid)) *entry = -1;
    }
    __syncthreads();
  }
  const Marks marks = no_marks(a, words, 0, tid);
  int64_t top = max(0, min(a.pool[0], a.pages));
  for (int64_t base = released.count - 1; base >= 0; base -= kTableThreads) {
    int id = -1;
    if (base >= tid) {
      int32_t* entry = released[base - tid];
      id = *entry;
      *entry = -1;
    }
    const bool valid = !taken_before(marks, id, ids, tid) && id >= 0 && id < a.pages;
    int64_t total;
    const int64_t place = top + scan_block(valid ? 1 : 0, tid, ends, &total);
    if (valid && place <= a.pages) a.pool[place] = id;
    top += total;
  }
  if (tid == 0) a.pool[0] = static_cast<int>(min(top, static_cast<int64_t>(a.pages)));
}

int check_page(int page) {
  return page >= 16 && page <= 256 && (page & (page - 1)) == 0
             ? 0
             : rosa_fail(1, "page must be a power of two in [16, 256]");
}

int check_tables(const rosa_page_tables* t) {
  if (t == nullptr) return rosa_fail(1, "page tables are NULL");
  if (t->slots < 1 || t->slots > kMostTableSlots) return rosa_fail(1, "page tables must have 1 to 8192 slots");
  if (t->columns < 1 || t->pages < 1) return rosa_fail(1, "page tables need columns >= 1 and pages >= 1");
  if (static_cast<int64_t>(t->slots) * t->columns > 0x7fffffff)
    return rosa_fail(1, "page tables must have fewer than 2^31 entries");
  if (const int bad = check_page(t->page)) return bad;
  if (!t->tables || !t->lengths || !t->pool) return rosa_fail(2, "page tables: NULL pointer");
  return 0;
}

TableArgs table_args(const rosa_page_tables& t) {
  TableArgs args{};
  args.tables = t.tables;
  args.pool = t.pool;
  args.lengths = t.lengths;
  args.slots = t.slots;
  args.columns = t.columns;
  args.pages = t.pages;
  args.page_shift = __builtin_ctz(static_cast<unsigned>(t.page));
  return args;
}

int check_call(const rosa_mixer_problem* p, const rosa_paged_cache* c, int count) {
  if (p == nullptr || c == nullptr) return rosa_fail(1, "paged update: problem or cache is NULL");
  if (p->dtype < ROSA_DTYPE_F32 || p->dtype > ROSA_DTYPE_BF16) return rosa_fail(1, "unsupported dtype");
  if (p->cu_seqlens != nullptr) {
    if (p->S < 1 || p->N < 1) return rosa_fail(1, "packed layout needs S >= 1 and N >= 1");
  } else {
    if (p->B < 1 || p->T < 1) return rosa_fail(1, "dense layout needs B >= 1 and T >= 1");
    if (static_cast<int64_t>(p->B) * p->T != p->N) return rosa_fail(1, "dense layout needs N = B * T");
  }
  if ((p->cu_seqlens != nullptr ? p->N : p->T) > kMostTokens)
    return rosa_fail(1, "a sequence must have at most 2^31 - 1025 tokens");
  if (p->H < 1 || p->Hkv < 1 || p->H % p->Hkv != 0)
    return rosa_fail(1, "query heads must be a positive multiple of key and value heads");
  if (p->D < 1 || p->D > kMostWidth || p->Dv < 1 || p->Dv > kMostWidth)
    return rosa_fail(1, "head widths must be in [1, 128]");
  if (!(p->scale > 0.0f) || !std::isfinite(p->scale)) return rosa_fail(1, "scale must be finite and > 0");
  if (const int bad = check_page(c->page)) return bad;
  if (c->columns < 1 || c->pages < 1) return rosa_fail(1, "paged update needs columns >= 1 and pages >= 1");
  if (count < 0 || count > kMostCount) return rosa_fail(1, "count must be in [0, 1024]");
  // Rows, blocks and portions are counted in 32 bits.
  const int64_t sequences = p->cu_seqlens == nullptr ? p->B : p->S;
  const int64_t most = int64_t{0x7fffffff} - 2048;
  if (static_cast<int64_t>(p->N) * p->H > most || sequences * p->Hkv > most / 64)
    return rosa_fail(1, "too many blocks: tokens and slots times heads must be fewer");
  return 0;
}

int launched(const char* what) {
  const hipError_t status = hipGetLastError();
  return status == hipSuccess ? 0 : rosa_fail_hip(status, what);
}

}  // namespace

}  // namespace rosa_mixer

using namespace rosa_mixer;

extern "C" {

int rosa_hip_page_tables_update(const rosa_page_tables* tables, const int32_t* cu_seqlens, int T,
                                int N, int64_t* rows, void* stream) {
  if (const int bad = check_tables(tables)) return bad;
  if (N < 0 || T < 0 || (cu_seqlens == nullptr && static_cast<int64_t>(tables->slots) * T != N))
    return rosa_fail(1, "page_tables_update: needs N >= 0 tokens, slots * T of them if dense");
  if (N == 0) return 0;
  if (!rows) return rosa_fail(2, "page_tables_update: NULL pointer");
  TableArgs args = table_args(*tables);
  args.offsets = cu_seqlens;
  args.rows = rows;
  args.T = T;
  args.N = N;
  const bool all_rows = N <= kTokensOfBlock;
  const auto on = static_cast<hipStream_t>(stream);
  const size_t shared = static_cast<size_t>(tables->slots) * (cu_seqlens ? 8 : 4);
  page_tables_update_kernel<<<1, kTableThreads, shared, on>>>(args, all_rows);
  if (!all_rows) page_rows_kernel<<<(N - 1) / kThreads + 1, kThreads, 0, on>>>(args);
  return launched("page_tables_update launch");
}

int rosa_hip_page_tables_release(const rosa_page_tables* tables, const int32_t* keep, void* stream) {
  if (const int bad = check_tables(tables)) return bad;
  if (!keep) return rosa_fail(2, "page_tables_release: NULL pointer");
  TableArgs args = table_args(*tables);
  args.keep = keep;
  const auto on = static_cast<hipStream_t>(stream);
  const size_t shared = static_cast<size_t>(tables->slots) * 4;
  const int64_t runs = static_cast<int64_t>(tables->slots) * ((tables->columns - 1) / kRun + 1);
  const int64_t blocks = std::min<int64_t>((runs - 1) / (kTableThreads / 64) + 1, kBlocks / 2);
  page_tables_keep_kernel<<<static_cast<unsigned>(blocks), kTableThreads, shared, on>>>(args);
  page_tables_release_kernel<<<1, kTableThreads, shared, on>>>(args);
  return launched("page_tables_release launch");
}

size_t rosa_hip_paged_workspace_bytes(const rosa_mixer_problem* problem,
                                      const rosa_paged_cache* cache, int count) {
  if (check_call(problem, cache, count) != 0) return 0;
  return std::max<size_t>(paged_plan(*problem, *cache, count).bytes(), 256);
}

int rosa_hip_paged_update(const rosa_mixer_problem* problem, const rosa_paged_cache* cache, int count,
                          const rosa_mixer_tensor* query, const rosa_mixer_tensor* key,
                          const rosa_mixer_tensor* value, void* output, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (const int bad = check_call(problem, cache, count)) return bad;
  for (const rosa_mixer_tensor* t : {query, key, value})
    if (t == nullptr || t->data == nullptr) return rosa_fail(2, "paged_update: NULL tensor");
  if (!cache->key_pages || !cache->value_pages || !cache->tables || !cache->lengths || !cache->rows || !output)
    return rosa_fail(2, "paged_update: NULL pointer");
  if (count > 0 && !cache->key_bounds) return rosa_fail(2, "paged_update: selected pages need key_bounds");
  const size_t needed = paged_plan(*problem, *cache, count).bytes();
  if (needed > 0 && !workspace) return rosa_fail(2, "paged_update: NULL pointer");
  if (workspace_bytes < needed) return rosa_fail(3, "paged_update: workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return rosa_fail(1, "mixer workspaces must be 16-byte aligned");
  PagedCall call{};
  call.problem = problem;
  call.cache = cache;
  call.count = count;
  call.query = query;
  call.key = key;
  call.value = value;
  call.out = output;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  (problem->dtype == ROSA_DTYPE_F32   ? paged_update_float32
   : problem->dtype == ROSA_DTYPE_F16 ? paged_update_float16
                                      : paged_update_bfloat16)(call);
  return launched("paged_update launch");
}

}  // extern "C"
