// What the C entry points of the paged cache (paged.hip) hand to the kernels of one element type
// and padded width (paged_instances.hip).
#pragma once

#include "mixer_calls.hpp"

namespace rosa_mixer {

// Slots of the tables that one call changes, at most: a prefix of each is kept in LDS.
constexpr int kMostTableSlots = 8192;
constexpr int kMostCount = 1024;  // selected pages of a token

// How the keys of one kernel's calls are shared out (see portion_of in paged_attention.hpp).
struct PagedShare {
  bool used;
  int rows;              // of a tile: (token, member of the group) pairs
  int unit_rows;         // of a tile that may be there
  int target;            // portions of a head of keys that a call is cut into, beside one for each tile
  int least;             // tiles of keys of a portion, at least
  int round;             // eighths of a portion from which on a walk has one more
  int64_t tiles;         // of rows, at most
  int64_t items;         // portions of a head of keys, at most
  int64_t parts;         // portions of tiles that are cut, at most: those with partial sums
  size_t part_bytes, task_bytes;
  size_t bytes() const { return part_bytes + task_bytes; }
  // tiles that are cut, at most: each has two parts or more
  int64_t cut() const { return parts / 2 < tiles ? parts / 2 : tiles; }
};

struct PagedPlan {
  int width;                // padded
  PagedShare few, many;     // slots of few rows, and the others
  int most_few;             // rows of a slot that few takes
  size_t list_bytes, seen_bytes, score_bytes;  // selected pages
  size_t bytes() const { return few.bytes() + many.bytes() + list_bytes + seen_bytes + score_bytes; }
};
PagedPlan paged_plan(const rosa_mixer_problem& p, const rosa_paged_cache& cache, int count);

struct PagedCall {
  const rosa_mixer_problem* problem;
  const rosa_paged_cache* cache;
  int count;  // selected pages of a token, or 0: all
  const rosa_mixer_tensor *query, *key, *value;
  void* out;
  char* workspace;
  hipStream_t stream;
};

void paged_update_float32(const PagedCall& call);
void paged_update_float16(const PagedCall& call);
void paged_update_bfloat16(const PagedCall& call);

}  // namespace rosa_mixer
