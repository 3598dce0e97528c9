// What the C entry points of the mixers (mixers.hip) hand to the kernels of one element type and
// padded width (mixer_instances.hip), and how a failure is reported.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/rosa_soft_hip.h"

// (defined beside rosa_hip_last_error)
__attribute__((visibility("hidden"))) int rosa_fail(int code, const char* message);
__attribute__((visibility("hidden"))) int rosa_fail_hip(hipError_t status, const char* what);

namespace rosa_mixer {

constexpr int kWidths[] = {32, 64, 128};  // padded head widths that kernels exist for
constexpr int kMostWidth = 128;
constexpr int kMostSinks = 64;
constexpr int kMostSplits = 512;
// Tokens of a call that is packed, or of a sequence: kernels count a tile and a window past the last.
constexpr int kMostTokens = 0x7fffffff - 1024;

constexpr int padded_width(int widest) { return widest <= 32 ? 32 : widest <= 64 ? 64 : 128; }

struct WindowCall {
  const rosa_mixer_problem* problem;
  int window, sinks;
  const rosa_mixer_tensor *query, *key, *value, *grad_output;
  const void* output;
  float* log_sum;                             // [H][tokens], exponents of two
  void *out, *grad_query, *grad_key, *grad_value;
  void *key_cache, *value_cache;              // update: [S][Hkv][capacity][width]
  const int32_t* lengths;
  int64_t capacity;
  char* workspace;
  hipStream_t stream;
};

struct DecayCall {
  const rosa_mixer_problem* problem;
  const rosa_mixer_tensor *query, *key, *value, *grad_output;
  const float* log_decay;
  void *out, *grad_query, *grad_key, *grad_value;
  const float* state_in;                      // update: [S][H][D][Dv]
  float* state_out;
  char* workspace;
  hipStream_t stream;
};

// Work division, on the host alone.  Arrays in a workspace begin 256 bytes apart, whatever their
// widths: kernels store four elements at once.
constexpr size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }
constexpr int decay_slice(int width) { return width < 64 ? width : 64; }  // value columns of a block
struct DecayPlan {
  int width;            // padded width of keys
  int segment;          // tokens of a segment; >= the longest sequence where there is but one
  bool segmented;
  int64_t slots;
  size_t state_bytes;   // incoming states of all segments, all passes
  size_t key_partial_bytes, value_partial_bytes;  // gradients of shared heads before the sum over a group
};
DecayPlan decay_plan(const rosa_mixer_problem& p, int passes);

struct WindowPlan {
  int64_t sink_slots;   // pieces of the tokens that see sinks beyond their window, or none
  int sink_rows;        // tokens of a piece
  int sink_far;         // sequences of no more tokens than this have no pieces
  int key_block;        // keys of a block of the keys' gradients
  int key_parts;        // blocks that share the walk over the tokens that see them
  size_t delta_bytes, sink_bytes, sink_part_bytes, key_sum_bytes, value_sum_bytes;
  size_t bytes() const {
    return delta_bytes + sink_bytes + sink_part_bytes + key_sum_bytes + value_sum_bytes;
  }
};
WindowPlan window_plan(const rosa_mixer_problem& p, int window, int sinks);

struct TokenPlan {
  int splits, head_blocks;
  size_t partial_bytes;
};
TokenPlan token_plan(const rosa_mixer_problem& p, int64_t capacity);

constexpr int kSinkRows = 256;    // tokens of a piece, where memory allows

#define ROSA_MIXER_LAUNCHERS(NAME)                                     \
  void window_forward_##NAME(const WindowCall& call);                  \
  void window_backward_##NAME(const WindowCall& call);                 \
  void window_update_##NAME(const WindowCall& call);                   \
  void decay_forward_##NAME(const DecayCall& call);                    \
  void decay_backward_##NAME(const DecayCall& call);                   \
  void decay_update_##NAME(const DecayCall& call);
ROSA_MIXER_LAUNCHERS(float32)
ROSA_MIXER_LAUNCHERS(float16)
ROSA_MIXER_LAUNCHERS(bfloat16)

}  // namespace rosa_mixer
