// C entry points of the mixers: checks, work division and workspace, in host arithmetic; the
// kernels are in mixer_instances.hip, one translation unit per element type and operator.
#include "mixer_calls.hpp"

#include <algorithm>
#include <cmath>

namespace rosa_mixer {

namespace {

constexpr int kDecayChunk = 64;
// Blocks that a launch should have: two for each of 256 compute units.
constexpr int64_t kBlocks = 512;
// Most memory that the states between the segments of a call may take, and the sums of sinks.
constexpr int64_t kMostStateBytes = int64_t{2} << 30;

int64_t tile_slots(const rosa_mixer_problem& p, int64_t rows) {
  return p.cu_seqlens == nullptr ? static_cast<int64_t>(p.B) * ((p.T + rows - 1) / rows)
                                 : static_cast<int64_t>(p.N) / rows + p.S;
}

}  // namespace

// A sequence is walked by one block per head and slice of 64 value columns, chunk after chunk; where
// that leaves compute units idle it is cut into segments, whose states are summed by a walk of
// their own over keys and values and joined.  The number of segments is the one with the least
// time by this count, in chunks of a block that has a compute unit to itself (2.5 us at a width of
// 128): two blocks on one take 1.65 times as long, a chunk that is only summed takes half as long,
// a block's beginning and end take one and a half chunks, and the states' traffic and the two more
// launches take what they take.  At 2 x 4096 tokens and 32 heads of 128, bfloat16, forward:
// 1 segment 128 us, 2 126, 4 113, 8 129; backward, with three times the blocks: 1 segment 205 us,
// 2 266, 4 293.  12 heads of 48 and 80, float16, 6728 tokens, forward: 1 segment 179 us, 8 57,
// 18 51, 53 81.  Four prompts of 2048 tokens, 32 heads of 128 with their states: 1 segment 89 us,
// 2 127, 4 136.  Segments have at least two chunks.
DecayPlan decay_plan(const rosa_mixer_problem& p, int passes) {
  DecayPlan plan{};
  // The backward passes have both widths in both places.  Forward, values are sliced anyway, and
  // the narrower kernel would only make more slices of wide ones.
  plan.width = padded_width(std::max(p.D, passes > 1 ? p.Dv : std::min(p.Dv, 64)));
  const int slice = decay_slice(plan.width);
  const auto slices = [slice](int columns) { return (columns + slice - 1) / slice; };
  const int64_t longest = p.cu_seqlens == nullptr ? p.T : p.N;
  // blocks of every slot; the queries' and keys' gradients have D columns
  const int64_t walks = static_cast<int64_t>(p.H) * (slices(p.Dv) + (passes > 1 ? 2 * slices(p.D) : 0));
  const int64_t state = static_cast<int64_t>(passes) * p.H * p.D * p.Dv * 4;
  const int64_t chunks = (longest + kDecayChunk - 1) / kDecayChunk;
  const auto chunk_time = [](int64_t blocks) {  // of all blocks together
    const int64_t left = blocks % kBlocks;
    return 1.65 * static_cast<double>(blocks / kBlocks) + (left == 0 ? 0.0 : left <= kBlocks / 2 ? 1.0 : 1.65);
  };
  int64_t best_segment = chunks;
  double best = -1.0;
  for (int64_t cuts = 1; cuts <= std::min<int64_t>(chunks, 256); ++cuts) {
    const int64_t segment = (chunks + cuts - 1) / cuts;
    if (cuts > 1 && segment < 2) break;
    const int64_t slots = tile_slots(p, segment * kDecayChunk);
    // (packed: how many slots hold tokens is not known here; as many as the tokens fill)
    const int64_t filled = p.cu_seqlens == nullptr
                               ? slots
                               : std::max<int64_t>(1, p.N / (segment * kDecayChunk));
    const double length = static_cast<double>(segment) + 1.5;
    double cost = chunk_time(filled * walks) * length;
    if (cuts > 1) {
      if (slots * state > kMostStateBytes) break;
      const double joined = 2.0 * static_cast<double>(filled * state) / 4.5e6 + 8.0;  // us
      cost += 0.5 * chunk_time(filled * walks * (cuts - 1) / cuts) * length + joined / 2.5;
    }
    if (best < 0.0 || cost < best) {
      best = cost;
      best_segment = segment;
      plan.segmented = cuts > 1;
    }
  }
  plan.segment = static_cast<int>(std::min<int64_t>(best_segment, 0x7fffffff / kDecayChunk)) * kDecayChunk;
  plan.slots = tile_slots(p, plan.segment);
  plan.state_bytes = plan.segmented ? aligned(static_cast<size_t>(plan.slots) * state) : 0;
  if (passes > 1 && p.H > p.Hkv) {
    plan.key_partial_bytes = aligned(static_cast<size_t>(p.N) * p.H * p.D * 4);
    plan.value_partial_bytes = aligned(static_cast<size_t>(p.N) * p.H * p.Dv * 4);
  }
  return plan;
}

WindowPlan window_plan(const rosa_mixer_problem& p, int window, int sinks) {
  WindowPlan plan{};
  plan.delta_bytes = aligned(static_cast<size_t>(p.H) * p.N * 4);
  const int longest = p.cu_seqlens == nullptr ? p.T : p.N;
  // Keys of a block: 128, so that an operand read from LDS serves two products, or 64 where that
  // makes fewer than two blocks for each compute unit (240 blocks of 128 took 77 us where 448 of 64
  // take 56, 336 took 47 us where 600 take 31; 512 take 390 us, 1024 of 64 402) and where 128 do not
  // fit the registers (float32, 128 columns).  Few blocks with long walks have them shared out
  // until there are two for each compute unit, or one of those float32 ones, as long as a part has
  // eight tiles of tokens (4096 tokens, 8 query heads of 128 on one, window 1024, bfloat16: 59 us
  // with 8 parts, 89 with 4).
  const int columns = padded_width(std::max(p.D, p.Dv));
  const bool pairs = p.dtype != ROSA_DTYPE_F32 || columns < 128;
  plan.key_block = pairs && tile_slots(p, 128) * p.Hkv >= kBlocks ? 128 : 64;
  // Tokens beyond the sinks' window are up to eight more steps of the first key block's walk, or have
  // two kernels of their own: small calls wait for the host (256 tokens, 4 heads on 2, window 64:
  // 51 and 85 us a pass with the kernels, 46 and 76 without, on a fast and a slow host).
  const int64_t share = p.H / p.Hkv, near = static_cast<int64_t>(plan.key_block) + window - 1;
  int64_t far = near + 8 / (share * (pairs ? 1 : 2)) * 64;
  plan.sink_far = 0x7fffffff;
  // (the join has up to 64 blocks for a sequence's head of keys, counted in 32 bits)
  const int64_t sequences = p.cu_seqlens == nullptr ? p.B : p.S;
  if (sinks > 0 && longest > far && sequences * p.Hkv <= (int64_t{1} << 25)) {
    // A packed sequence with pieces begins more than `far` tokens behind the one before it, so that
    // tokens alone bound their number (see sink_place).  Their sums take at most kMostStateBytes or
    // as many bytes as the queries and output gradients in 16 bits: with many sinks and a short
    // window pieces get longer, and what is shorter than a piece is left to the first key block.
    const int64_t size = static_cast<int64_t>(sinks) * (p.D + p.Dv) * 4;
    const int64_t most = std::max<int64_t>(kMostStateBytes, int64_t{2} * p.N * p.H * (p.D + p.Dv));
    int64_t rows = kSinkRows, pieces, sums;
    for (;; rows *= 2, far = std::max(far, rows)) {
      pieces = p.cu_seqlens == nullptr ? tile_slots(p, rows) : p.N / rows + p.N / far + 1;
      sums = p.cu_seqlens == nullptr ? p.B : p.N / far + 1;
      if (longest <= far || (pieces * p.H + sums * p.Hkv) * size <= most) break;
    }
    if (longest > far) {
      plan.sink_rows = static_cast<int>(rows);
      plan.sink_far = static_cast<int>(far);
      plan.sink_slots = tile_slots(p, rows);
      plan.sink_bytes = aligned(sums * p.Hkv * size);
      plan.sink_part_bytes = aligned(pieces * p.H * size);
    }
  }
  const int64_t blocks = tile_slots(p, plan.key_block) * p.Hkv;
  const int64_t walk = std::min<int64_t>(longest, static_cast<int64_t>(plan.key_block) + window);
  const int64_t tiles = (walk + 63) / 64 * (p.H / p.Hkv);
  plan.key_parts = static_cast<int>(std::max<int64_t>(1, std::min((pairs ? kBlocks : kBlocks / 2) / blocks, tiles / 8)));
  if (plan.key_parts > 1) {
    const size_t rows = static_cast<size_t>(plan.key_parts) * p.N * p.Hkv;
    plan.key_sum_bytes = aligned(rows * p.D * 4);
    plan.value_sum_bytes = aligned(rows * p.Dv * 4);
  }
  return plan;
}

// A block of four waves takes tiles of 32 keys in turn; the cache of a slot is shared out until
// there are two blocks for a compute unit or a wave has but two tiles.
TokenPlan token_plan(const rosa_mixer_problem& p, int64_t capacity) {
  TokenPlan plan{};
  const int share = p.H / p.Hkv;
  plan.head_blocks = (share + 15) / 16;
  const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * plan.head_blocks;
  const int64_t tiles = (capacity + 31) / 32;
  plan.splits = static_cast<int>(std::max<int64_t>(1, std::min((kBlocks + blocks - 1) / blocks, tiles / 8)));
  if (plan.splits > 1)
    plan.partial_bytes = aligned(static_cast<size_t>(p.B) * p.H * plan.splits * (p.Dv + 2) * 4);
  return plan;
}

namespace {

int check(const rosa_mixer_problem* p, bool update) {
  if (p == nullptr) return rosa_fail(1, "mixer problem is NULL");
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
  // Blocks are counted in 32 bits.  The finest division is 64 tokens (or a sequence) of a head, with
  // two slices in each of three passes; of an update 16 value columns of a state.  (Joins of segments
  // and of sinks are bounded by the memory of what they join, and by window_plan.)
  const int64_t sequences = p->cu_seqlens == nullptr ? p->B : p->S;
  const int64_t most = int64_t{0x7fffffff} - 8;
  if ((static_cast<int64_t>(p->N) / 64 + sequences) * p->H * 6 > most ||
      (update && sequences * p->H * 8 > most))
    return rosa_fail(1, "too many blocks: tokens and sequences times heads must be fewer");
  return 0;
}

int check_tensors(std::initializer_list<const rosa_mixer_tensor*> tensors, const char* message) {
  for (const rosa_mixer_tensor* t : tensors)
    if (t == nullptr || t->data == nullptr) return rosa_fail(2, message);
  return 0;
}

int check_window(int window, int sinks) {
  if (window < 1) return rosa_fail(1, "window must be >= 1");
  if (sinks < 0 || sinks > kMostSinks) return rosa_fail(1, "sinks must be in [0, 64]");
  return 0;
}

int check_aligned(const void* workspace) {
  return reinterpret_cast<uintptr_t>(workspace) % 16 == 0
             ? 0
             : rosa_fail(1, "mixer workspaces must be 16-byte aligned");
}

int launched(const char* what) {
  const hipError_t status = hipGetLastError();
  return status == hipSuccess ? 0 : rosa_fail_hip(status, what);
}

template <typename Call>
void by_type(int dtype, const Call& call, void (*f32)(const Call&), void (*f16)(const Call&),
             void (*bf16)(const Call&)) {
  (dtype == ROSA_DTYPE_F32 ? f32 : dtype == ROSA_DTYPE_F16 ? f16 : bf16)(call);
}

bool is_token(const rosa_mixer_problem& p) { return p.cu_seqlens == nullptr && p.T == 1; }

size_t decay_bytes(const rosa_mixer_problem& p, int backward) {
  if (backward == 2 && is_token(p)) return 0;
  const DecayPlan plan = decay_plan(p, backward == 1 ? 3 : 1);
  return plan.state_bytes + plan.key_partial_bytes + plan.value_partial_bytes;
}

size_t window_update_bytes(const rosa_mixer_problem& p, int64_t capacity) {
  return is_token(p) ? token_plan(p, capacity).partial_bytes : 0;
}

}  // namespace

}  // namespace rosa_mixer

using namespace rosa_mixer;

extern "C" {

size_t rosa_hip_decay_workspace_bytes(const rosa_mixer_problem* problem, int call) {
  if (call < 0 || call > 2) {
    rosa_fail(1, "decay workspace: call must be 0 (forward), 1 (backward) or 2 (update)");
    return 0;
  }
  if (check(problem, call == 2) != 0) return 0;
  return std::max<size_t>(decay_bytes(*problem, call), 256);
}

int rosa_hip_decay_forward(const rosa_mixer_problem* problem, const rosa_mixer_tensor* query,
                           const rosa_mixer_tensor* key, const rosa_mixer_tensor* value,
                           const float* log_decay, void* output, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (const int bad = check(problem, false)) return bad;
  if (const int bad = check_tensors({query, key, value}, "decay_forward: NULL tensor")) return bad;
  if (!log_decay || !output || !workspace) return rosa_fail(2, "decay_forward: NULL pointer");
  if (workspace_bytes < decay_bytes(*problem, 0)) return rosa_fail(3, "decay_forward: workspace too small");
  if (const int bad = check_aligned(workspace)) return bad;
  DecayCall call{};
  call.problem = problem;
  call.query = query;
  call.key = key;
  call.value = value;
  call.log_decay = log_decay;
  call.out = output;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, decay_forward_float32, decay_forward_float16, decay_forward_bfloat16);
  return launched("decay_forward launch");
}

int rosa_hip_decay_backward(const rosa_mixer_problem* problem, const rosa_mixer_tensor* query,
                            const rosa_mixer_tensor* key, const rosa_mixer_tensor* value,
                            const rosa_mixer_tensor* grad_output, const float* log_decay,
                            void* grad_query, void* grad_key, void* grad_value, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int bad = check(problem, false)) return bad;
  if (const int bad = check_tensors({query, key, value, grad_output}, "decay_backward: NULL tensor"))
    return bad;
  if (!log_decay || !workspace) return rosa_fail(2, "decay_backward: NULL pointer");
  if (workspace_bytes < decay_bytes(*problem, 1)) return rosa_fail(3, "decay_backward: workspace too small");
  if (!grad_query && !grad_key && !grad_value) return 0;
  if (const int bad = check_aligned(workspace)) return bad;
  DecayCall call{};
  call.problem = problem;
  call.query = query;
  call.key = key;
  call.value = value;
  call.grad_output = grad_output;
  call.log_decay = log_decay;
  call.grad_query = grad_query;
  call.grad_key = grad_key;
  call.grad_value = grad_value;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, decay_backward_float32, decay_backward_float16, decay_backward_bfloat16);
  return launched("decay_backward launch");
}

int rosa_hip_decay_update(const rosa_mixer_problem* problem, const rosa_mixer_tensor* query,
                          const rosa_mixer_tensor* key, const rosa_mixer_tensor* value,
                          const float* log_decay, const float* state_in, float* state_out,
                          void* output, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int bad = check(problem, true)) return bad;
  if (const int bad = check_tensors({query, key, value}, "decay_update: NULL tensor")) return bad;
  if (!log_decay || !state_in || !state_out || !output)
    return rosa_fail(2, "decay_update: NULL pointer");
  const size_t needed = decay_bytes(*problem, 2);
  if (needed > 0 && !workspace) return rosa_fail(2, "decay_update: NULL pointer");
  if (workspace_bytes < needed) return rosa_fail(3, "decay_update: workspace too small");
  if (const int bad = check_aligned(workspace)) return bad;
  DecayCall call{};
  call.problem = problem;
  call.query = query;
  call.key = key;
  call.value = value;
  call.log_decay = log_decay;
  call.state_in = state_in;
  call.state_out = state_out;
  call.out = output;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, decay_update_float32, decay_update_float16, decay_update_bfloat16);
  return launched("decay_update launch");
}

size_t rosa_hip_window_workspace_bytes(const rosa_mixer_problem* problem, int window, int sinks,
                                       int64_t capacity) {
  if (check(problem, capacity > 0) != 0 || check_window(window, sinks) != 0) return 0;
  if (capacity > 0) return std::max<size_t>(window_update_bytes(*problem, capacity), 256);
  const WindowPlan plan = window_plan(*problem, window, sinks);
  return plan.bytes();
}

int rosa_hip_window_forward(const rosa_mixer_problem* problem, int window, int sinks,
                            const rosa_mixer_tensor* query, const rosa_mixer_tensor* key,
                            const rosa_mixer_tensor* value, void* output, float* log_sum,
                            void* stream) {
  if (const int bad = check(problem, false)) return bad;
  if (const int bad = check_window(window, sinks)) return bad;
  if (const int bad = check_tensors({query, key, value}, "window_forward: NULL tensor")) return bad;
  if (!output) return rosa_fail(2, "window_forward: NULL pointer");
  WindowCall call{};
  call.problem = problem;
  call.window = window;
  call.sinks = sinks;
  call.query = query;
  call.key = key;
  call.value = value;
  call.out = output;
  call.log_sum = log_sum;
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, window_forward_float32, window_forward_float16, window_forward_bfloat16);
  return launched("window_forward launch");
}

int rosa_hip_window_backward(const rosa_mixer_problem* problem, int window, int sinks,
                             const rosa_mixer_tensor* query, const rosa_mixer_tensor* key,
                             const rosa_mixer_tensor* value, const void* output,
                             const float* log_sum, const rosa_mixer_tensor* grad_output,
                             void* grad_query, void* grad_key, void* grad_value, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (const int bad = check(problem, false)) return bad;
  if (const int bad = check_window(window, sinks)) return bad;
  if (const int bad = check_tensors({query, key, value, grad_output}, "window_backward: NULL tensor"))
    return bad;
  if (!output || !log_sum || !workspace) return rosa_fail(2, "window_backward: NULL pointer");
  const WindowPlan plan = window_plan(*problem, window, sinks);
  if (workspace_bytes < plan.bytes())
    return rosa_fail(3, "window_backward: workspace too small");
  if (!grad_query && !grad_key && !grad_value) return 0;
  if (const int bad = check_aligned(workspace)) return bad;
  WindowCall call{};
  call.problem = problem;
  call.window = window;
  call.sinks = sinks;
  call.query = query;
  call.key = key;
  call.value = value;
  call.output = output;
  call.log_sum = const_cast<float*>(log_sum);
  call.grad_output = grad_output;
  call.grad_query = grad_query;
  call.grad_key = grad_key;
  call.grad_value = grad_value;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, window_backward_float32, window_backward_float16,
          window_backward_bfloat16);
  return launched("window_backward launch");
}

int rosa_hip_window_update(const rosa_mixer_problem* problem, int window, int sinks,
                           const rosa_mixer_tensor* query, const rosa_mixer_tensor* key,
                           const rosa_mixer_tensor* value, void* key_cache, void* value_cache,
                           int64_t capacity, const int32_t* lengths, void* output, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (const int bad = check(problem, true)) return bad;
  if (const int bad = check_window(window, sinks)) return bad;
  if (const int bad = check_tensors({query, key, value}, "window_update: NULL tensor")) return bad;
  if (!key_cache || !value_cache || !lengths || !output) return rosa_fail(2, "window_update: NULL pointer");
  if (capacity < static_cast<int64_t>(window) + sinks || capacity > 0x7fffffff)
    return rosa_fail(1, "window_update: the cache must hold the sinks and the window, and fewer than 2^31 tokens");
  const size_t needed = window_update_bytes(*problem, capacity);
  if (needed > 0 && !workspace) return rosa_fail(2, "window_update: NULL pointer");
  if (workspace_bytes < needed) return rosa_fail(3, "window_update: workspace too small");
  if (const int bad = check_aligned(workspace)) return bad;
  WindowCall call{};
  call.problem = problem;
  call.window = window;
  call.sinks = sinks;
  call.query = query;
  call.key = key;
  call.value = value;
  call.key_cache = key_cache;
  call.value_cache = value_cache;
  call.capacity = capacity;
  call.lengths = lengths;
  call.out = output;
  call.workspace = static_cast<char*>(workspace);
  call.stream = static_cast<hipStream_t>(stream);
  by_type(problem->dtype, call, window_update_float32, window_update_float16, window_update_bfloat16);
  return launched("window_update launch");
}

}  // extern "C"
