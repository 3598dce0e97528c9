// Dispatcher layer of the mixers (module rosa_soft_amd._C, beside rosa_dispatch.cpp): schemas,
// validation, allocation and stream of decayed linear attention and window attention.  Inputs are
// taken with their strides as long as the elements of a head are neighbours; outputs are
// contiguous and of the inputs' dtype.  No device code lives in this file.

#include <ATen/Context.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <tuple>

#include "../../include/rosa_soft_hip.h"

namespace {

using torch::Tensor;
using OptionalTensor = std::optional<Tensor>;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

constexpr int64_t kIntMax = std::numeric_limits<int>::max();
constexpr int64_t kMostWidth = 128;
constexpr int64_t kMostSinks = 64;

int dtype_code(c10::ScalarType dtype) {
  switch (dtype) {
    case torch::kFloat32: return ROSA_DTYPE_F32;
    case torch::kFloat16: return ROSA_DTYPE_F16;
    case torch::kBFloat16: return ROSA_DTYPE_BF16;
    default: return -1;
  }
}

void* current_stream() {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

void raise_on_failure(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed (", status, "): ", rosa_hip_last_error());
}

// The backward of this build is not recorded into HIP graphs, however it is reached.
void refuse_capture(const char* what) {
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  const hipError_t queried = hipStreamIsCapturing(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(), &capture);
  TORCH_CHECK(queried == hipSuccess, what, ": hipStreamIsCapturing failed: ",
              hipGetErrorString(queried));
  TORCH_CHECK(capture == hipStreamCaptureStatusNone, what,
              ": the backward cannot be recorded into a HIP graph in this build; run it eagerly");
}

// elements of a head next to each other; everything else by strides
Tensor readable(const Tensor& tensor) {
  return tensor.size(-1) == 1 || tensor.stride(-1) == 1 ? tensor : tensor.contiguous();
}

rosa_mixer_tensor describe(const Tensor& tensor) {
  const bool dense = tensor.dim() == 4;
  return {tensor.data_ptr(), dense ? tensor.stride(0) : 0, tensor.stride(dense ? 1 : 0),
          tensor.stride(dense ? 2 : 1)};
}

// A call's tensors after its checks, kept alive for the launches.
struct Call {
  Tensor query, key, value, offsets;
  rosa_mixer_problem problem;
  rosa_mixer_tensor q, k, v;
};

void check_call(const Tensor& query, const Tensor& key, const Tensor& value,
                const OptionalTensor& cu_seqlens, double scale) {
  const int64_t rank = cu_seqlens ? 3 : 4;
  TORCH_CHECK(query.is_cuda() && key.is_cuda() && value.is_cuda(),
              "query, key and value must be CUDA tensors");
  TORCH_CHECK(query.device() == key.device() && query.device() == value.device(),
              "query, key and value must be on the same CUDA device");
  TORCH_CHECK(dtype_code(query.scalar_type()) >= 0,
              "query must be float32, float16, or bfloat16");
  TORCH_CHECK(query.scalar_type() == key.scalar_type() &&
                  query.scalar_type() == value.scalar_type(),
              "query, key and value must have the same dtype");
  TORCH_CHECK(query.dim() == rank && key.dim() == rank && value.dim() == rank,
              "query, key and value must have shape ",
              cu_seqlens ? "(N, heads, width)" : "(B, T, heads, width)");
  for (int64_t axis = 0; axis + 2 < rank; ++axis)
    TORCH_CHECK(query.size(axis) == key.size(axis) && query.size(axis) == value.size(axis),
                "query, key and value must share their token dimensions");
  TORCH_CHECK(key.size(-2) == value.size(-2), "key and value head counts must match");
  TORCH_CHECK(key.size(-2) > 0 && query.size(-2) > 0 && query.size(-2) % key.size(-2) == 0,
              "query heads must be a positive multiple of key heads");
  TORCH_CHECK(query.size(-1) == key.size(-1), "query and key widths must match");
  TORCH_CHECK(query.size(-1) >= 1 && query.size(-1) <= kMostWidth && value.size(-1) >= 1 &&
                  value.size(-1) <= kMostWidth,
              "head widths must be in [1, 128]");
  const int64_t tokens = query.numel() / (query.size(-2) * query.size(-1));
  TORCH_CHECK(tokens <= kIntMax && tokens * query.size(-2) <= kIntMax,
              "tokens times heads must fit in int32");
  const float narrowed = static_cast<float>(scale);
  TORCH_CHECK(std::isnormal(narrowed) && narrowed > 0.0f,
              "scale must be representable as a positive normal float32 value");
  if (cu_seqlens) {
    TORCH_CHECK(cu_seqlens->is_cuda() && cu_seqlens->device() == query.device(),
                "cu_seqlens must be on the CUDA device of the inputs");
    TORCH_CHECK(cu_seqlens->scalar_type() == torch::kInt32, "cu_seqlens must be int32");
    TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->numel() >= 2,
                "cu_seqlens must be one-dimensional with at least two entries");
    TORCH_CHECK(cu_seqlens->numel() - 1 <= kIntMax, "too many packed sequences");
  }
}

Call make_call(const Tensor& query, const Tensor& key, const Tensor& value,
               const OptionalTensor& cu_seqlens, double scale) {
  Call call;
  call.query = readable(query);
  call.key = readable(key);
  call.value = readable(value);
  rosa_mixer_problem& p = call.problem;
  p = {};
  p.dtype = dtype_code(query.scalar_type());
  if (cu_seqlens) {
    call.offsets = cu_seqlens->contiguous();
    p.cu_seqlens = call.offsets.data_ptr<int32_t>();
    p.N = static_cast<int>(query.size(0));
    p.S = static_cast<int>(call.offsets.numel() - 1);
  } else {
    p.B = static_cast<int>(query.size(0));
    p.T = static_cast<int>(query.size(1));
    p.N = p.B * p.T;
  }
  p.H = static_cast<int>(query.size(-2));
  p.Hkv = static_cast<int>(key.size(-2));
  p.D = static_cast<int>(query.size(-1));
  p.Dv = static_cast<int>(value.size(-1));
  p.scale = static_cast<float>(scale);
  call.q = describe(call.query);
  call.k = describe(call.key);
  call.v = describe(call.value);
  return call;
}

Tensor new_output(const Call& call) {
  auto sizes = call.query.sizes().vec();
  sizes.back() = call.value.size(-1);
  return torch::empty(sizes, call.query.options());
}

Tensor new_workspace(size_t bytes, const Tensor& like) {
  TORCH_CHECK(bytes > 0, "mixer workspace: ", rosa_hip_last_error());
  return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

Tensor check_log_decay(const Tensor& log_decay, const Tensor& query) {
  TORCH_CHECK(log_decay.is_cuda() && log_decay.device() == query.device(),
              "log_decay must be on the CUDA device of the inputs");
  TORCH_CHECK(log_decay.scalar_type() == torch::kFloat32, "log_decay must be float32");
  TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == query.size(-2),
              "log_decay must have one entry per query head");
  return log_decay.contiguous();
}

void check_grad_output(const Tensor& grad_output, const Tensor& query, const Tensor& value) {
  auto sizes = query.sizes().vec();
  sizes.back() = value.size(-1);
  TORCH_CHECK(grad_output.device() == query.device(),
              "grad_output must be on the CUDA device of the inputs");
  TORCH_CHECK(grad_output.scalar_type() == query.scalar_type(), "grad_output dtype mismatch");
  TORCH_CHECK(grad_output.sizes() == torch::IntArrayRef(sizes), "grad_output shape mismatch");
}

void check_training(const Tensor& query) {
  TORCH_CHECK(query.numel() > 0, "batch and sequence dimensions must be >= 1");
}

void check_window(int64_t window, int64_t sinks) {
  TORCH_CHECK(window >= 1, "window must be >= 1");
  TORCH_CHECK(sinks >= 0 && sinks <= kMostSinks, "sinks must be in [0, 64]");
}

int narrow_window(int64_t window) { return static_cast<int>(std::min(window, kIntMax)); }

void check_mask(int64_t gradient_mask) {
  TORCH_CHECK(gradient_mask >= 1 && gradient_mask <= 7,
              "gradient_mask must be an integer bit mask in [1, 7]");
}

// the requested gradients, each in the layout and dtype of its input
struct Gradients {
  Tensor query, key, value;
  Gradients(const Call& call, int64_t mask) {
    const auto make = [&](int bit, const Tensor& like) {
      return (mask & bit) != 0 ? torch::empty(like.sizes(), like.options())
                               : torch::empty({0}, like.options());
    };
    query = make(ROSA_GRAD_QUERY, call.query);
    key = make(ROSA_GRAD_KEY, call.key);
    value = make(ROSA_GRAD_VALUE, call.value);
  }
  static void* pointer(const Tensor& tensor) {
    return tensor.numel() > 0 ? tensor.data_ptr() : nullptr;
  }
};

// ---------------------------------------------------------------------------
// decayed linear attention
// ---------------------------------------------------------------------------

Tensor decay_attention_op(const Tensor& query, const Tensor& key, const Tensor& value,
                          const OptionalTensor& cu_seqlens, const Tensor& log_decay, double scale) {
  check_call(query, key, value, cu_seqlens, scale);
  check_training(query);
  const Tensor rates = check_log_decay(log_decay, query);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor output = new_output(call);
  const size_t bytes = rosa_hip_decay_workspace_bytes(&call.problem, 0);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(rosa_hip_decay_forward(&call.problem, &call.q, &call.k, &call.v,
                                          rates.data_ptr<float>(), output.data_ptr(),
                                          workspace.data_ptr(), bytes, current_stream()),
                   "rosa_hip_decay_forward");
  return output;
}

std::tuple<Tensor, Tensor, Tensor> decay_attention_vjp_op(
    const Tensor& query, const Tensor& key, const Tensor& value, const OptionalTensor& cu_seqlens,
    const Tensor& log_decay, const Tensor& grad_output, double scale, int64_t gradient_mask) {
  check_call(query, key, value, cu_seqlens, scale);
  check_training(query);
  const Tensor rates = check_log_decay(log_decay, query);
  check_grad_output(grad_output, query, value);
  check_mask(gradient_mask);
  const Guard guard(query.device());
  refuse_capture("decay_attention_vjp");
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor grad = readable(grad_output);
  const rosa_mixer_tensor go = describe(grad);
  const Gradients gradients(call, gradient_mask);
  const size_t bytes = rosa_hip_decay_workspace_bytes(&call.problem, 1);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(
      rosa_hip_decay_backward(&call.problem, &call.q, &call.k, &call.v, &go,
                              rates.data_ptr<float>(), Gradients::pointer(gradients.query),
                              Gradients::pointer(gradients.key),
                              Gradients::pointer(gradients.value), workspace.data_ptr(), bytes,
                              current_stream()),
      "rosa_hip_decay_backward");
  return {gradients.query, gradients.key, gradients.value};
}

int64_t slot_count(const Tensor& query, const OptionalTensor& cu_seqlens) {
  return cu_seqlens ? cu_seqlens->numel() - 1 : query.size(0);
}

Tensor decay_attention_update_out_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                     const OptionalTensor& cu_seqlens, const Tensor& log_decay,
                                     const Tensor& state, Tensor state_out, double scale) {
  check_call(query, key, value, cu_seqlens, scale);
  const Tensor rates = check_log_decay(log_decay, query);
  const int64_t slots = slot_count(query, cu_seqlens);
  for (const Tensor* tensor : {&state, const_cast<const Tensor*>(&state_out)}) {
    TORCH_CHECK(tensor->device() == query.device(),
                "state must be on the CUDA device of the inputs");
    TORCH_CHECK(tensor->scalar_type() == torch::kFloat32, "state must be float32");
    TORCH_CHECK(tensor->sizes() == torch::IntArrayRef({slots, query.size(-2), query.size(-1),
                                                       value.size(-1)}),
                "state must have shape (slots, heads, key width, value width)");
    TORCH_CHECK(tensor->is_contiguous(), "state must be contiguous");
  }
  TORCH_CHECK(slots >= 1, "an update needs at least one slot");
  at::assert_no_partial_overlap(state_out, state);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor output = new_output(call);
  if (query.numel() == 0) {  // nobody brings a token
    if (!state_out.is_same(state)) state_out.copy_(state);
    return output;
  }
  const size_t bytes = rosa_hip_decay_workspace_bytes(&call.problem, 2);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(rosa_hip_decay_update(&call.problem, &call.q, &call.k, &call.v,
                                         rates.data_ptr<float>(), state.data_ptr<float>(),
                                         state_out.data_ptr<float>(), output.data_ptr(),
                                         workspace.data_ptr(), bytes, current_stream()),
                   "rosa_hip_decay_update");
  return output;
}

Tensor decay_attention_update_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                 const OptionalTensor& cu_seqlens, const Tensor& log_decay,
                                 Tensor state, double scale) {
  return decay_attention_update_out_op(query, key, value, cu_seqlens, log_decay, state, state,
                                       scale);
}

// ---------------------------------------------------------------------------
// window attention
// ---------------------------------------------------------------------------

std::tuple<Tensor, Tensor> window_attention_op(const Tensor& query, const Tensor& key,
                                               const Tensor& value,
                                               const OptionalTensor& cu_seqlens, int64_t window,
                                               int64_t sinks, double scale, bool want_log_sum) {
  check_call(query, key, value, cu_seqlens, scale);
  check_training(query);
  check_window(window, sinks);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor output = new_output(call);
  const auto options = query.options().dtype(torch::kFloat32);
  const Tensor log_sum = want_log_sum ? torch::empty({call.problem.H, call.problem.N}, options)
                                      : torch::empty({0}, options);
  raise_on_failure(
      rosa_hip_window_forward(&call.problem, narrow_window(window), static_cast<int>(sinks),
                              &call.q, &call.k, &call.v, output.data_ptr(),
                              want_log_sum ? log_sum.data_ptr<float>() : nullptr,
                              current_stream()),
      "rosa_hip_window_forward");
  return {output, log_sum};
}

std::tuple<Tensor, Tensor, Tensor> window_attention_vjp_op(
    const Tensor& query, const Tensor& key, const Tensor& value, const OptionalTensor& cu_seqlens,
    const Tensor& output, const Tensor& log_sum, const Tensor& grad_output, int64_t window,
    int64_t sinks, double scale, int64_t gradient_mask) {
  check_call(query, key, value, cu_seqlens, scale);
  check_training(query);
  check_window(window, sinks);
  check_grad_output(grad_output, query, value);
  check_mask(gradient_mask);
  TORCH_CHECK(output.device() == query.device() && output.scalar_type() == query.scalar_type() &&
                  output.sizes() == grad_output.sizes(),
              "output must be the forward's");
  TORCH_CHECK(log_sum.device() == query.device() && log_sum.scalar_type() == torch::kFloat32 &&
                  log_sum.sizes() == torch::IntArrayRef({query.size(-2),
                                                         query.numel() / (query.size(-2) *
                                                                          query.size(-1))}),
              "log_sum must be the forward's");
  const Guard guard(query.device());
  refuse_capture("window_attention_vjp");
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor grad = readable(grad_output);
  const Tensor out = output.contiguous(), sums = log_sum.contiguous();
  const rosa_mixer_tensor go = describe(grad);
  const Gradients gradients(call, gradient_mask);
  const size_t bytes = rosa_hip_window_workspace_bytes(&call.problem, narrow_window(window),
                                                       static_cast<int>(sinks), 0);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(
      rosa_hip_window_backward(&call.problem, narrow_window(window), static_cast<int>(sinks),
                               &call.q, &call.k, &call.v, out.data_ptr(), sums.data_ptr<float>(),
                               &go, Gradients::pointer(gradients.query),
                               Gradients::pointer(gradients.key),
                               Gradients::pointer(gradients.value), workspace.data_ptr(), bytes,
                               current_stream()),
      "rosa_hip_window_backward");
  return {gradients.query, gradients.key, gradients.value};
}

Tensor window_attention_update_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                  Tensor key_cache, Tensor value_cache, const Tensor& lengths,
                                  const OptionalTensor& cu_seqlens, int64_t window, int64_t sinks,
                                  double scale) {
  check_call(query, key, value, cu_seqlens, scale);
  check_window(window, sinks);
  const int64_t slots = slot_count(query, cu_seqlens);
  TORCH_CHECK(slots >= 1, "an update needs at least one slot");
  TORCH_CHECK(key_cache.dim() == 4 && value_cache.dim() == 4,
              "caches must have shape (slots, key heads, capacity, width)");
  const int64_t capacity = key_cache.size(2);
  TORCH_CHECK(key_cache.sizes() ==
                      torch::IntArrayRef({slots, key.size(-2), capacity, key.size(-1)}) &&
                  value_cache.sizes() ==
                      torch::IntArrayRef({slots, key.size(-2), capacity, value.size(-1)}),
              "caches must have shape (slots, key heads, capacity, width)");
  TORCH_CHECK(window <= kIntMax && capacity >= window + sinks && capacity <= kIntMax,
              "caches must hold the sinks and the window, and fewer than 2^31 tokens");
  for (const Tensor* cache : {&key_cache, &value_cache}) {
    TORCH_CHECK(cache->device() == query.device(),
                "caches must be on the CUDA device of the inputs");
    TORCH_CHECK(cache->scalar_type() == query.scalar_type(),
                "caches must have the dtype of the inputs");
    TORCH_CHECK(cache->is_contiguous(), "caches must be contiguous");
    at::assert_no_overlap(*cache, query);
    at::assert_no_overlap(*cache, key);
    at::assert_no_overlap(*cache, value);
  }
  at::assert_no_overlap(key_cache, value_cache);
  TORCH_CHECK(lengths.device() == query.device() && lengths.scalar_type() == torch::kInt32 &&
                  lengths.dim() == 1 && lengths.size(0) == slots,
              "lengths must be int32 with one entry per slot, on the CUDA device of the inputs");
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, scale);
  const Tensor output = new_output(call);
  if (query.numel() == 0) return output;
  const Tensor seen = lengths.contiguous();
  const size_t bytes = rosa_hip_window_workspace_bytes(&call.problem, narrow_window(window),
                                                       static_cast<int>(sinks), capacity);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(
      rosa_hip_window_update(&call.problem, narrow_window(window), static_cast<int>(sinks),
                             &call.q, &call.k, &call.v, key_cache.data_ptr(),
                             value_cache.data_ptr(), capacity, seen.data_ptr<int32_t>(),
                             output.data_ptr(), workspace.data_ptr(), bytes, current_stream()),
      "rosa_hip_window_update");
  return output;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rosa_soft, m) {
  m.def(
      "decay_attention(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, float scale) -> Tensor output");
  m.def(
      "decay_attention_vjp(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor grad_output, float scale, int gradient_mask) -> "
      "(Tensor grad_query, Tensor grad_key, Tensor grad_value)");
  m.def(
      "decay_attention_update(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor(a!) state, float scale) -> Tensor output");
  m.def(
      "decay_attention_update_out(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor state, Tensor(a!) state_out, float scale) -> Tensor output");
  m.def(
      "window_attention(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, int window, "
      "int sinks, float scale, bool want_log_sum) -> (Tensor output, Tensor log_sum)");
  m.def(
      "window_attention_vjp(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor output, Tensor log_sum, Tensor grad_output, int window, int sinks, float scale, "
      "int gradient_mask) -> (Tensor grad_query, Tensor grad_key, Tensor grad_value)");
  m.def(
      "window_attention_update(Tensor query, Tensor key, Tensor value, Tensor(a!) key_cache, "
      "Tensor(b!) value_cache, Tensor lengths, Tensor? cu_seqlens, int window, int sinks, "
      "float scale) -> Tensor output");
}

TORCH_LIBRARY_IMPL(rosa_soft, CUDA, m) {
  m.impl("decay_attention", &decay_attention_op);
  m.impl("decay_attention_vjp", &decay_attention_vjp_op);
  m.impl("decay_attention_update", &decay_attention_update_op);
  m.impl("decay_attention_update_out", &decay_attention_update_out_op);
  m.impl("window_attention", &window_attention_op);
  m.impl("window_attention_vjp", &window_attention_vjp_op);
  m.impl("window_attention_update", &window_attention_update_op);
}
