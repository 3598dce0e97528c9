// Dispatcher layer of the mixers (module rosa_soft_amd._C, beside rosa_dispatch.cpp): schemas,
// validation, allocation and stream of decayed linear attention and window attention.  Inputs are
// taken with their strides as long as the elements of a head are neighbours; outputs are
// contiguous and of the inputs' dtype.  All checks are made here, whatever the inputs' device, so
// that a call costs the interpreter nothing but the call; the autograd nodes are here as well, so
// that a backward does not wait for the interpreter.  No device code lives in this file.

#include <ATen/Context.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
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
constexpr int64_t kMostTokens = kIntMax - 1024;  // of a sequence, or of a packed call
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

bool is_capturing(const Tensor& on) {
  // (tracing: nothing is being launched)
  if (!on.is_cuda() || on.key_set().has(c10::DispatchKey::Python)) return false;
  const Guard guard(on.device());
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  const hipError_t queried = hipStreamIsCapturing(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(), &capture);
  TORCH_CHECK(queried == hipSuccess, "hipStreamIsCapturing failed: ", hipGetErrorString(queried));
  return capture != hipStreamCaptureStatusNone;
}

// The backward of this build is not recorded into HIP graphs, however it is reached.
void refuse_capture(const char* what, const Tensor& on) {
  TORCH_CHECK(!is_capturing(on), what,
              ": the backward cannot be recorded into a HIP graph in this build; capture the "
              "forward under torch.no_grad() or run the training step eagerly");
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

#define REQUIRE TORCH_CHECK_VALUE

// Shapes, dtypes, devices and scale; returns the scale.  `empty`: calls without tokens are meant.
double check_call(const Tensor& query, const Tensor& key, const Tensor& value,
                  const OptionalTensor& cu_seqlens, const std::optional<double>& scale, bool empty) {
  const int64_t rank = cu_seqlens ? 3 : 4;
  REQUIRE(query.dim() == rank && key.dim() == rank && value.dim() == rank,
          "query, key, and value must have shape ",
          cu_seqlens ? "(N, heads, width)" : "(B, T, heads, width)");
  int64_t tokens = 1;
  for (int64_t axis = 0; axis + 2 < rank; ++axis) {
    REQUIRE(query.size(axis) == key.size(axis) && query.size(axis) == value.size(axis),
            "all inputs must share their token dimensions");
    tokens *= query.size(axis);
  }
  const int64_t heads = query.size(-2), shared = key.size(-2), width = query.size(-1);
  REQUIRE(shared == value.size(-2), "key and value head counts must match");
  REQUIRE(heads >= 1 && shared >= 1, "query and key must have at least one head");
  REQUIRE(heads % shared == 0, "query heads must be divisible by key heads");
  REQUIRE(width == key.size(-1), "query and key widths must match");
  REQUIRE(width >= 1 && width <= kMostWidth && value.size(-1) >= 1 && value.size(-1) <= kMostWidth,
          "head widths must be in [1, 128]");
  REQUIRE(empty || tokens >= 1, "batch and sequence dimensions must be >= 1");
  REQUIRE(tokens <= kIntMax && tokens * heads <= kIntMax, "tokens times heads must fit in int32");
  REQUIRE(query.size(rank - 3) <= kMostTokens, "a sequence must have at most 2^31 - 1025 tokens");
  REQUIRE(query.device() == key.device() && query.device() == value.device(),
          "all inputs must be on the same device");
  REQUIRE(query.scalar_type() == key.scalar_type() && query.scalar_type() == value.scalar_type(),
          "all inputs must have the same dtype");
  REQUIRE(dtype_code(query.scalar_type()) >= 0, "the mixers support float32, float16, and bfloat16");
  if (cu_seqlens) {
    REQUIRE(cu_seqlens->device() == query.device(),
            "all inputs and cu_seqlens must be on the same device");
    REQUIRE(cu_seqlens->scalar_type() == torch::kInt32, "cu_seqlens must have dtype int32");
    REQUIRE(cu_seqlens->dim() == 1 && cu_seqlens->numel() >= 2,
            "cu_seqlens must be a one-dimensional int32 tensor");
    REQUIRE(cu_seqlens->numel() - 1 <= kIntMax, "too many packed sequences");
  }
  const double given = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(width));
  const float narrowed = static_cast<float>(given);
  REQUIRE(std::isnormal(narrowed) && narrowed > 0.0f,
          "scale must be representable as a positive normal float32 value");
  return given;
}

// Whether the spans of memory that two tensors' elements lie in meet.
bool overlap(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t axis = 0; axis < t.dim(); ++axis) last += (t.size(axis) - 1) * t.stride(axis);
    return reinterpret_cast<uintptr_t>(t.const_data_ptr()) + (last + 1) * t.element_size();
  };
  return reinterpret_cast<uintptr_t>(a.const_data_ptr()) < end(b) &&
         reinterpret_cast<uintptr_t>(b.const_data_ptr()) < end(a);
}

// (after every other check)
void check_device(const Tensor& query) { REQUIRE(query.is_cuda(), "the mixers require CUDA tensors"); }

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

void check_log_decay(const Tensor& log_decay, const Tensor& query) {
  REQUIRE(log_decay.dim() == 1 && log_decay.size(0) == query.size(-2),
          "log_decay must have one entry per query head");
  REQUIRE(log_decay.scalar_type() == torch::kFloat32, "log_decay must have dtype float32");
  REQUIRE(log_decay.device() == query.device(),
          "all inputs and log_decay must be on the same device");
}

void check_grad_output(const Tensor& grad_output, const Tensor& query, const Tensor& value) {
  auto sizes = query.sizes().vec();
  sizes.back() = value.size(-1);
  REQUIRE(grad_output.device() == query.device(),
          "grad_output must be on the device of the inputs");
  REQUIRE(grad_output.scalar_type() == query.scalar_type(), "grad_output dtype mismatch");
  REQUIRE(grad_output.sizes() == torch::IntArrayRef(sizes), "grad_output shape mismatch");
}

void check_window(int64_t window, int64_t sinks) {
  REQUIRE(window >= 1, "window must be >= 1");
  REQUIRE(sinks >= 0 && sinks <= kMostSinks, "sinks must be in [0, 64]");
}

int narrow_window(int64_t window) { return static_cast<int>(std::min(window, kIntMax)); }

void check_mask(int64_t gradient_mask) {
  REQUIRE(gradient_mask >= 1 && gradient_mask <= 7,
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

using Scale = std::optional<double>;
using Triple = std::tuple<Tensor, Tensor, Tensor>;

Tensor decay_attention_op(const Tensor& query, const Tensor& key, const Tensor& value,
                          const OptionalTensor& cu_seqlens, const Tensor& log_decay, Scale scale) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, false);
  check_log_decay(log_decay, query);
  check_device(query);
  const Guard guard(query.device());
  const Tensor rates = log_decay.contiguous();
  const Call call = make_call(query, key, value, cu_seqlens, factor);
  const Tensor output = new_output(call);
  const size_t bytes = rosa_hip_decay_workspace_bytes(&call.problem, 0);
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(rosa_hip_decay_forward(&call.problem, &call.q, &call.k, &call.v,
                                          rates.data_ptr<float>(), output.data_ptr(),
                                          workspace.data_ptr(), bytes, current_stream()),
                   "rosa_hip_decay_forward");
  return output;
}

Triple decay_attention_vjp_op(const Tensor& query, const Tensor& key, const Tensor& value,
                              const OptionalTensor& cu_seqlens, const Tensor& log_decay,
                              const Tensor& grad_output, Scale scale, int64_t gradient_mask) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, false);
  check_log_decay(log_decay, query);
  check_grad_output(grad_output, query, value);
  check_mask(gradient_mask);
  check_device(query);
  const Guard guard(query.device());
  refuse_capture("decay_attention_vjp", query);
  const Tensor rates = log_decay.contiguous();
  const Call call = make_call(query, key, value, cu_seqlens, factor);
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

int64_t check_slots(const Tensor& query, const OptionalTensor& cu_seqlens) {
  const int64_t slots = cu_seqlens ? cu_seqlens->numel() - 1 : query.size(0);
  REQUIRE(slots >= 1, "an update needs at least one slot");
  return slots;
}

Tensor decay_attention_update_out_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                     const OptionalTensor& cu_seqlens, const Tensor& log_decay,
                                     const Tensor& state, Tensor state_out, Scale scale) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, true);
  check_log_decay(log_decay, query);
  const int64_t slots = check_slots(query, cu_seqlens);
  for (const Tensor* tensor : {&state, const_cast<const Tensor*>(&state_out)}) {
    REQUIRE(tensor->sizes() ==
                torch::IntArrayRef({slots, query.size(-2), query.size(-1), value.size(-1)}),
            "state must have shape (slots, heads, key width, value width)");
    REQUIRE(tensor->scalar_type() == torch::kFloat32, "state must have dtype float32");
    REQUIRE(tensor->device() == query.device(), "all inputs and state must be on the same device");
    REQUIRE(tensor->is_contiguous(), "state must be contiguous");
    if (state_out.is_same(state)) break;
  }
  REQUIRE(state_out.const_data_ptr() == state.const_data_ptr() || !overlap(state_out, state),
          "state_out must be state or share no memory with it");
  for (const Tensor* input : {&query, &key, &value, &log_decay})
    REQUIRE(!overlap(state_out, *input), "states must share no memory with the inputs");
  check_device(query);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, factor);
  const Tensor output = new_output(call);
  if (query.numel() == 0) {  // nobody brings a token
    if (!state_out.is_same(state)) state_out.copy_(state);
    return output;
  }
  const Tensor rates = log_decay.contiguous();
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
                                 Tensor state, Scale scale) {
  return decay_attention_update_out_op(query, key, value, cu_seqlens, log_decay, state, state,
                                       scale);
}

// ---------------------------------------------------------------------------
// window attention
// ---------------------------------------------------------------------------

std::tuple<Tensor, Tensor> window_attention_op(const Tensor& query, const Tensor& key,
                                               const Tensor& value,
                                               const OptionalTensor& cu_seqlens, int64_t window,
                                               int64_t sinks, Scale scale, bool want_log_sum) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, false);
  check_window(window, sinks);
  check_device(query);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, factor);
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

Triple window_attention_vjp_op(const Tensor& query, const Tensor& key, const Tensor& value,
                               const OptionalTensor& cu_seqlens, const Tensor& output,
                               const Tensor& log_sum, const Tensor& grad_output, int64_t window,
                               int64_t sinks, Scale scale, int64_t gradient_mask) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, false);
  check_window(window, sinks);
  check_grad_output(grad_output, query, value);
  check_mask(gradient_mask);
  REQUIRE(output.device() == query.device() && output.scalar_type() == query.scalar_type() &&
              output.sizes() == grad_output.sizes(),
          "output must be the forward's");
  REQUIRE(log_sum.device() == query.device() && log_sum.scalar_type() == torch::kFloat32 &&
              log_sum.sizes() == torch::IntArrayRef({query.size(-2),
                                                     query.numel() / (query.size(-2) *
                                                                      query.size(-1))}),
          "log_sum must be the forward's");
  check_device(query);
  const Guard guard(query.device());
  refuse_capture("window_attention_vjp", query);
  const Call call = make_call(query, key, value, cu_seqlens, factor);
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
                                  Scale scale) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, true);
  check_window(window, sinks);
  const int64_t slots = check_slots(query, cu_seqlens);
  REQUIRE(key_cache.dim() == 4 && value_cache.dim() == 4,
          "caches must have shape (slots, key heads, capacity, width)");
  const int64_t capacity = key_cache.size(2);
  REQUIRE(key_cache.sizes() ==
                  torch::IntArrayRef({slots, key.size(-2), capacity, key.size(-1)}) &&
              value_cache.sizes() ==
                  torch::IntArrayRef({slots, key.size(-2), capacity, value.size(-1)}),
          "caches must have shape (slots, key heads, capacity, width)");
  REQUIRE(window <= kIntMax && capacity >= window + sinks && capacity <= kIntMax,
          "caches must hold the sinks and the window, and fewer than 2^31 tokens");
  for (const Tensor* cache : {&key_cache, &value_cache}) {
    REQUIRE(cache->scalar_type() == query.scalar_type(),
            "caches must have the dtype of the inputs");
    REQUIRE(cache->device() == query.device(), "all inputs and caches must be on the same device");
    REQUIRE(cache->is_contiguous(), "caches must be contiguous");
    REQUIRE(!overlap(*cache, query) && !overlap(*cache, key) && !overlap(*cache, value),
            "caches must share no memory with the inputs");
  }
  REQUIRE(!overlap(key_cache, value_cache), "the caches must share no memory");
  REQUIRE(lengths.dim() == 1 && lengths.size(0) == slots && lengths.scalar_type() == torch::kInt32,
          "lengths must be an int32 tensor with one entry per slot");
  REQUIRE(lengths.device() == query.device(), "all inputs and lengths must be on the same device");
  check_device(query);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, factor);
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

// ---------------------------------------------------------------------------
// autograd
// ---------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the operators as the dispatcher has them, so that tracing sees them
template <typename Signature>
auto operator_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<Signature>();
}
Tensor call_decay(const Tensor& q, const Tensor& k, const Tensor& v, const OptionalTensor& cu,
                  const Tensor& log_decay, Scale scale) {
  static const auto handle =
      operator_handle<decltype(decay_attention_op)>("rosa_soft::decay_attention");
  return handle.call(q, k, v, cu, log_decay, scale);
}
Triple call_decay_vjp(const Tensor& q, const Tensor& k, const Tensor& v, const OptionalTensor& cu,
                      const Tensor& log_decay, const Tensor& go, Scale scale, int64_t mask) {
  static const auto handle =
      operator_handle<decltype(decay_attention_vjp_op)>("rosa_soft::decay_attention_vjp");
  return handle.call(q, k, v, cu, log_decay, go, scale, mask);
}
std::tuple<Tensor, Tensor> call_window(const Tensor& q, const Tensor& k, const Tensor& v,
                                       const OptionalTensor& cu, int64_t window, int64_t sinks,
                                       Scale scale, bool want_log_sum) {
  static const auto handle =
      operator_handle<decltype(window_attention_op)>("rosa_soft::window_attention");
  return handle.call(q, k, v, cu, window, sinks, scale, want_log_sum);
}
Triple call_window_vjp(const Tensor& q, const Tensor& k, const Tensor& v, const OptionalTensor& cu,
                       const Tensor& output, const Tensor& log_sum, const Tensor& go,
                       int64_t window, int64_t sinks, Scale scale, int64_t mask) {
  static const auto handle =
      operator_handle<decltype(window_attention_vjp_op)>("rosa_soft::window_attention_vjp");
  return handle.call(q, k, v, cu, output, log_sum, go, window, sinks, scale, mask);
}

int64_t gradient_mask_of(AutogradContext* ctx) {
  int64_t mask = 0;
  for (int i = 0; i < 3; ++i)  // query, key, value
    if (ctx->needs_input_grad(i)) mask |= int64_t{1} << i;
  return mask;
}

// The requested gradients in front of `others` empty ones.  They are differentiable once: with a
// graph being made they lead to an error instead of nowhere.
variable_list gradient_list(const Triple& gradients, int64_t mask, int others) {
  variable_list list = {std::get<0>(gradients), std::get<1>(gradients), std::get<2>(gradients)};
  for (int i = 0; i < 3; ++i)
    if ((mask >> i & 1) == 0) list[i] = Tensor();
  if (at::GradMode::is_enabled()) {
    for (Tensor& gradient : list) {
      if (!gradient.defined()) continue;
      gradient.set_requires_grad(true);
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a mixer, whose gradients are differentiable once", 1);
      gradient = (*error)({gradient})[0];
    }
  }
  list.resize(3 + others);
  return list;
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& query, const Tensor& key,
                        const Tensor& value, const OptionalTensor& cu_seqlens,
                        const Tensor& log_decay, Scale scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({query, key, value, cu_seqlens.value_or(Tensor()), log_decay});
    if (scale) ctx->saved_data["scale"] = *scale;
    return call_decay(query, key, value, cu_seqlens, log_decay, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const OptionalTensor cu_seqlens = saved[3].defined() ? OptionalTensor(saved[3]) : std::nullopt;
    const Scale scale = ctx->saved_data.count("scale")
                            ? Scale(ctx->saved_data["scale"].toDouble()) : std::nullopt;
    const int64_t mask = gradient_mask_of(ctx);
    Triple gradients;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      gradients = call_decay_vjp(saved[0], saved[1], saved[2], cu_seqlens, saved[4], grads[0],
                                 scale, mask);
    }
    return gradient_list(gradients, mask, 3);
  }
};

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& query, const Tensor& key,
                               const Tensor& value, const OptionalTensor& cu_seqlens,
                               int64_t window, int64_t sinks, Scale scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, log_sum] =
        call_window(query, key, value, cu_seqlens, window, sinks, scale, true);
    ctx->save_for_backward({query, key, value, cu_seqlens.value_or(Tensor()), output, log_sum});
    ctx->mark_non_differentiable({log_sum});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    if (scale) ctx->saved_data["scale"] = *scale;
    return {output, log_sum};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const OptionalTensor cu_seqlens = saved[3].defined() ? OptionalTensor(saved[3]) : std::nullopt;
    const Scale scale = ctx->saved_data.count("scale")
                            ? Scale(ctx->saved_data["scale"].toDouble()) : std::nullopt;
    const int64_t mask = gradient_mask_of(ctx);
    Triple gradients;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      gradients = call_window_vjp(saved[0], saved[1], saved[2], cu_seqlens, saved[4], saved[5],
                                  grads[0], ctx->saved_data["window"].toInt(),
                                  ctx->saved_data["sinks"].toInt(), scale, mask);
    }
    return gradient_list(gradients, mask, 4);
  }
};

template <typename... Tensors>
bool needs_backward(const Tensors&... tensors) {
  return at::GradMode::is_enabled() && (tensors.requires_grad() || ...);
}

// There is no forward-mode derivative: a tangent is refused, not dropped.
bool has_tangent(const Tensor& tensor) { return tensor._fw_grad(/*level=*/0).defined(); }
template <typename... Tensors>
void refuse_tangents(const Tensors&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !(c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(tensors) || ...)),
      "the mixers have no forward-mode derivative: their inputs must not be dual tensors");
}

Tensor decay_attention_autograd(const Tensor& query, const Tensor& key, const Tensor& value,
                                const OptionalTensor& cu_seqlens, const Tensor& log_decay,
                                Scale scale) {
  refuse_tangents(query, key, value, log_decay);
  REQUIRE(!needs_backward(log_decay),
          "log_decay is a constant of each head and takes no gradient: detach it");
  if (!needs_backward(query, key, value)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_decay(query, key, value, cu_seqlens, log_decay, scale);
  }
  refuse_capture("decay_attention", query);
  return DecayAttention::apply(query, key, value, cu_seqlens, log_decay, scale);
}

std::tuple<Tensor, Tensor> window_attention_autograd(const Tensor& query, const Tensor& key,
                                                     const Tensor& value,
                                                     const OptionalTensor& cu_seqlens,
                                                     int64_t window, int64_t sinks, Scale scale,
                                                     bool want_log_sum) {
  refuse_tangents(query, key, value);
  if (!needs_backward(query, key, value)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_window(query, key, value, cu_seqlens, window, sinks, scale, want_log_sum);
  }
  refuse_capture("window_attention", query);
  const auto results =
      WindowAttention::apply(query, key, value, cu_seqlens, window, sinks, scale);
  return {results[0], results[1]};
}

// A tensor that an operator changes (taken by value) has a new version for whoever saved it.
template <typename Declared>
void note_change(const std::decay_t<Declared>& argument) {
  if constexpr (std::is_same_v<Declared, Tensor>)
    if (!argument.is_inference()) torch::autograd::impl::bump_version(argument);
}

// Operators without a backward: whatever asks for one is refused, not cut off in silence.
template <auto* kOperator, typename... Arguments>
auto without_backward(Arguments... arguments) {
  const auto look_at = [](const auto& argument) {
    if constexpr (std::is_same_v<std::decay_t<decltype(argument)>, Tensor>) refuse_tangents(argument);
  };
  (look_at(arguments), ...);
  const auto asks = [](const auto& argument) {
    if constexpr (std::is_same_v<std::decay_t<decltype(argument)>, Tensor>)
      return argument.requires_grad();
    else
      return false;
  };
  TORCH_CHECK(!(at::GradMode::is_enabled() && (asks(arguments) || ...)),
              "an update and the gradients of a mixer have no backward: call them under "
              "torch.no_grad()");
  const auto result = [&] {
    at::AutoDispatchBelowADInplaceOrView below;
    return (*kOperator)(arguments...);
  }();
  (note_change<Arguments>(arguments), ...);
  return result;
}

Tensor call_decay_update(const Tensor& q, const Tensor& k, const Tensor& v,
                         const OptionalTensor& cu, const Tensor& log_decay, Tensor state,
                         Scale scale) {
  static const auto handle =
      operator_handle<decltype(decay_attention_update_op)>("rosa_soft::decay_attention_update");
  return handle.call(q, k, v, cu, log_decay, state, scale);
}
Tensor call_decay_update_out(const Tensor& q, const Tensor& k, const Tensor& v,
                             const OptionalTensor& cu, const Tensor& log_decay,
                             const Tensor& state, Tensor state_out, Scale scale) {
  static const auto handle = operator_handle<decltype(decay_attention_update_out_op)>(
      "rosa_soft::decay_attention_update_out");
  return handle.call(q, k, v, cu, log_decay, state, state_out, scale);
}
Tensor call_window_update(const Tensor& q, const Tensor& k, const Tensor& v, Tensor key_cache,
                          Tensor value_cache, const Tensor& lengths, const OptionalTensor& cu,
                          int64_t window, int64_t sinks, Scale scale) {
  static const auto handle =
      operator_handle<decltype(window_attention_update_op)>("rosa_soft::window_attention_update");
  return handle.call(q, k, v, key_cache, value_cache, lengths, cu, window, sinks, scale);
}

template <auto* kOperator, typename Result, typename... Arguments>
Result refuse_backward(Arguments... arguments) {
  return without_backward<kOperator, Arguments...>(std::forward<Arguments>(arguments)...);
}
template <auto* kOperator, typename Result, typename... Arguments>
constexpr auto refusing(Result (*)(Arguments...)) {
  return &refuse_backward<kOperator, Result, Arguments...>;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rosa_soft, m) {
  m.def(
      "decay_attention(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, float? scale=None) -> Tensor output");
  m.def(
      "decay_attention_vjp(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor grad_output, float? scale, int gradient_mask) -> "
      "(Tensor grad_query, Tensor grad_key, Tensor grad_value)");
  m.def(
      "decay_attention_update(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor(a!) state, float? scale=None) -> Tensor output");
  m.def(
      "decay_attention_update_out(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor log_decay, Tensor state, Tensor(a!) state_out, float? scale=None) -> Tensor output");
  m.def(
      "window_attention(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, int window, "
      "int sinks, float? scale=None, bool want_log_sum=False) -> (Tensor output, Tensor log_sum)");
  m.def(
      "window_attention_vjp(Tensor query, Tensor key, Tensor value, Tensor? cu_seqlens, "
      "Tensor output, Tensor log_sum, Tensor grad_output, int window, int sinks, float? scale, "
      "int gradient_mask) -> (Tensor grad_query, Tensor grad_key, Tensor grad_value)");
  m.def(
      "window_attention_update(Tensor query, Tensor key, Tensor value, Tensor(a!) key_cache, "
      "Tensor(b!) value_cache, Tensor lengths, Tensor? cu_seqlens, int window, int sinks, "
      "float? scale=None) -> Tensor output");
}

#define ROSA_MIXER_OPERATORS(m)                                           \
  m.impl("decay_attention", &decay_attention_op);                         \
  m.impl("decay_attention_vjp", &decay_attention_vjp_op);                 \
  m.impl("decay_attention_update", &decay_attention_update_op);           \
  m.impl("decay_attention_update_out", &decay_attention_update_out_op);   \
  m.impl("window_attention", &window_attention_op);                       \
  m.impl("window_attention_vjp", &window_attention_vjp_op);               \
  m.impl("window_attention_update", &window_attention_update_op);

TORCH_LIBRARY_IMPL(rosa_soft, CUDA, m) { ROSA_MIXER_OPERATORS(m) }

// host tensors meet the same checks, the last of which refuses them
TORCH_LIBRARY_IMPL(rosa_soft, CPU, m) { ROSA_MIXER_OPERATORS(m) }

TORCH_LIBRARY_IMPL(rosa_soft, Autograd, m) {
  m.impl("decay_attention", &decay_attention_autograd);
  m.impl("window_attention", &window_attention_autograd);
  m.impl("decay_attention_vjp", refusing<&call_decay_vjp>(&call_decay_vjp));
  m.impl("window_attention_vjp", refusing<&call_window_vjp>(&call_window_vjp));
  m.impl("decay_attention_update", refusing<&call_decay_update>(&call_decay_update));
  m.impl("decay_attention_update_out", refusing<&call_decay_update_out>(&call_decay_update_out));
  m.impl("window_attention_update", refusing<&call_window_update>(&call_window_update));
}
