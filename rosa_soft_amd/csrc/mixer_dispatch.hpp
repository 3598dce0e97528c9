// What the dispatcher layers of the mixers and of the paged cache share: checks of a call's tensors,
// their description for the C entry points, and the refusal of derivatives that do not exist.  Inputs
// are taken with their strides as long as the elements of a head are neighbours; outputs are
// contiguous and of the inputs' dtype.
#pragma once

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

namespace rosa_dispatch {

using torch::Tensor;
using OptionalTensor = std::optional<Tensor>;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

constexpr int64_t kIntMax = std::numeric_limits<int>::max();
constexpr int64_t kMostTokens = kIntMax - 1024;  // of a sequence, or of a packed call
constexpr int64_t kMostWidth = 128;

inline int dtype_code(c10::ScalarType dtype) {
  switch (dtype) {
    case torch::kFloat32: return ROSA_DTYPE_F32;
    case torch::kFloat16: return ROSA_DTYPE_F16;
    case torch::kBFloat16: return ROSA_DTYPE_BF16;
    default: return -1;
  }
}

inline void* current_stream() {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

inline void raise_on_failure(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed (", status, "): ", rosa_hip_last_error());
}

// elements of a head next to each other; everything else by strides
inline Tensor readable(const Tensor& tensor) {
  return tensor.size(-1) == 1 || tensor.stride(-1) == 1 ? tensor : tensor.contiguous();
}

inline rosa_mixer_tensor describe(const Tensor& tensor) {
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
inline double check_call(const Tensor& query, const Tensor& key, const Tensor& value,
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
inline bool overlap(const Tensor& a, const Tensor& b) {
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
inline void check_device(const Tensor& query) { REQUIRE(query.is_cuda(), "the mixers require CUDA tensors"); }

inline Call make_call(const Tensor& query, const Tensor& key, const Tensor& value,
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

inline Tensor new_output(const Call& call) {
  auto sizes = call.query.sizes().vec();
  sizes.back() = call.value.size(-1);
  return torch::empty(sizes, call.query.options());
}

inline Tensor new_workspace(size_t bytes, const Tensor& like) {
  TORCH_CHECK(bytes > 0, "mixer workspace: ", rosa_hip_last_error());
  return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

inline int64_t check_slots(const Tensor& query, const OptionalTensor& cu_seqlens) {
  const int64_t slots = cu_seqlens ? cu_seqlens->numel() - 1 : query.size(0);
  REQUIRE(slots >= 1, "an update needs at least one slot");
  return slots;
}

// the operators as the dispatcher has them, so that tracing sees them
template <typename Signature>
auto operator_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<Signature>();
}
// There is no forward-mode derivative: a tangent is refused, not dropped.
inline bool has_tangent(const Tensor& tensor) { return tensor._fw_grad(/*level=*/0).defined(); }
template <typename... Tensors>
inline void refuse_tangents(const Tensors&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !(c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(tensors) || ...)),
      "the mixers have no forward-mode derivative: their inputs must not be dual tensors");
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
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView below;
    return (*kOperator)(arguments...);
  };
  if constexpr (std::is_void_v<decltype(call())>) {
    call();
    (note_change<Arguments>(arguments), ...);
  } else {
    const auto result = call();
    (note_change<Arguments>(arguments), ...);
    return result;
  }
}

template <auto* kOperator, typename Result, typename... Arguments>
Result refuse_backward(Arguments... arguments) {
  return without_backward<kOperator, Arguments...>(std::forward<Arguments>(arguments)...);
}
template <auto* kOperator, typename Result, typename... Arguments>
constexpr auto refusing(Result (*)(Arguments...)) {
  return &refuse_backward<kOperator, Result, Arguments...>;
}

}  // namespace rosa_dispatch
