// Dispatcher layer of the paged cache (module rosa_soft_amd._C, beside mixer_dispatch.cpp): schemas,
// validation, allocation and stream of the page tables and of attention over pages.  No device code
// lives in this file.

#include "mixer_dispatch.hpp"

namespace {

using namespace rosa_dispatch;
using Scale = std::optional<double>;

constexpr int64_t kMostTableSlots = 8192;
constexpr int64_t kMostCount = 1024;

void check_page(int64_t page) {
  REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0,
          "page must be a power of two in [16, 256]");
}

void check_integers(const Tensor& tensor, const char* name, const Tensor& tables) {
  REQUIRE(tensor.scalar_type() == torch::kInt32, name, " must have dtype int32");
  REQUIRE(tensor.device() == tables.device(), "all tensors must be on the same device");
}

// ---------------------------------------------------------------------------
// tables
// ---------------------------------------------------------------------------

// Tables, lengths and pool; returns the number of slots.
int64_t check_tables(const Tensor& tables, const Tensor& lengths, const Tensor& pool, int64_t page) {
  REQUIRE(tables.dim() == 2 && tables.size(0) >= 1 && tables.size(1) >= 1,
          "tables must have shape (slots, columns)");
  const int64_t slots = tables.size(0);
  check_integers(tables, "tables", tables);
  check_integers(lengths, "lengths", tables);
  check_integers(pool, "pool", tables);
  REQUIRE(slots <= kMostTableSlots, "tables must have at most 8192 slots");
  REQUIRE(tables.numel() <= kIntMax, "tables must have fewer than 2^31 entries");
  REQUIRE(lengths.dim() == 1 && lengths.size(0) == slots, "lengths must have one entry per slot");
  REQUIRE(pool.dim() == 1 && pool.size(0) >= 2 && pool.size(0) - 1 <= kIntMax,
          "pool must have shape (pages + 1,)");
  REQUIRE(tables.is_contiguous() && pool.is_contiguous(), "tables and pool must be contiguous");
  REQUIRE(!overlap(tables, pool) && !overlap(tables, lengths) && !overlap(pool, lengths),
          "tables, pool, and lengths must share no memory");
  check_page(page);
  return slots;
}

rosa_page_tables describe_tables(const Tensor& tables, const Tensor& lengths, const Tensor& pool,
                                 int64_t page) {
  return {tables.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), pool.data_ptr<int32_t>(),
          static_cast<int>(tables.size(0)), static_cast<int>(tables.size(1)),
          static_cast<int>(pool.size(0) - 1), static_cast<int>(page)};
}

Tensor page_tables_update_op(Tensor tables, const Tensor& lengths, Tensor pool,
                             const OptionalTensor& cu_seqlens, int64_t tokens, int64_t page) {
  const int64_t slots = check_tables(tables, lengths, pool, page);
  REQUIRE(tokens >= 0, "tokens must be >= 0");
  REQUIRE(tokens <= kMostTokens && (cu_seqlens || tokens <= kIntMax / slots),
          "tokens of all slots must fit in int32");
  if (cu_seqlens) {
    check_integers(*cu_seqlens, "cu_seqlens", tables);
    REQUIRE(cu_seqlens->dim() == 1 && cu_seqlens->size(0) == slots + 1,
            "cu_seqlens must have slots + 1 entries");
    REQUIRE(!overlap(tables, *cu_seqlens) && !overlap(pool, *cu_seqlens),
            "tables, pool, and cu_seqlens must share no memory");
  }
  check_device(tables);
  const Guard guard(tables.device());
  const auto options = tables.options().dtype(torch::kInt64);
  const Tensor rows = cu_seqlens ? torch::empty({tokens}, options) : torch::empty({slots, tokens}, options);
  if (tokens == 0) return rows;
  const Tensor seen = lengths.contiguous();
  const Tensor offsets = cu_seqlens ? cu_seqlens->contiguous() : Tensor();
  const rosa_page_tables described = describe_tables(tables, seen, pool, page);
  raise_on_failure(
      rosa_hip_page_tables_update(&described, cu_seqlens ? offsets.data_ptr<int32_t>() : nullptr,
                                  cu_seqlens ? 0 : static_cast<int>(tokens),
                                  static_cast<int>(rows.numel()), rows.data_ptr<int64_t>(),
                                  current_stream()),
      "rosa_hip_page_tables_update");
  return rows;
}

void page_tables_release_op(Tensor tables, const Tensor& lengths, const Tensor& keep, Tensor pool,
                            int64_t page) {
  const int64_t slots = check_tables(tables, lengths, pool, page);
  check_integers(keep, "keep", tables);
  REQUIRE(keep.dim() == 1 && keep.size(0) == slots, "keep must have one entry per slot");
  REQUIRE(!overlap(tables, keep) && !overlap(pool, keep), "tables, pool, and keep must share no memory");
  check_device(tables);
  const Guard guard(tables.device());
  const Tensor seen = lengths.contiguous(), kept = keep.contiguous();
  const rosa_page_tables described = describe_tables(tables, seen, pool, page);
  raise_on_failure(
      rosa_hip_page_tables_release(&described, kept.data_ptr<int32_t>(), current_stream()),
      "rosa_hip_page_tables_release");
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

Tensor paged_update(const Tensor& query, const Tensor& key, const Tensor& value,
                    const Tensor& key_pages, const Tensor& value_pages, const Tensor* key_bounds,
                    const Tensor& tables, const Tensor& rows, const Tensor& lengths,
                    const OptionalTensor& cu_seqlens, int64_t count, Scale scale) {
  const double factor = check_call(query, key, value, cu_seqlens, scale, true);
  const int64_t slots = check_slots(query, cu_seqlens);
  REQUIRE(key_pages.dim() == 4 && value_pages.dim() == 4,
          "pages must have shape (pages, key heads, page, width)");
  const int64_t pages = key_pages.size(0), page = key_pages.size(2), heads = key.size(-2);
  REQUIRE(key_pages.sizes() == torch::IntArrayRef({pages, heads, page, key.size(-1)}) &&
              value_pages.sizes() == torch::IntArrayRef({pages, heads, page, value.size(-1)}),
          "pages must have shape (pages, key heads, page, width)");
  check_page(page);
  REQUIRE(pages >= 1 && pages <= kIntMax, "there must be 1 to 2^31 - 1 pages");
  if (key_bounds != nullptr)
    REQUIRE(key_bounds->sizes() == torch::IntArrayRef({pages, heads, 2, key.size(-1)}),
            "key_bounds must have shape (pages, key heads, 2, key width)");
  REQUIRE(tables.dim() == 2 && tables.size(0) == slots && tables.size(1) >= 1 &&
              tables.size(1) <= kIntMax && tables.scalar_type() == torch::kInt32,
          "tables must be an int32 tensor of shape (slots, columns)");
  REQUIRE(tables.is_contiguous(), "tables must be contiguous");
  REQUIRE(rows.scalar_type() == torch::kInt64 &&
              rows.sizes() == query.sizes().slice(0, query.dim() - 2),
          "rows must be an int64 tensor with one entry per new token");
  REQUIRE(lengths.dim() == 1 && lengths.size(0) == slots && lengths.scalar_type() == torch::kInt32,
          "lengths must be an int32 tensor with one entry per slot");
  for (const Tensor* tensor : {&tables, &rows, &lengths})
    REQUIRE(tensor->device() == query.device(),
            "all inputs, tables, rows, and lengths must be on the same device");
  for (const Tensor* cache : {&key_pages, &value_pages, key_bounds}) {
    if (cache == nullptr) continue;
    REQUIRE(cache->scalar_type() == query.scalar_type(), "pages must have the dtype of the inputs");
    REQUIRE(cache->device() == query.device(), "all inputs and pages must be on the same device");
    REQUIRE(cache->is_contiguous(), "pages must be contiguous");
    for (const Tensor* input : {&query, &key, &value, &tables, &rows, &lengths})
      REQUIRE(!overlap(*cache, *input), "pages must share no memory with the inputs");
    REQUIRE(!cu_seqlens || !overlap(*cache, *cu_seqlens), "pages must share no memory with the inputs");
  }
  REQUIRE(!overlap(key_pages, value_pages) &&
              (key_bounds == nullptr ||
               (!overlap(key_pages, *key_bounds) && !overlap(value_pages, *key_bounds))),
          "pages and bounds must share no memory");
  check_device(query);
  const Guard guard(query.device());
  const Call call = make_call(query, key, value, cu_seqlens, factor);
  const Tensor output = new_output(call);
  if (query.numel() == 0) return output;  // nobody brings a token
  const Tensor seen = lengths.contiguous(), places = rows.contiguous();
  const rosa_paged_cache cache = {key_pages.data_ptr(),
                                  value_pages.data_ptr(),
                                  key_bounds == nullptr ? nullptr : key_bounds->data_ptr(),
                                  tables.data_ptr<int32_t>(),
                                  seen.data_ptr<int32_t>(),
                                  places.data_ptr<int64_t>(),
                                  static_cast<int>(tables.size(1)),
                                  static_cast<int>(pages),
                                  static_cast<int>(page)};
  const size_t bytes = rosa_hip_paged_workspace_bytes(&call.problem, &cache, static_cast<int>(count));
  const Tensor workspace = new_workspace(bytes, query);
  raise_on_failure(rosa_hip_paged_update(&call.problem, &cache, static_cast<int>(count), &call.q,
                                         &call.k, &call.v, output.data_ptr(), workspace.data_ptr(),
                                         bytes, current_stream()),
                   "rosa_hip_paged_update");
  return output;
}

// (tensors that an operator changes are taken by value)
Tensor paged_attention_update_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                 Tensor key_pages, Tensor value_pages, const Tensor& tables,
                                 const Tensor& rows, const Tensor& lengths,
                                 const OptionalTensor& cu_seqlens, Scale scale) {
  return paged_update(query, key, value, key_pages, value_pages, nullptr, tables, rows, lengths,
                      cu_seqlens, 0, scale);
}

Tensor paged_attention_update_bounds_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                        Tensor key_pages, Tensor value_pages, Tensor key_bounds,
                                        const Tensor& tables, const Tensor& rows,
                                        const Tensor& lengths, const OptionalTensor& cu_seqlens,
                                        Scale scale) {
  return paged_update(query, key, value, key_pages, value_pages, &key_bounds, tables, rows, lengths,
                      cu_seqlens, 0, scale);
}

Tensor selected_attention_update_op(const Tensor& query, const Tensor& key, const Tensor& value,
                                    Tensor key_pages, Tensor value_pages, Tensor key_bounds,
                                    const Tensor& tables, const Tensor& rows, const Tensor& lengths,
                                    const OptionalTensor& cu_seqlens, int64_t count, Scale scale) {
  REQUIRE(count >= 1 && count <= kMostCount, "count must be in [1, 1024]");
  return paged_update(query, key, value, key_pages, value_pages, &key_bounds, tables, rows, lengths,
                      cu_seqlens, count, scale);
}

// the operators as the dispatcher has them, so that tracing sees them
template <auto* kOperator>
struct Traced;
#define ROSA_TRACED(op)                                                                    \
  template <>                                                                              \
  struct Traced<&op##_op> {                                                                \
    template <typename... Arguments>                                                       \
    static auto call(Arguments... arguments) {                                             \
      static const auto handle = operator_handle<decltype(op##_op)>("rosa_soft::" #op);    \
      return handle.call(std::forward<Arguments>(arguments)...);                           \
    }                                                                                      \
  };
ROSA_TRACED(page_tables_update)
ROSA_TRACED(page_tables_release)
ROSA_TRACED(paged_attention_update)
ROSA_TRACED(paged_attention_update_bounds)
ROSA_TRACED(selected_attention_update)

template <auto* kOperator, typename Signature>
struct Dispatched;
template <auto* kOperator, typename Result, typename... Arguments>
struct Dispatched<kOperator, Result(Arguments...)> {
  static Result call(Arguments... arguments) {
    return Traced<kOperator>::template call<Arguments...>(std::forward<Arguments>(arguments)...);
  }
};

}  // namespace

TORCH_LIBRARY_FRAGMENT(rosa_soft, m) {
  m.def(
      "page_tables_update(Tensor(a!) tables, Tensor lengths, Tensor(b!) pool, Tensor? cu_seqlens, "
      "int tokens, int page) -> Tensor rows");
  m.def(
      "page_tables_release(Tensor(a!) tables, Tensor lengths, Tensor keep, Tensor(b!) pool, "
      "int page) -> ()");
  m.def(
      "paged_attention_update(Tensor query, Tensor key, Tensor value, Tensor(a!) key_pages, "
      "Tensor(b!) value_pages, Tensor tables, Tensor rows, Tensor lengths, Tensor? cu_seqlens, "
      "float? scale=None) -> Tensor output");
  m.def(
      "paged_attention_update_bounds(Tensor query, Tensor key, Tensor value, Tensor(a!) key_pages, "
      "Tensor(b!) value_pages, Tensor(c!) key_bounds, Tensor tables, Tensor rows, Tensor lengths, "
      "Tensor? cu_seqlens, float? scale=None) -> Tensor output");
  m.def(
      "selected_attention_update(Tensor query, Tensor key, Tensor value, Tensor(a!) key_pages, "
      "Tensor(b!) value_pages, Tensor(c!) key_bounds, Tensor tables, Tensor rows, Tensor lengths, "
      "Tensor? cu_seqlens, int count, float? scale=None) -> Tensor output");
}

#define ROSA_PAGED_OPERATORS(m)                                                   \
  m.impl("page_tables_update", &page_tables_update_op);                           \
  m.impl("page_tables_release", &page_tables_release_op);                         \
  m.impl("paged_attention_update", &paged_attention_update_op);                   \
  m.impl("paged_attention_update_bounds", &paged_attention_update_bounds_op);     \
  m.impl("selected_attention_update", &selected_attention_update_op);

TORCH_LIBRARY_IMPL(rosa_soft, CUDA, m) { ROSA_PAGED_OPERATORS(m) }

// host tensors meet the same checks, the last of which refuses them
TORCH_LIBRARY_IMPL(rosa_soft, CPU, m) { ROSA_PAGED_OPERATORS(m) }

#define ROSA_REFUSING(m, op)                                          \
  m.impl(#op, refusing<&Dispatched<&op##_op, decltype(op##_op)>::call>( \
                  &Dispatched<&op##_op, decltype(op##_op)>::call));

TORCH_LIBRARY_IMPL(rosa_soft, Autograd, m) {
  ROSA_REFUSING(m, page_tables_update)
  ROSA_REFUSING(m, page_tables_release)
  ROSA_REFUSING(m, paged_attention_update)
  ROSA_REFUSING(m, paged_attention_update_bounds)
  ROSA_REFUSING(m, selected_attention_update)
}
