// Bindings of the mixture-of-experts operators.  A call refuses whatever vericcl_b200/ops/experts.py documents as
// refused before it launches anything; that file then says which argument was wrong.  Small calls cost what their
// host side costs, so results are allocated and cut without going through the dispatcher.
#include <cuda_runtime.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>
#include <stdexcept>
#include <string>

#include "vb/launch.h"

namespace py = pybind11;
using namespace vb;
using torch::Tensor;

namespace {

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DT_F32;
    case at::kBFloat16: return DT_BF16;
    case at::kHalf: return DT_F16;
    default: TORCH_CHECK(false, "unsupported tensor dtype (float32, bfloat16, float16)");
  }
}

void done(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  cudaGetLastError();            // reported here, not again by the next call that looks
  throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

constexpr int64_t kMaxColumns = 1 << 22;

// the kernels carry no forward-mode tangents, and a result without them would read as one that does not change
void check_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK(!t._fw_grad(0).defined(), name, " carries a forward-mode gradient");
}

// a CUDA matrix on `like`'s device whose rows are contiguous
void check_matrix(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " is not on the call's GPU");
  TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && t.size(1) <= kMaxColumns, name,
              " is no matrix of contiguous rows");
  check_tangent(t, name);
}

void check_table(const Tensor& t, const Tensor& like, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.scalar_type() == type, name,
              " is not a contiguous table of its type on the call's GPU");
  check_tangent(t, name);
}

// A matrix in memory, in bytes; a contiguous tensor of other dimensions is one row.
struct Extent {
  int64_t lo, width, pitch, rows;
};
Extent extent(const Tensor& t) {
  const int64_t lo = (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr()), size = t.element_size();
  if (!t.numel()) return {lo, 0, 0, 0};
  if (t.dim() != 2) return {lo, t.numel() * size, 0, 1};
  return {lo, t.size(1) * size, t.stride(0) * size, t.size(0)};
}

// Column ranges of one matrix lie in one span of memory without meeting: with one pitch, what counts is the distance
// of the first columns within it.  Different pitches are compared by their spans.
bool apart(const Extent& a, const Extent& b) {
  if (!a.rows || !b.rows) return true;
  if (a.lo + (a.rows - 1) * a.pitch + a.width <= b.lo || b.lo + (b.rows - 1) * b.pitch + b.width <= a.lo) return true;
  const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
  if ((b.rows > 1 && b.pitch != pitch) || (a.rows == 1 && b.rows == 1) || pitch < a.width || pitch < b.width) return false;
  const int64_t between = ((b.lo - a.lo) % pitch + pitch) % pitch;
  return between >= a.width && between + b.width <= pitch;
}

void check_apart(const Tensor& out, const Tensor& in) {
  TORCH_CHECK(apart(extent(out), extent(in)), "out overlaps an input");
}
void check_apart(const Tensor& out, const std::optional<Tensor>& in) {
  if (in) check_apart(out, *in);
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// a contiguous tensor of `type` (4 bytes an element) inside the int32 tensor `pool`, from element `offset` on
Tensor cut(const Tensor& pool, int64_t offset, at::IntArrayRef sizes, at::ScalarType type = at::kInt) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(pool.storage()), pool.key_set(),
                                                    at::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  return t;
}

void check_order(const Tensor& slot, const Tensor& source, const Tensor& like) {
  check_table(slot, like, at::kInt, "slot");
  check_table(source, like, at::kInt, "source");
  TORCH_CHECK(slot.dim() == 2 && source.dim() == 1 && slot.size(1) >= 1 && slot.size(1) <= kMaxChoices,
              "slot is [tokens, k], source [rows]");
  TORCH_CHECK(slot.numel() <= INT_MAX && source.numel() <= INT_MAX, "more than 2^31 - 1 assignments or rows");
}

ExchangeRowsArgs row_args(const Tensor& in, const Tensor& out, const Tensor& slot, const Tensor& source) {
  ExchangeRowsArgs a{};
  a.in = in.data_ptr();
  a.out = out.data_ptr();
  a.in_stride = in.stride(0);
  a.out_stride = out.stride(0);
  a.slot = slot.data_ptr<int>();
  a.source = source.data_ptr<int>();
  a.tokens = slot.size(0);
  a.rows = source.numel();
  a.hidden = in.size(1);
  a.k = (int)slot.size(1);
  a.dtype = code_of(in);
  return a;
}

// The result [rows, columns] of `like`'s dtype: a new tensor, or `out` if it is one of that kind, away from `like` and
// the other inputs.  A write into `out` counts as an in-place change, so that a graph that has saved it sees it (tensors of inference
// mode have no versions, and no graph can have saved them).
template <typename... Inputs>
Tensor made(const std::optional<Tensor>& out, int64_t rows, int64_t columns, const Tensor& like, const Inputs&... inputs) {
  if (!out) return empty({rows, columns}, like.scalar_type(), like);
  check_matrix(*out, like, "out");
  TORCH_CHECK(out->size(0) == rows && out->size(1) == columns && out->scalar_type() == like.scalar_type(),
              "out has another shape or dtype than the result");
  TORCH_CHECK(rows <= 1 || out->stride(0) >= columns, "out's rows overlap");
  check_apart(*out, like);
  (check_apart(*out, inputs), ...);
  TORCH_CHECK(!(out->requires_grad() && at::GradMode::is_enabled()), "out requires a gradient");
  if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
  return *out;
}

py::tuple route(const Tensor& logits, int64_t k, bool renormalize) {
  check_matrix(logits, logits, "logits");
  TORCH_CHECK(k >= 1 && k <= kMaxChoices && k <= logits.size(1) && logits.size(1) <= kMaxExperts &&
              logits.size(0) * k <= INT_MAX, "bad k, experts or tokens");
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t n = logits.size(0) * k, sizes[2] = {logits.size(0), k};
  auto pool = empty({2 * n}, at::kInt, logits);
  auto ids = cut(pool, 0, sizes), weights = cut(pool, n, sizes, at::kFloat);
  RouteArgs a{};
  a.logits = logits.data_ptr();
  a.logits_stride = logits.stride(0);
  a.tokens = logits.size(0);
  a.dtype = code_of(logits);
  a.experts = (int)logits.size(1);
  a.k = (int)k;
  a.renormalize = renormalize ? 1 : 0;
  a.ids = ids.data_ptr<int>();
  a.weights = weights.data_ptr<float>();
  done(launch_route(a, stream()), "route launch");
  return py::make_tuple(ids, weights);
}

Tensor route_backward(const Tensor& logits, const Tensor& ids, const Tensor& weights, const Tensor& grad,
                      bool renormalize) {
  check_matrix(logits, logits, "logits");
  check_table(ids, logits, at::kInt, "ids");
  check_table(weights, logits, at::kFloat, "weights");
  check_table(grad, logits, at::kFloat, "grad_weights");
  TORCH_CHECK(ids.dim() == 2 && ids.size(0) == logits.size(0) && ids.size(1) >= 1 && ids.size(1) <= kMaxChoices &&
              ids.size(1) <= logits.size(1) && ids.numel() <= INT_MAX && weights.sizes() == ids.sizes() && grad.sizes() == ids.sizes() && logits.size(1) <= kMaxExperts,
              "ids, weights and grad_weights are [tokens, k]");
  c10::cuda::CUDAGuard guard(logits.device());
  auto out = empty({logits.size(0), logits.size(1)}, logits.scalar_type(), logits);
  RouteArgs a{};
  a.logits = logits.data_ptr();
  a.logits_stride = logits.stride(0);
  a.tokens = logits.size(0);
  a.dtype = code_of(logits);
  a.experts = (int)logits.size(1);
  a.k = (int)ids.size(1);
  a.renormalize = renormalize ? 1 : 0;
  a.ids = ids.data_ptr<int>();
  a.weights = weights.data_ptr<float>();
  a.grad_weights = grad.data_ptr<float>();
  a.grad_logits = out.data_ptr();
  done(launch_route_backward(a, stream()), "route backward launch");
  return out;
}

py::tuple sort_by_expert(const Tensor& ids, int64_t experts, int64_t capacity) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.dim() == 2 &&
              (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong), "ids are contiguous int32 or int64");
  TORCH_CHECK(experts >= 1 && experts <= kMaxExperts && capacity >= 0 && capacity <= INT_MAX && ids.size(1) >= 1 &&
              ids.size(1) <= kMaxChoices, "bad experts, capacity or choices");
  const int64_t rows = capacity ? experts * capacity : ids.numel();
  TORCH_CHECK(ids.numel() <= INT_MAX && rows <= INT_MAX, "more than 2^31 - 1 assignments or rows");
  c10::cuda::CUDAGuard guard(ids.device());
  // one allocation for the four tables
  const int64_t n = ids.numel();
  auto pool = empty({n + rows + 2 * experts}, at::kInt, ids);
  auto slot = cut(pool, 0, ids.sizes()), source = cut(pool, n, {rows});
  auto counts = cut(pool, n + rows, {experts}), starts = cut(pool, n + rows + experts, {experts});
  SortArgs a{};
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == at::kLong ? 1 : 0;
  a.assignments = ids.numel();
  a.rows = rows;
  a.experts = (int)experts;
  a.capacity = capacity;
  a.slot = slot.data_ptr<int>();
  a.source = source.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.starts = starts.data_ptr<int>();
  done(launch_sort(a, stream()), "expert sort launch");
  return py::make_tuple(slot, source, counts, starts);
}

Tensor dispatch(const Tensor& x, const Tensor& slot, const Tensor& source, const std::optional<Tensor>& out) {
  check_matrix(x, x, "x");
  check_order(slot, source, x);
  TORCH_CHECK(x.size(0) == slot.size(0), "x has another number of tokens than the order");
  c10::cuda::CUDAGuard guard(x.device());
  auto rows = made(out, source.numel(), x.size(1), x, slot, source);
  done(launch_dispatch(row_args(x, rows, slot, source), stream()), "dispatch launch");
  return rows;
}

Tensor combine(const Tensor& rows, const std::optional<Tensor>& weights, const Tensor& slot, const Tensor& source,
               const std::optional<Tensor>& out) {
  check_matrix(rows, rows, "rows");
  check_order(slot, source, rows);
  TORCH_CHECK(rows.size(0) == source.numel(), "rows has another number of rows than the order");
  if (weights) {
    check_table(*weights, rows, at::kFloat, "weights");
    TORCH_CHECK(weights->sizes() == slot.sizes(), "weights are [tokens, k]");
  }
  c10::cuda::CUDAGuard guard(rows.device());
  auto tokens = made(out, slot.size(0), rows.size(1), rows, slot, source, weights);
  auto a = row_args(rows, tokens, slot, source);
  if (weights) a.weights = weights->data_ptr<float>();
  done(launch_combine(a, stream()), "combine launch");
  return tokens;
}

py::tuple combine_backward(const Tensor& grad, const Tensor& rows, const Tensor& weights, const Tensor& slot,
                           const Tensor& source, const std::optional<Tensor>& out) {
  check_matrix(grad, grad, "grad_out");
  check_matrix(rows, grad, "rows");
  check_order(slot, source, grad);
  check_table(weights, grad, at::kFloat, "weights");
  TORCH_CHECK(grad.size(0) == slot.size(0) && rows.size(0) == source.numel() && rows.size(1) == grad.size(1) &&
              rows.scalar_type() == grad.scalar_type() && weights.sizes() == slot.sizes(),
              "grad_out, rows, weights and the order do not fit together");
  c10::cuda::CUDAGuard guard(grad.device());
  auto grad_rows = made(out, source.numel(), grad.size(1), grad, rows, weights, slot, source);
  auto grad_weights = empty(slot.sizes(), at::kFloat, grad);
  auto a = row_args(grad, grad_rows, slot, source);
  a.saved = rows.data_ptr();
  a.saved_stride = rows.stride(0);
  a.weights = weights.data_ptr<float>();
  a.grad_weights = grad_weights.data_ptr<float>();
  done(launch_combine_backward(a, stream()), "combine backward launch");
  return py::make_tuple(grad_rows, grad_weights);
}

Tensor int4_product(const Tensor& x, const Tensor& starts, const Tensor& counts, const Tensor& packed,
                    const Tensor& scales, const std::optional<Tensor>& out, bool give_up) {
  check_matrix(x, x, "rows");
  check_table(starts, x, at::kInt, "starts");
  check_table(counts, x, at::kInt, "counts");
  check_table(packed, x, at::kByte, "packed");
  check_table(scales, x, scales.scalar_type(), "scales");
  TORCH_CHECK(packed.dim() == 3 && scales.dim() == 3 && packed.size(0) == scales.size(0) &&
              packed.size(1) == scales.size(1) && packed.size(2) * 2 == x.size(1) && scales.size(2) > 0 &&
              x.size(1) % scales.size(2) == 0, "packed is [experts, n, inner / 2], scales [experts, n, inner / group]");
  const int64_t group = x.size(1) / scales.size(2), segments = starts.numel();
  TORCH_CHECK(group == 32 || group == 64 || group == 128, "groups of 32, 64 or 128");
  TORCH_CHECK(starts.dim() == 1 && counts.numel() == segments && segments >= 1 && packed.size(0) >= 1 &&
              segments % packed.size(0) == 0 && segments <= kMaxExperts, "segments are a multiple of the experts");
  TORCH_CHECK(x.scalar_type() != at::kFloat && (scales.scalar_type() == at::kFloat || scales.scalar_type() == x.scalar_type()),
              "16-bit rows, scales of their type or fp32");
  TORCH_CHECK(x.size(0) <= INT_MAX && packed.size(0) * packed.size(1) <= INT_MAX && x.size(1) <= INT_MAX,
              "more than 2^31 - 1 rows, weight rows or inner values");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(packed.data_ptr()) % 16 == 0, "packed starts on a 16-byte boundary");
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(!(x.requires_grad() && at::GradMode::is_enabled()), "4-bit products have no gradient");
  auto y = made(out, x.size(0), packed.size(1), x, starts, counts, packed, scales);
  Int4Args a{};
  a.x = x.data_ptr();
  a.x_stride = x.stride(0);
  a.rows = x.size(0);
  a.starts = starts.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.segments = (int)segments;
  a.experts = (int)packed.size(0);
  a.packed = packed.data_ptr<uint8_t>();
  a.scales = scales.data_ptr();
  a.scales_fp32 = scales.scalar_type() == at::kFloat ? 1 : 0;
  a.n = packed.size(1);
  a.inner = x.size(1);
  a.group = (int)group;
  a.dtype = code_of(x);
  a.out = y.data_ptr();
  a.out_stride = y.stride(0);
  a.give_up = give_up ? 1 : 0;
  done(launch_int4_product(a, stream()), "4-bit product launch");
  return y;
}

}  // namespace

void bind_experts(py::module_& m) {
  m.attr("max_experts") = kMaxExperts;
  m.attr("max_choices") = kMaxChoices;
  m.def("route", &route);
  m.def("route_backward", &route_backward);
  m.def("sort_by_expert", &sort_by_expert);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("combine_backward", &combine_backward);
  m.def("int4_product", &int4_product);
  m.def("int4_late_copies", []() {
    py::gil_scoped_release release;      // it waits for the GPU
    int flag = 0;
    done(int4_late_copies(&flag), "read the late-copy flag");
    return flag != 0;
  });
}
