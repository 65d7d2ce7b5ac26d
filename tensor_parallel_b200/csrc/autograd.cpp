// Autograd nodes of the layers whose training calls are bound by the host at ordinary sizes: linear and norms.  And, without nodes, the calls of
// 8-bit serving and of ragged batches, whose kernels take a few microseconds each at decode sizes.
//
// A small call (100 tokens through a 768 x 3072 projection with bias, forward and backward) keeps the GPU busy for 37 us.  As Python
// autograd functions over ctypes it took 176 us: each of its launches cost 10 to 20 us of interpreter work, and the backward nodes
// ran under the interpreter lock on the autograd thread.  The same nodes in C++ enqueue the same kernels, with the same shapes,
// copies and saved tensors, without entering the interpreter.
//
// The module has no link to the kernel library: `bind` receives the entry points of the library that ops/native.py loaded
// (a variant with index checks, for instance), and the two callbacks that need Python objects.
#include <torch/extension.h>

#include <ATen/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <stdexcept>
#include <string>

#include "tpb_api.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Library {
  decltype(&tpb_gemm_plan_ex) plan = nullptr;
  decltype(&tpb_gemm_bf16_ex) gemm = nullptr;
  decltype(&tpb_norm_fwd) norm_fwd = nullptr;
  decltype(&tpb_norm_bwd) norm_bwd = nullptr;
  decltype(&tpb_norm_bwd_parts) norm_bwd_parts = nullptr;
  decltype(&tpb_col_sum_parts) col_sum_parts = nullptr;
  decltype(&tpb_col_sum) col_sum = nullptr;
  decltype(&tpb_rows_int8) rows_int8 = nullptr;
  decltype(&tpb_gemm_int8) gemm_int8 = nullptr;
  decltype(&tpb_paged_attention_workspace) paged_attention_workspace = nullptr;
  decltype(&tpb_paged_attention) paged_attention = nullptr;
  decltype(&tpb_paged_append) paged_append = nullptr;
  decltype(&tpb_adjust_logits) adjust_logits = nullptr;
};
Library lib;
PyObject* error_text = nullptr;     // (code, what) -> message
PyObject* reserve_slots = nullptr;  // (device index, fp32 elements) -> address of the device's reduction context
constexpr int MAX_DEVICES = 64;
std::atomic<tpb_reduce_ctx_t*> contexts[MAX_DEVICES];
std::atomic<long long> launched{0};

void check(int code, const char* what) {
  if (code == TPB_OK) return;
  std::string text = std::string(what) + " failed: " + std::to_string(code);
  {
    py::gil_scoped_acquire gil;
    try {
      text = py::reinterpret_borrow<py::function>(error_text)(code, what).cast<std::string>();
    } catch (py::error_already_set& e) {
      e.discard_as_unraisable("error text of a native kernel");
    }
  }
  throw std::runtime_error(text);
}

// The reduction context of a device, with at least `elems` fp32 elements per slot.  It lives as long as the process.
tpb_reduce_ctx_t* context(const Tensor& t, size_t elems) {
  const int device = t.is_cuda() ? t.get_device() : 0;
  TORCH_CHECK(device >= 0 && device < MAX_DEVICES, "device index out of range");
  tpb_reduce_ctx_t* c = contexts[device].load(std::memory_order_acquire);
  if (c && elems <= c->slot_stride) return c;
  std::string problem;
  {
    py::gil_scoped_acquire gil;
    try {
      const auto address = py::reinterpret_borrow<py::function>(reserve_slots)(device, elems).cast<uintptr_t>();
      c = reinterpret_cast<tpb_reduce_ctx_t*>(address);
    } catch (py::error_already_set& e) {
      problem = e.what();
    }
  }
  if (!problem.empty()) throw std::runtime_error(problem);
  contexts[device].store(c, std::memory_order_release);
  return c;
}

void* stream_of(const Tensor& t) {
  return t.is_cuda() ? static_cast<void*>(c10::cuda::getCurrentCUDAStream().stream()) : nullptr;
}

Tensor or_undefined(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// TMA needs a unit inner stride, a 16-byte aligned base and a row pitch that is a multiple of 16 bytes; other operands are copied.
Tensor tma_ready(const Tensor& t) {
  if (t.stride(1) == 1 && t.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0) return t;
  const int64_t rows = t.size(0), cols = t.size(1);
  Tensor view = at::empty({rows, (cols + 7) / 8 * 8}, t.options()).slice(1, 0, cols);
  view.copy_(t);
  return view;
}

// out[tokens, features] = x w^T + bias; x_t / w_t: that operand lies transposed in memory ([k, tokens] / [k, features]).  `sum`, if defined, is
// what the product is added to, and what is returned.
Tensor gemm(const Tensor& x_in, const Tensor& w_in, const Tensor& bias, bool x_t, bool w_t, const Tensor& sum = Tensor()) {
  if (x_in.scalar_type() != at::kBFloat16 || w_in.scalar_type() != at::kBFloat16)  // (the kernel takes its operands' element size for granted)
    throw py::type_error("native GEMMs take bf16 operands, got " + std::string(at::toString(x_in.scalar_type())) + " and " + at::toString(w_in.scalar_type()));
  const int64_t tokens = x_in.size(x_t ? 1 : 0), k = x_in.size(x_t ? 0 : 1), features = w_in.size(w_t ? 1 : 0);
  TORCH_CHECK(x_in.dim() == 2 && w_in.dim() == 2 && w_in.size(w_t ? 0 : 1) == k, "operands of a native GEMM of ", x_in.sizes(), " and ", w_in.sizes(),
              " do not contract");
  const Tensor x = tma_ready(x_in), w = tma_ready(w_in);
  Tensor out = sum.defined() ? sum : at::empty({tokens, features}, x.options());
  tpb_gemm_plan_t plan;
  check(lib.plan(int(tokens), int(features), int(k), 1, 0, 0, int(x_t || w_t), &plan), "gemm_plan");
  tpb_reduce_ctx_t* rc = context(x, plan.reduce && !plan.stream ? size_t(tokens) * size_t(out.stride(0)) : 0);
  tpb_gemm_opts_t opts = {};
  opts.x_mn = x_t;
  opts.w_mn = w_t;
  check(lib.gemm(x.const_data_ptr(), w.const_data_ptr(), out.mutable_data_ptr(), data(bias), data(sum), int(tokens), int(features), int(k), int(x.stride(0)),
                 int(w.stride(0)), int(out.stride(0)), 0, 1.f, &plan, rc, x_t || w_t ? &opts : nullptr, stream_of(x)),
        "tpb_gemm_bf16");
  launched.fetch_add(1, std::memory_order_relaxed);
  return out;
}

// What a call costs beside its launches is tensor operations that change nothing, 0.5 to 1 us each: a view or a conversion is taken only where
// shape or type ask for it.
Tensor rows_of(const Tensor& x) { return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}); }
Tensor as_type(const Tensor& t, at::ScalarType dtype) { return t.scalar_type() == dtype ? t : t.to(dtype); }

// Rows as the leading dimensions of x have it.
Tensor shaped_as(const Tensor& rows, const Tensor& x) {
  if (x.dim() == 2) return rows;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = rows.size(1);
  return rows.view(shape);
}
// The shape of an input, kept for its gradient where that is not its rows' (empty otherwise).
std::vector<int64_t> shape_of(const Tensor& x) { return x.dim() == 2 ? std::vector<int64_t>() : x.sizes().vec(); }
Tensor in_shape(const Tensor& rows, const c10::IValue& shape) {
  const auto sizes = shape.toIntVector();
  return sizes.empty() ? rows : rows.view(sizes);
}

// Whether something goes on around a gradient that a kernel would drop out of: a graph of its own (create_graph), a batch of gradients
// (is_grads_batched) or another transform, a tensor subclass.
bool more_than_numbers(const Tensor& g) {
  return (at::GradMode::is_enabled() && g.requires_grad()) || !g.has_storage() || g.unsafeGetTensorImpl()->is_python_dispatch();
}

// The gradient of a bias: column sums of g in fp32, as `dtype`.
Tensor column_sums(const Tensor& g, at::ScalarType dtype) {
  if (!lib.col_sum || more_than_numbers(g) || g.size(0) == 0 || g.size(1) % 8 || (dtype != at::kBFloat16 && dtype != at::kFloat) ||
      reinterpret_cast<uintptr_t>(g.const_data_ptr()) % 16)
    return g.sum(at::IntArrayRef{0}, false, at::kFloat).to(dtype);  // (summed in fp32 without an fp32 copy of the gradient)
  const int rows = int(g.size(0)), cols = int(g.size(1)), parts = lib.col_sum_parts(rows, cols);
  Tensor out = at::empty({cols}, g.options().dtype(dtype)), partials = parts > 1 ? at::empty({parts, cols}, g.options().dtype(at::kFloat)) : Tensor();
  check(lib.col_sum(g.const_data_ptr(), out.mutable_data_ptr(), parts > 1 ? partials.data_ptr<float>() : nullptr, rows, cols, dtype == at::kFloat, stream_of(g)),
        "tpb_col_sum");  // (not among the launches: those of a linear layer are its GEMMs)
  return out;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_) {
    const Tensor bias = or_undefined(bias_);
    const Tensor x2d = rows_of(x);
    const Tensor out = gemm(x2d, weight, bias, false, false);
    ctx->save_for_backward({x2d, weight});
    ctx->saved_data["shape"] = shape_of(x);
    ctx->saved_data["bias"] = bias.defined();
    return shaped_as(out, x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2d = saved[0], &weight = saved[1], &grad = grads[0];
    const Tensor g = as_type(rows_of(grad), at::kBFloat16).contiguous();
    Tensor gx, gw, gb;
    if (ctx->needs_input_grad(0)) gx = in_shape(gemm(g, weight, Tensor(), false, true), ctx->saved_data["shape"]);
    if (ctx->needs_input_grad(1)) gw = gemm(g, x2d, Tensor(), true, true);
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2))
      gb = column_sums(g, grad.scalar_type());
    return {gx, gw, gb};
  }
};

// Several projections of one input, without biases.  As nodes of their own they leave the sum of their gradients of the input to the engine, which
// reads and writes each of them once more (three of 8192 x 4096: 59 us); here the second and third GEMM add to what the one before stored.
struct LinearsFn : torch::autograd::Function<LinearsFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, at::TensorList weights) {
    const Tensor x2d = rows_of(x);
    torch::autograd::variable_list outs, saved{x2d};
    for (const Tensor& w : weights) {
      outs.push_back(shaped_as(gemm(x2d, w, Tensor(), false, false), x));
      saved.push_back(w);
    }
    ctx->save_for_backward(saved);
    ctx->saved_data["shape"] = shape_of(x);
    ctx->set_materialize_grads(false);
    return outs;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list out(1 + grads.size());
    Tensor gx;
    for (size_t i = grads.size(); i-- > 0;) {  // (the engine's order, so that there are only roundings fewer; q, the largest where k and v have fewer heads, last)
      if (!grads[i].defined()) continue;       // (nobody used that projection)
      const Tensor g = as_type(rows_of(grads[i]), at::kBFloat16).contiguous();
      if (ctx->needs_input_grad(0)) gx = gemm(g, saved[1 + i], Tensor(), false, true, gx);
      if (ctx->needs_input_grad(1 + i)) out[1 + i] = gemm(g, saved[0], Tensor(), true, true);
    }
    if (gx.defined()) out[0] = in_shape(gx, ctx->saved_data["shape"]);
    return out;
  }
};

std::vector<Tensor> linears(const Tensor& x, const std::vector<Tensor>& weights) { return LinearsFn::apply(x, at::TensorList(weights)); }

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_) {
  const Tensor bias = or_undefined(bias_);
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad())))
    return LinearFn::apply(x, weight, bias_);
  return shaped_as(gemm(rows_of(x), weight, bias, false, false), x);
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return 0;
  if (t.scalar_type() == at::kFloat) return 1;
  throw py::type_error("native kernels take bf16 or fp32 tensors, got " + std::string(at::toString(t.scalar_type())));
}

// mode 0: RMSNorm, 1: LayerNorm, of bf16 or fp32 rows.
struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_,
                        double eps, int64_t mode) {
    const Tensor weight = or_undefined(weight_), bias = or_undefined(bias_);
    const int dtype = dtype_code(x);
    const Tensor x2d = rows_of(x).contiguous();
    const Tensor w = weight.defined() ? as_type(weight, x.scalar_type()).contiguous() : Tensor();
    const Tensor b = bias.defined() ? as_type(bias, x.scalar_type()).contiguous() : Tensor();
    const int64_t rows = x2d.size(0), cols = x2d.size(1);
    Tensor out = at::empty_like(x2d);
    Tensor stats = at::empty({mode == 1 ? 2 : 1, rows}, x2d.options().dtype(at::kFloat));  // 1 / deviation, and for LayerNorm the mean, of every row
    float* rstd = stats.data_ptr<float>();
    check(lib.norm_fwd(x2d.const_data_ptr(), nullptr, data(w), data(b), out.mutable_data_ptr(), nullptr, rstd, mode == 1 ? rstd + rows : nullptr, int(rows),
                       int(cols), float(eps), int(mode), dtype, stream_of(x2d)),
          "tpb_norm_fwd");
    launched.fetch_add(1, std::memory_order_relaxed);
    ctx->save_for_backward({x2d, w, stats});
    ctx->saved_data["shape"] = shape_of(x);
    ctx->saved_data["meta"] = std::vector<int64_t>{mode, weight.defined() ? int64_t(weight.scalar_type()) : int64_t(-1),
                                                   bias.defined() ? int64_t(bias.scalar_type()) : int64_t(-1)};
    return shaped_as(out, x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2d = saved[0], &w = saved[1], &stats = saved[2];
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const int64_t mode = meta[0], wdtype = meta[1], bdtype = meta[2];
    const Tensor g = as_type(rows_of(grads[0]), x2d.scalar_type()).contiguous();
    const int64_t rows = x2d.size(0), cols = x2d.size(1);
    Tensor dx = at::empty_like(x2d);
    // column sums: one fp32 partial row per CTA, added up by a second kernel that writes the gradients in their own dtype
    const bool has_w = wdtype >= 0, has_b = bdtype >= 0;
    const bool narrow = has_w && (!has_b || bdtype == wdtype) && wdtype == int64_t(at::kBFloat16);
    const int parts = lib.norm_bwd_parts(int(rows), int(cols));
    const auto fp32 = x2d.options().dtype(at::kFloat);
    const auto as_grad = narrow ? x2d.options().dtype(at::kBFloat16) : fp32;
    Tensor partials = has_w || has_b ? at::empty({int(has_w) + int(has_b), parts, cols}, fp32) : Tensor();
    float* part_w = has_w ? partials.data_ptr<float>() : nullptr;
    float* part_b = has_b ? partials.data_ptr<float>() + (has_w ? int64_t(parts) * cols : 0) : nullptr;
    const float* rstd = stats.const_data_ptr<float>();
    Tensor dw = has_w ? at::empty({cols}, as_grad) : Tensor(), db = has_b ? at::empty({cols}, as_grad) : Tensor();
    auto out = [](Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
    check(lib.norm_bwd(g.const_data_ptr(), x2d.const_data_ptr(), data(w), rstd, mode == 1 ? rstd + rows : nullptr, dx.mutable_data_ptr(), part_w, part_b, out(dw),
                       out(db), int(rows), int(cols), int(mode), dtype_code(x2d), narrow ? 0 : 1, stream_of(x2d)),
          "tpb_norm_bwd");
    launched.fetch_add(has_w || has_b ? 2 : 1, std::memory_order_relaxed);
    if (has_w) dw = as_type(dw, at::ScalarType(wdtype));
    if (has_b) db = as_type(db, at::ScalarType(bdtype));
    return {in_shape(dx, ctx->saved_data["shape"]), dw, db, Tensor(), Tensor()};
  }
};

Tensor norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps, int64_t mode) {
  return NormFn::apply(x, weight, bias, eps, mode);
}

// ---- 8-bit serving ----
// The ordinary calls: plain CUDA tensors that fit together and lie as the kernels read them, nothing that takes a gradient or has a tangent, nothing around the call that
// wants to see its steps.  Every other call gets no value here and goes on in Python, which says what is wrong with it, makes the copies that it needs, or takes the steps.

// Whether something stands between a call and its kernels that they would drop out of: a dispatch mode (fake tensors, make_fx, which follows tensors without wrapping
// them), its form ahead of dispatch, a functorch transform, functionalization, tracing.  The thread knows, not the tensors.
bool interposed() {
  constexpr c10::DispatchKeySet around({c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::Functionalize, c10::DispatchKey::PreDispatch});
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || (c10::impl::tls_local_dispatch_key_set().included_ & around).raw_repr() != 0 ||
         torch::jit::tracer::isTracing();
}

bool plain(const Tensor& t, at::ScalarType dtype, const c10::Device& device) {
  return t.scalar_type() == dtype && t.device() == device && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.is_neg() &&
         !(at::GradMode::is_enabled() && t.requires_grad()) && !t._fw_grad(0).defined();
}
// Rows that lie one pitch apart: their number, and the pitch (of a single row, its length rounded up).
bool rows_apart(const Tensor& t, int64_t* rows, int64_t* pitch) {
  const int64_t dims = t.dim(), cols = dims ? t.size(-1) : 0;
  if (dims < 1 || cols == 0 || (t.stride(-1) != 1 && cols != 1)) return false;
  *rows = 1;
  *pitch = (cols + 15) / 16 * 16;
  for (int64_t d = dims - 2; d >= 0; --d) {
    const int64_t n = t.size(d);
    if (n != 1) {
      if (*rows == 1) *pitch = t.stride(d);
      else if (t.stride(d) != *pitch * *rows) return false;
    }
    *rows *= n;
  }
  return *rows > 0 && *pitch >= cols && *rows < (int64_t(1) << 31) && cols < (int64_t(1) << 31);
}
bool vector_of(const Tensor& t, int64_t n) { return t.dim() == 1 && t.size(0) == n && (t.stride(0) == 1 || n == 1); }

// Uninitialised memory of the current device, without the detour through the dispatcher.
Tensor room_for(at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, std::nullopt);
}

struct Int8Out {
  Tensor values, scales;
};
// Values a multiple of 16 bytes apart.  An allocation each: two types over one storage cannot be saved.
Int8Out int8_out(const Tensor& x, int64_t rows) {
  const int64_t dims = x.dim(), pitch = (x.size(-1) + 15) / 16 * 16;
  Tensor values = room_for({rows * pitch}, at::kChar);
  std::vector<int64_t> strides(dims, 1);
  for (int64_t d = dims - 2, next = pitch; d >= 0; next *= x.size(d--)) strides[d] = next;
  values.unsafeGetTensorImpl()->set_sizes_and_strides(x.sizes(), strides);
  return {values, room_for(x.sizes().slice(0, dims - 1), at::kFloat)};
}

// norm: -1 the rows as they are, 0 RMSNorm, 1 LayerNorm.  Values, scales, and with a residual the sum (`out` and `sum` stay as they are where it returns false).
bool rows_int8(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, int64_t norm, const Tensor& residual, Int8Out* out, Tensor* sum) {
  const auto dtype = x.scalar_type();
  int64_t rows, pitch, residual_rows, residual_pitch = 0;
  if (!lib.rows_int8 || !x.is_cuda() || (dtype != at::kBFloat16 && dtype != at::kFloat) || interposed() || !plain(x, dtype, x.device()) ||
      !rows_apart(x, &rows, &pitch))
    return false;
  const int64_t cols = x.size(-1);
  for (const Tensor* t : {&weight, &bias})
    if (t->defined() && (!plain(*t, dtype, x.device()) || !vector_of(*t, cols))) return false;
  if (residual.defined() && (!plain(residual, dtype, x.device()) || residual.sizes() != x.sizes() || !rows_apart(residual, &residual_rows, &residual_pitch)))
    return false;
  const py::gil_scoped_release unlocked;
  const c10::cuda::CUDAGuard guard(x.device());
  *out = int8_out(x, rows);
  if (residual.defined()) *sum = room_for(x.sizes(), dtype);
  check(lib.rows_int8(x.const_data_ptr(), data(residual), data(weight), data(bias), sum && sum->defined() ? sum->mutable_data_ptr() : nullptr,
                      static_cast<int8_t*>(out->values.mutable_data_ptr()), out->scales.mutable_data_ptr<float>(), int(rows), int(cols), pitch, residual_pitch, cols,
                      (cols + 15) / 16 * 16, float(eps), int(norm) + 1, dtype == at::kFloat, 0, context(x, 0)->status, stream_of(x)),
        "tpb_rows_int8");
  launched.fetch_add(1, std::memory_order_relaxed);
  return true;
}

// The product, or no tensor.
Tensor linear_int8(const Tensor& x, const Tensor& sx, const Tensor& w, const Tensor& sw, const Tensor& bias, int64_t act, const Tensor& residual) {
  int64_t tokens, ldx, features, ldw, residual_rows, ld_res = 0;
  const auto device = x.device();
  if (!lib.gemm_int8 || !x.is_cuda() || interposed() || !plain(x, at::kChar, device) || !plain(w, at::kChar, device) ||
      !plain(sx, at::kFloat, device) || !plain(sw, at::kFloat, device) || x.dim() < 2 || w.dim() != 2 || !rows_apart(x, &tokens, &ldx) ||
      !rows_apart(w, &features, &ldw) || x.size(-1) != w.size(1) || !vector_of(sw, features) || sx.sizes() != x.sizes().slice(0, x.dim() - 1) ||
      !sx.is_contiguous())
    return {};
  const int64_t k = w.size(1), cols = act == 5 ? features / 2 : features;
  auto aligned = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; };
  if (k > 131071 || ldx % 16 || ldw % 16 || !aligned(x) || !aligned(w) || (act == 5 && (features % 32 || residual.defined()))) return {};
  if (bias.defined() && (!plain(bias, at::kBFloat16, device) || !vector_of(bias, features))) return {};
  c10::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = cols;
  if (residual.defined() && (!plain(residual, at::kBFloat16, device) || residual.sizes() != at::IntArrayRef(shape) || !rows_apart(residual, &residual_rows, &ld_res)))
    return {};
  const py::gil_scoped_release unlocked;
  const c10::cuda::CUDAGuard guard(device);
  Tensor out = room_for(shape, at::kBFloat16);
  check(lib.gemm_int8(static_cast<const int8_t*>(x.const_data_ptr()), sx.const_data_ptr<float>(), static_cast<const int8_t*>(w.const_data_ptr()),
                      sw.const_data_ptr<float>(), out.mutable_data_ptr(), data(bias), data(residual), int(tokens), int(features), int(k), ldx, ldw, cols, ld_res,
                      int(act), 0, context(x, 0)->status, stream_of(x)),
        "tpb_gemm_int8");
  launched.fetch_add(1, std::memory_order_relaxed);
  return out;
}

// ---- sequences of different lengths ----
// As the 8-bit calls: the ordinary ones are taken here, every other goes on in Python.

bool ints(const Tensor& t, int64_t dims, const c10::Device& device) {
  return plain(t, at::kInt, device) && t.dim() == dims && (t.stride(dims - 1) == 1 || t.size(dims - 1) <= 1);
}
// bf16 with the last dimension together and every row on a 16-byte boundary.
bool vectors(const Tensor& t, int64_t dims, const c10::Device& device) {
  if (!plain(t, at::kBFloat16, device) || t.dim() != dims || t.stride(dims - 1) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16) return false;
  for (int64_t d = 0; d + 1 < dims; ++d)
    if (t.size(d) > 1 && t.stride(d) % 8) return false;
  return true;
}
long long step(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

struct Pages {
  const Tensor *keys, *values, *table, *starts, *past;
  int64_t n() const { return past->size(0); }
};
bool pages_fit(const Pages& p, int64_t least_page) {
  const Tensor& k = *p.keys;
  const auto device = k.device();
  if (!k.is_cuda() || !vectors(k, 4, device) || !vectors(*p.values, 4, device) || k.sizes() != p.values->sizes() || k.numel() == 0) return false;
  for (int64_t d = 0; d < 3; ++d)
    if (k.size(d) > 1 && (k.stride(d) <= 0 || p.values->stride(d) <= 0)) return false;
  const int64_t page = k.size(2), limit = int64_t(1) << 31;
  return page >= least_page && (page & (page - 1)) == 0 && page < limit && k.size(0) < limit && ints(*p.table, 2, device) && ints(*p.starts, 1, device) &&
         ints(*p.past, 1, device) && p.starts->size(0) == p.n() + 1 && p.table->size(0) == p.n() && p.n() > 0 && p.n() < limit - 1 && p.table->size(1) > 0 &&
         p.table->size(1) < limit;
}
bool rows_like(const Tensor& t, int64_t heads, const Pages& p, int64_t tokens) {
  return vectors(t, 3, p.keys->device()) && t.size(2) == p.keys->size(3) && t.size(0) == tokens && (heads < 0 || t.size(1) == heads);
}
bool written_once(const Tensor& t) {
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) == 0) return false;
  return true;
}

// scale 0: the usual one.  The result, or no tensor.
Tensor paged_attention(const Tensor& q, const Pages& p, double scale, int64_t window, int64_t most_new, const Tensor& given) {
  if (!lib.paged_attention || interposed() || !pages_fit(p, 16) || q.dim() != 3) return {};
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = p.keys->size(1);
  if ((dim != 64 && dim != 128) || tokens <= 0 || heads <= 0 || heads % kv_heads || tokens * heads >= (int64_t(1) << 30) || !rows_like(q, -1, p, tokens)) return {};
  if (given.defined() && (!rows_like(given, heads, p, tokens) || !written_once(given))) return {};
  const py::gil_scoped_release unlocked;
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = given.defined() ? given : room_for(q.sizes(), at::kBFloat16);
  tpb_paged_attn_t a = {};
  const int64_t most = most_new < 0 ? tokens : std::min(most_new, tokens);
  a.workspace_bytes = lib.paged_attention_workspace(int(p.n()), int(tokens), int(p.table->size(1)), int(p.keys->size(2)), int(most), int(kv_heads),
                                                    int(heads / kv_heads), int(dim));
  const Tensor workspace = room_for({a.workspace_bytes}, at::kByte);
  a.q = q.const_data_ptr(), a.out = out.mutable_data_ptr(), a.keys = p.keys->const_data_ptr(), a.values = p.values->const_data_ptr();
  a.table = p.table->const_data_ptr<int>(), a.starts = p.starts->const_data_ptr<int>(), a.past = p.past->const_data_ptr<int>();
  a.status = context(q, 0)->status, a.workspace = workspace.mutable_data_ptr();
  a.q_st = step(q, 0), a.q_sh = step(q, 1), a.o_st = step(out, 0), a.o_sh = step(out, 1);
  a.k_sp = step(*p.keys, 0), a.k_sh = step(*p.keys, 1), a.k_ss = step(*p.keys, 2);
  a.v_sp = step(*p.values, 0), a.v_sh = step(*p.values, 1), a.v_ss = step(*p.values, 2), a.table_ld = p.table->stride(0);
  a.n = int(p.n()), a.tokens = int(tokens), a.heads = int(heads), a.kv_heads = int(kv_heads), a.head_dim = int(dim), a.pages = int(p.keys->size(0));
  a.page_size = int(p.keys->size(2)), a.table_width = int(p.table->size(1)), a.window = int(std::min<int64_t>(window, 1 << 30)), a.most_new = int(most);
  a.fill_rest = !given.defined(), a.scale = scale == 0. ? float(1. / std::sqrt(double(dim))) : float(scale);
  check(lib.paged_attention(&a, stream_of(q)), "tpb_paged_attention");
  launched.fetch_add(a.launches, std::memory_order_relaxed);
  return out;
}

struct Turn {
  Tensor frequencies;
  bool interleaved = false;
  double factor = 1.;
};
enum class Queries { not_taken, kept, made };

Queries paged_append(const Pages& p, const Tensor& q, const Tensor& k, const Tensor& v, const Turn& turn, const Tensor& q_norm, const Tensor& k_norm, double eps,
                     const Tensor& given, Tensor* result) {
  if (!lib.paged_append || interposed() || !pages_fit(p, 1) || k.dim() != 3) return Queries::not_taken;
  const int64_t tokens = k.size(0), kv_heads = p.keys->size(1), dim = p.keys->size(3);
  const auto device = p.keys->device();
  if (dim % 8 || dim > 256 || tokens <= 0 || tokens >= (int64_t(1) << 31) || !rows_like(k, kv_heads, p, tokens) || !rows_like(v, kv_heads, p, tokens) ||
      !written_once(*p.keys) || !written_once(*p.values))
    return Queries::not_taken;
  for (const Tensor* t : {&q_norm, &k_norm})
    if (t->defined() && (!vectors(*t, 1, device) || t->size(0) != dim)) return Queries::not_taken;
  if (turn.frequencies.defined() && (!plain(turn.frequencies, at::kFloat, device) || turn.frequencies.dim() != 1 || !turn.frequencies.is_contiguous() ||
                                     turn.frequencies.size(0) == 0 || 2 * turn.frequencies.size(0) > dim))
    return Queries::not_taken;
  if (q.defined() && (!rows_like(q, -1, p, tokens) || q.size(1) == 0)) return Queries::not_taken;
  if (given.defined() && (!q.defined() || !rows_like(given, q.size(1), p, tokens) || !written_once(given))) return Queries::not_taken;
  for (const Tensor* t : {&q, &k, &v, &given})
    if (t->defined() && (step(*t, 0) >= TPB_APPEND_ROW_STRIDE || step(*t, 1) >= TPB_APPEND_ROW_STRIDE)) return Queries::not_taken;
  if (step(*p.keys, 1) >= TPB_APPEND_HEAD_STRIDE || step(*p.values, 1) >= TPB_APPEND_HEAD_STRIDE) return Queries::not_taken;
  const bool makes = q.defined() && (turn.frequencies.defined() || q_norm.defined() || given.defined());
  const py::gil_scoped_release unlocked;
  const c10::cuda::CUDAGuard guard(device);
  tpb_paged_append_t a = {};
  if (makes) {
    *result = given.defined() ? given : room_for(q.sizes(), at::kBFloat16);
    a.q = q.const_data_ptr(), a.q_out = result->mutable_data_ptr(), a.heads = int(q.size(1));
    a.q_st = step(q, 0), a.q_sh = step(q, 1), a.o_st = step(*result, 0), a.o_sh = step(*result, 1);
  }
  a.k = k.const_data_ptr(), a.v = v.const_data_ptr(), a.keys = p.keys->mutable_data_ptr(), a.values = p.values->mutable_data_ptr();
  a.table = p.table->const_data_ptr<int>(), a.starts = p.starts->const_data_ptr<int>(), a.past = p.past->const_data_ptr<int>();
  a.q_norm = data(q_norm), a.k_norm = data(k_norm), a.status = context(k, 0)->status;
  if (turn.frequencies.defined()) {
    a.frequencies = turn.frequencies.const_data_ptr<float>();
    a.rotary_dim = int(2 * turn.frequencies.size(0)), a.interleaved = turn.interleaved;
  }
  a.k_st = step(k, 0), a.k_sh = step(k, 1), a.v_st = step(v, 0), a.v_sh = step(v, 1);
  a.k_sp = step(*p.keys, 0), a.k_shead = step(*p.keys, 1), a.k_ss = step(*p.keys, 2);
  a.v_sp = step(*p.values, 0), a.v_shead = step(*p.values, 1), a.v_ss = step(*p.values, 2), a.table_ld = p.table->stride(0);
  a.n = int(p.n()), a.tokens = int(tokens), a.kv_heads = int(kv_heads), a.head_dim = int(dim), a.pages = int(p.keys->size(0)), a.page_size = int(p.keys->size(2));
  a.table_width = int(p.table->size(1)), a.fill_rest = !given.defined(), a.factor = float(turn.factor), a.eps = float(eps);
  check(lib.paged_append(&a, stream_of(k)), "tpb_paged_append");
  launched.fetch_add(1, std::memory_order_relaxed);
  return makes ? Queries::made : Queries::kept;
}

struct PerRow {  // a penalty: fp32 [rows], or one number for all
  Tensor rows;
  double all;
};
Tensor adjust_logits(const Tensor& x, const Tensor& tokens, const Tensor& lengths, const Tensor& prompts, const PerRow& repetition, const PerRow& frequency,
                     const PerRow& presence, const Tensor& bias, const Tensor& allowed) {
  const auto device = x.device();
  const auto dtype = x.scalar_type();
  const int64_t limit = int64_t(1) << 31;
  if (!lib.adjust_logits || !x.is_cuda() || (dtype != at::kBFloat16 && dtype != at::kFloat) || interposed() || !plain(x, dtype, device) || x.dim() != 2) return {};
  const int64_t rows = x.size(0), vocab = x.size(1), words = (vocab + 31) / 32;
  if (rows <= 0 || vocab <= 0 || rows >= limit || vocab >= limit || (x.stride(1) != 1 && vocab != 1)) return {};
  if (!tokens.defined() && (lengths.defined() || prompts.defined() || repetition.rows.defined() || frequency.rows.defined() || presence.rows.defined())) return {};
  if (tokens.defined() && (!plain(tokens, at::kLong, device) || tokens.dim() != 2 || tokens.size(0) != rows || tokens.size(1) >= limit ||
                           (tokens.stride(1) != 1 && tokens.size(1) > 1)))
    return {};
  for (const Tensor* t : {&lengths, &prompts})
    if (t->defined() && (!ints(*t, 1, device) || t->size(0) != rows)) return {};
  for (const PerRow* t : {&repetition, &frequency, &presence})
    if (t->rows.defined() && (!plain(t->rows, at::kFloat, device) || !vector_of(t->rows, rows))) return {};
  if (bias.defined() && ((bias.scalar_type() != at::kFloat && bias.scalar_type() != at::kBFloat16) || !plain(bias, bias.scalar_type(), device) || bias.dim() < 1 ||
                         bias.dim() > 2 || bias.size(-1) != vocab || (bias.dim() == 2 && bias.size(0) != rows) || (bias.stride(-1) != 1 && vocab != 1)))
    return {};
  if (allowed.defined() && (allowed.dim() < 1 || allowed.dim() > 2 || !ints(allowed, allowed.dim(), device) || allowed.size(-1) != words ||
                            (allowed.dim() == 2 && allowed.size(0) != rows)))
    return {};
  const py::gil_scoped_release unlocked;
  const c10::cuda::CUDAGuard guard(device);
  Tensor out = room_for(x.sizes(), dtype);
  tpb_adjust_logits_t a = {};
  a.logits = x.const_data_ptr(), a.out = out.mutable_data_ptr(), a.status = context(x, 0)->status;
  a.logits_ld = x.stride(0), a.out_ld = vocab, a.rows = int(rows), a.vocab = int(vocab), a.dtype = dtype == at::kFloat, a.repetition_all = 1.f;
  if (tokens.defined() && tokens.size(1) > 0) {
    auto numbers = [](const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; };
    a.tokens = reinterpret_cast<const long long*>(tokens.const_data_ptr<int64_t>()), a.tokens_ld = tokens.stride(0), a.width = int(tokens.size(1));
    a.lengths = lengths.defined() ? lengths.const_data_ptr<int>() : nullptr, a.prompts = prompts.defined() ? prompts.const_data_ptr<int>() : nullptr;
    a.repetition = numbers(repetition.rows), a.frequency = numbers(frequency.rows), a.presence = numbers(presence.rows);
    a.repetition_all = float(repetition.all), a.frequency_all = float(frequency.all), a.presence_all = float(presence.all);
  }
  if (bias.defined()) a.bias = bias.const_data_ptr(), a.bias_ld = bias.dim() == 2 ? bias.stride(0) : 0, a.bias_dtype = bias.scalar_type() == at::kFloat;
  if (allowed.defined()) a.allowed = allowed.const_data_ptr<int>(), a.allowed_ld = allowed.dim() == 2 ? allowed.stride(0) : 0;
  check(lib.adjust_logits(&a, stream_of(x)), "tpb_adjust_logits");
  launched.fetch_add(a.launches, std::memory_order_relaxed);
  return out;
}

// Whether operators are being captured or shapes followed (make_fx, fake tensors, capture ahead of dispatch): a kernel would leave nothing in the graph but the
// allocation of its result.  Other dispatch modes (recomputation with a policy, counters) let kernels run.
bool captured() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::PreDispatch)) return true;
  if (!Modes::any_modes_set()) return false;
  for (const auto key : {c10::impl::TorchDispatchModeKey::PROXY, c10::impl::TorchDispatchModeKey::FAKE, c10::impl::TorchDispatchModeKey::FUNCTIONAL})
    if (Modes::get_mode(key).has_value()) return true;
  return false;
}

// The interpreter's side of these calls, without pybind11's conversions, which cost 0.6 us of a call's 4.5.
PyObject* rows_type = nullptr;  // the named tuple (values, scales)
PyObject* act_codes = nullptr;  // activation -> code

const Tensor nothing;
// The tensor behind an argument (None: an undefined one), or null if it is neither.
const Tensor* tensor_of(PyObject* o) { return o == Py_None ? &nothing : THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
const Tensor* a_tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

PyObject* tuple_of(PyTypeObject* type, PyObject* a, PyObject* b) {  // takes the references
  PyObject* t = a && b ? type->tp_alloc(type, 2) : nullptr;
  if (!t) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}
PyObject* rows_object(const Int8Out& r) { return tuple_of(reinterpret_cast<PyTypeObject*>(rows_type), THPVariable_Wrap(r.values), THPVariable_Wrap(r.scales)); }

// (x) -> rows
PyObject* py_quantize_int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* x = n == 1 && rows_type ? a_tensor(args[0]) : nullptr;
  Int8Out out;
  if (!x || !rows_int8(*x, nothing, nothing, 0., -1, nothing, &out, nullptr)) Py_RETURN_NONE;
  return rows_object(out);
  END_HANDLE_TH_ERRORS
}
// (x, weight, bias, eps, 0 RMSNorm / 1 LayerNorm, residual) -> (rows, sum)
PyObject* py_norm_int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !rows_type) Py_RETURN_NONE;
  const Tensor *x = a_tensor(args[0]), *weight = tensor_of(args[1]), *bias = tensor_of(args[2]), *residual = tensor_of(args[5]);
  if (!x || !weight || !bias || !residual) Py_RETURN_NONE;
  const double eps = PyFloat_AsDouble(args[3]);
  const long norm = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  Int8Out out;
  Tensor sum;
  if (norm < 0 || norm > 1 || !rows_int8(*x, *weight, *bias, eps, norm, *residual, &out, &sum)) Py_RETURN_NONE;
  PyObject* rows = rows_object(out);
  return rows ? tuple_of(&PyTuple_Type, rows, sum.defined() ? THPVariable_Wrap(sum) : Py_NewRef(args[0])) : nullptr;
  END_HANDLE_TH_ERRORS
}
// (rows, weight's rows, bias, activation, residual) -> product
PyObject* py_linear_int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !act_codes) Py_RETURN_NONE;
  const Tensor *part[4], *bias = tensor_of(args[2]), *residual = tensor_of(args[4]);
  for (int i = 0; i < 2; ++i) {
    if (!PyTuple_Check(args[i]) || PyTuple_GET_SIZE(args[i]) != 2) Py_RETURN_NONE;
    for (int j = 0; j < 2; ++j)
      if (!(part[2 * i + j] = a_tensor(PyTuple_GET_ITEM(args[i], j)))) Py_RETURN_NONE;
  }
  if (!bias || !residual || (args[3] != Py_None && !PyUnicode_CheckExact(args[3]))) Py_RETURN_NONE;
  PyObject* code = PyDict_GetItemWithError(act_codes, args[3]);
  if (!code) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const Tensor out = linear_int8(*part[0], *part[1], *part[2], *part[3], *bias, PyLong_AsLong(code), *residual);
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}
// The tensors of a cache and of a batch's lengths.
bool pages_of(PyObject* cache, PyObject* starts, PyObject* past, Pages* p) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 3) return false;
  p->keys = a_tensor(PyTuple_GET_ITEM(cache, 0));
  p->values = a_tensor(PyTuple_GET_ITEM(cache, 1));
  p->table = a_tensor(PyTuple_GET_ITEM(cache, 2));
  p->starts = a_tensor(starts);
  p->past = a_tensor(past);
  return p->keys && p->values && p->table && p->starts && p->past && p->past->dim() == 1 && p->starts->dim() == 1 && p->table->dim() == 2;
}
// (q, cache, starts, past, scale, window, most_new, out) -> result
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  const Tensor *q = n == 8 ? a_tensor(args[0]) : nullptr, *given = n == 8 ? tensor_of(args[7]) : nullptr;
  if (!q || !given || !pages_of(args[1], args[2], args[3], &p)) Py_RETURN_NONE;
  double scale = 0.;
  int64_t window = 0, most_new = -1;
  if (args[4] != Py_None) {
    if (!PyFloat_CheckExact(args[4]) || !(PyFloat_AS_DOUBLE(args[4]) > 0.) || std::isinf(PyFloat_AS_DOUBLE(args[4]))) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(args[4]);
  }
  for (int i = 5; i < 7; ++i) {
    if (args[i] == Py_None) continue;
    if (!PyLong_CheckExact(args[i])) Py_RETURN_NONE;
    int over = 0;
    const long long value = PyLong_AsLongLongAndOverflow(args[i], &over);
    if (over || value < (i == 5 ? 1 : 0)) Py_RETURN_NONE;
    (i == 5 ? window : most_new) = value;
  }
  const Tensor out = paged_attention(*q, p, scale, window, most_new, *given);
  if (!out.defined()) Py_RETURN_NONE;
  return given->defined() ? Py_NewRef(args[7]) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}
// (cache, q, k, v, starts, past, rotary, q_norm, k_norm, eps, out) -> (queries,)
PyObject* py_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  if (n != 11 || !pages_of(args[0], args[4], args[5], &p)) Py_RETURN_NONE;
  const Tensor *q = tensor_of(args[1]), *k = a_tensor(args[2]), *v = a_tensor(args[3]), *q_norm = tensor_of(args[7]), *k_norm = tensor_of(args[8]), *given = tensor_of(args[10]);
  if (!q || !k || !v || !q_norm || !k_norm || !given || !PyFloat_CheckExact(args[9])) Py_RETURN_NONE;
  Turn turn;
  if (args[6] != Py_None) {
    PyObject* t = args[6];
    const Tensor* f = PyTuple_Check(t) && PyTuple_GET_SIZE(t) == 3 ? a_tensor(PyTuple_GET_ITEM(t, 0)) : nullptr;
    if (!f || !PyBool_Check(PyTuple_GET_ITEM(t, 1)) || !PyFloat_CheckExact(PyTuple_GET_ITEM(t, 2))) Py_RETURN_NONE;
    turn = {*f, PyTuple_GET_ITEM(t, 1) == Py_True, PyFloat_AS_DOUBLE(PyTuple_GET_ITEM(t, 2))};
  }
  Tensor result;
  const Queries done = paged_append(p, *q, *k, *v, turn, *q_norm, *k_norm, PyFloat_AS_DOUBLE(args[9]), *given, &result);
  if (done == Queries::not_taken) Py_RETURN_NONE;
  PyObject* queries = done == Queries::kept ? Py_NewRef(args[1]) : given->defined() ? Py_NewRef(args[10]) : THPVariable_Wrap(result);
  if (!queries) return nullptr;
  PyObject* one = PyTuple_New(1);  // (a call without queries is done as well)
  if (!one) {
    Py_DECREF(queries);
    return nullptr;
  }
  PyTuple_SET_ITEM(one, 0, queries);
  return one;
  END_HANDLE_TH_ERRORS
}
// (logits, tokens, lengths, prompt lengths, repetition, frequency, presence, bias, allowed) -> logits
PyObject* py_adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* x = n == 9 ? a_tensor(args[0]) : nullptr;
  if (!x) Py_RETURN_NONE;
  const Tensor *tokens = tensor_of(args[1]), *lengths = tensor_of(args[2]), *prompts = tensor_of(args[3]), *bias = tensor_of(args[7]), *allowed = tensor_of(args[8]);
  if (!tokens || !lengths || !prompts || !bias || !allowed) Py_RETURN_NONE;
  PerRow penalties[3] = {{Tensor(), 1.}, {Tensor(), 0.}, {Tensor(), 0.}};
  for (int i = 0; i < 3; ++i) {
    PyObject* o = args[4 + i];
    if (o == Py_None) continue;
    if (THPVariable_Check(o)) {
      penalties[i].rows = THPVariable_Unpack(o);
    } else {
      if (!PyFloat_CheckExact(o) || !tokens->defined() || (i == 0 && !(PyFloat_AS_DOUBLE(o) > 0.))) Py_RETURN_NONE;
      penalties[i].all = PyFloat_AS_DOUBLE(o);
    }
  }
  const Tensor out = adjust_logits(*x, *tokens, *lengths, *prompts, penalties[0], penalties[1], penalties[2], *bias, *allowed);
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}
// () -> whether a call would go on in Python for what is around it
PyObject* py_interposed(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  return PyBool_FromLong(interposed());
  END_HANDLE_TH_ERRORS
}
// () -> whether operators are being captured
PyObject* py_captured(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  return PyBool_FromLong(captured());
  END_HANDLE_TH_ERRORS
}
PyMethodDef plain_calls[] = {
    {"captured", py_captured, METH_NOARGS, nullptr},
    {"interposed", py_interposed, METH_NOARGS, nullptr},
    {"quantize_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_quantize_int8)), METH_FASTCALL, nullptr},
    {"norm_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_norm_int8)), METH_FASTCALL, nullptr},
    {"linear_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear_int8)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_paged_attention)), METH_FASTCALL, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_paged_append)), METH_FASTCALL, nullptr},
    {"adjust_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_adjust_logits)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

void bind_int8(py::object type, py::dict codes) {
  Py_XDECREF(rows_type);
  Py_XDECREF(act_codes);
  rows_type = type.release().ptr();  // (kept like the callbacks above)
  act_codes = codes.release().ptr();
}

template <typename F>
void entry(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& addresses, py::function text, py::function reserve) {
  entry(lib.plan, addresses, "tpb_gemm_plan_ex");
  entry(lib.gemm, addresses, "tpb_gemm_bf16_ex");
  entry(lib.norm_fwd, addresses, "tpb_norm_fwd");
  entry(lib.norm_bwd, addresses, "tpb_norm_bwd");
  entry(lib.norm_bwd_parts, addresses, "tpb_norm_bwd_parts");
  if (addresses.contains("tpb_col_sum")) {
    entry(lib.col_sum_parts, addresses, "tpb_col_sum_parts");
    entry(lib.col_sum, addresses, "tpb_col_sum");
  } else {
    lib.col_sum = nullptr;
  }
  lib.rows_int8 = nullptr;
  lib.gemm_int8 = nullptr;
  if (addresses.contains("tpb_gemm_int8")) {
    entry(lib.rows_int8, addresses, "tpb_rows_int8");
    entry(lib.gemm_int8, addresses, "tpb_gemm_int8");
  }
  lib.paged_attention = nullptr;
  lib.paged_append = nullptr;
  lib.adjust_logits = nullptr;
  if (addresses.contains("tpb_paged_attention")) {
    entry(lib.paged_attention_workspace, addresses, "tpb_paged_attention_workspace");
    entry(lib.paged_attention, addresses, "tpb_paged_attention");
    entry(lib.paged_append, addresses, "tpb_paged_append");
    entry(lib.adjust_logits, addresses, "tpb_adjust_logits");
  }
  Py_XDECREF(error_text);
  Py_XDECREF(reserve_slots);
  error_text = text.release().ptr();  // (kept for the life of the process, beyond the interpreter's teardown of module globals)
  reserve_slots = reserve.release().ptr();
  for (auto& c : contexts) c.store(nullptr, std::memory_order_release);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("layout", [] { return TPB_API_LAYOUT; });  // of the structures that it hands to the library it is bound to
  m.def("launches", [] { return launched.load(std::memory_order_relaxed); });
  const auto unlocked = py::call_guard<py::gil_scoped_release>();
  m.def("linear", &linear, unlocked);
  m.def("linears", &linears, unlocked);
  m.def("norm", &norm, unlocked);
  m.def("bind_int8", &bind_int8);
  if (PyModule_AddFunctions(m.ptr(), plain_calls) != 0) throw py::error_already_set();
}
