// The native side of the operators beside MSDA (cross attention, rotary positions, dropout):
// their launches on tensors, which the registered operators call, and one autograd node each
// for plain eager calls, as bridge.cpp has for MSDA.

#include "bridge.h"

#include <ATen/Functions.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "deformops_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&deformops_cross_attention_workspace_size) attention_size = nullptr;
  decltype(&deformops_cross_attention_forward) attention_forward = nullptr;
  decltype(&deformops_cross_attention_backward) attention_backward = nullptr;
  decltype(&deformops_rotary) rotary = nullptr;
  decltype(&deformops_dropout) dropout = nullptr;
  decltype(&deformops_last_error) last_error = nullptr;
} g;

template <typename F> void bind(F& entry, uintptr_t address) { entry = reinterpret_cast<F>(address); }

void init_operators(const std::vector<uintptr_t>& at) {
  TORCH_CHECK(at.size() == 6, "deformops: six entry points are expected");
  bind(g.attention_size, at[0]);
  bind(g.attention_forward, at[1]);
  bind(g.attention_backward, at[2]);
  bind(g.rotary, at[3]);
  bind(g.dropout, at[4]);
  bind(g.last_error, at[5]);
}

void check(int status) {
  if (status == MSDA_OK) return;
  const char* message = g.last_error();
  TORCH_CHECK(false, message && *message ? std::string(message) : "deformops call failed with status " + std::to_string(status));
}

bool kernel_dtype(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

int dtype_code(at::ScalarType t) { return t == at::kFloat ? MSDA_F32 : t == at::kHalf ? MSDA_F16 : MSDA_BF16; }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool on_gpu(const Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided; }

// Neither a trace, a mode nor a wrapper watches the call; as MSDA's direct call asks.
bool watched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
         torch::jit::tracer::isTracing();
}

constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::BatchedNestedTensor, c10::DispatchKey::Functionalize,
                                        c10::DispatchKey::Python, c10::DispatchKey::Negative,
                                        c10::DispatchKey::Conjugate});

// A Python argument as a plain tensor: false for anything else. None is an undefined tensor
// where `optional`.
bool plain(pybind11::handle h, Tensor& out, bool optional = false) {
  if (optional && h.is_none()) return true;
  if (!THPVariable_CheckExact(h.ptr())) return false;
  out = THPVariable_Unpack(h.ptr());
  return !out.key_set().has_any(kWrapped);
}

void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                                ": forward-mode differentiation is not supported (an operand has a tangent)");
}

// A backward under graph capture hands its gradients to the leaves' accumulators, which stay on
// the stream they were made on for as long as any autograd graph of the leaf lives. One that an
// earlier graph made on another stream would pull that stream into the capture, which ends the
// process; so such a backward is refused before it hands anything on.
void refuse_foreign_accumulators(const char* what, const Tensor& grad) {
  const auto stream = c10::hip::getCurrentHIPStream(grad.device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status != hipStreamCaptureStatusActive) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& edge : node->next_edges()) {
    if (!edge.function || !dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
    const auto own = edge.function->stream();
    TORCH_CHECK(!own || own->id() == stream.id(), what,
                ": a backward is being captured while an autograd graph of the same leaf, made on another stream, "
                "still lives; delete what holds it (outputs, losses) before the capture");
  }
}

// The kernels' gradients carry no graph: where one is asked for and would lead through the
// output's gradient, they come back behind a node that raises.
variable_list once(variable_list out, const Tensor& grad) {
  if (at::GradMode::is_enabled() && grad.requires_grad()) {
    for (Tensor& t : out)
      if (t.defined()) t = t.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", int64_t(out.size()));
    out = (*error)(std::move(out));
  }
  return out;
}

// ---------------------------------------------------------------------------
// Cross attention.

// Dense and aligned to 16 bytes, as the backward reads it: a gradient may be a slice of another.
Tensor dense(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// Channels side by side: any other layout is copied.
Tensor rows(const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }

bool attention_agrees(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, const Tensor& lengths) {
  for (const Tensor* t : {&q, &k, &v, &mask, &lengths})
    if (t->defined() && (!on_gpu(*t) || t->device() != q.device())) return false;
  if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes()) return false;
  const int64_t B = q.size(0), H = q.size(2), D = q.size(3), K = k.size(2);
  if (k.size(0) != B || k.size(3) != D || D < 1 || D > 128 || K < 1 || H < 1 || H % K) return false;
  const at::ScalarType dtype = q.scalar_type();
  if (!kernel_dtype(dtype) || k.scalar_type() != dtype || v.scalar_type() != dtype) return false;
  if (mask.defined()) {
    if (mask.scalar_type() != at::kBool && !kernel_dtype(mask.scalar_type())) return false;
    if (mask.dim() != 2 && mask.dim() != 4) return false;
    const int64_t full[4] = {B, H, q.size(1), k.size(1)};
    for (int64_t i = 1; i <= mask.dim(); ++i)
      if (mask.size(-i) != 1 && mask.size(-i) != full[4 - i]) return false;
  }
  if (lengths.defined() && (lengths.dim() != 1 || lengths.size(0) != B ||
                            (lengths.scalar_type() != at::kLong && lengths.scalar_type() != at::kInt)))
    return false;
  return true;
}

struct Attention {
  Tensor q, k, v, mask, lengths;  // as the call refers to them
  deformops_attention call = {};

  Attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& mask_in, const Tensor& lengths_in,
            double scale)
      : q(rows(q_in)), k(rows(k_in)), v(rows(v_in)) {
    TORCH_CHECK(attention_agrees(q, k, v, mask_in, lengths_in),
                "cross_attention: the operands disagree in rank, size, dtype or device");
    call.batch = q.size(0);
    call.queries = q.size(1);
    call.heads = q.size(2);
    call.channels = q.size(3);
    call.keys = k.size(1);
    call.key_heads = k.size(2);
    const Tensor* tensors[3] = {&q, &k, &v};
    int64_t* strides[3] = {call.query_strides, call.key_strides, call.value_strides};
    for (int i = 0; i < 3; ++i)
      for (int j = 0; j < 3; ++j) strides[i][j] = tensors[i]->size(j) > 1 ? tensors[i]->stride(j) : 0;
    call.query = q.data_ptr();
    call.key = k.data_ptr();
    call.value = v.data_ptr();
    call.dtype = dtype_code(q.scalar_type());
    call.scale = static_cast<float>(scale);
    if (mask_in.defined()) {
      mask = mask_in.expand({call.batch, call.heads, call.queries, call.keys});
      call.mask_kind = mask.scalar_type() == at::kBool ? 1 : 2;
      if (call.mask_kind == 2) call.mask_dtype = dtype_code(mask.scalar_type());
      call.mask = mask.data_ptr();
      for (int j = 0; j < 4; ++j) call.mask_strides[j] = mask.size(j) > 1 ? mask.stride(j) : j == 3 ? 1 : 0;
    }
    if (lengths_in.defined()) {
      lengths = lengths_in.contiguous();
      call.key_lengths = lengths.data_ptr();
      call.index_dtype = lengths.scalar_type() == at::kLong ? MSDA_I64 : MSDA_I32;
    }
  }
};

// (out, stats); no statistics without `training`.
std::tuple<Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                                             const Tensor& lengths, double scale, bool training) {
  const c10::OptionalDeviceGuard guard(q.device());
  Attention a(q, k, v, mask, lengths, scale);
  Tensor out = at::empty({a.call.batch, a.call.queries, a.call.heads * a.call.channels}, q.options());
  Tensor stats = at::empty({training ? a.call.batch * a.call.heads * a.call.queries : 0, 2}, q.options().dtype(at::kFloat));
  a.call.output = out.data_ptr();
  int64_t bytes = 0, backward = 0;
  check(g.attention_size(&a.call, &bytes, &backward));
  Tensor workspace;
  if (bytes) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
  check(g.attention_forward(&a.call, training ? stats.data_ptr() : nullptr, bytes ? workspace.data_ptr() : nullptr, bytes,
                            stream_of(q)));
  return {out, stats};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                                                      const Tensor& lengths, double scale, const Tensor& out_in,
                                                      const Tensor& stats_in, const Tensor& grad_in) {
  const c10::OptionalDeviceGuard guard(q.device());
  Attention a(q, k, v, mask, lengths, scale);
  const Tensor grad = dense(grad_in.to(q.scalar_type())), out = dense(out_in), stats = dense(stats_in);
  const at::DimVector expected = {a.call.batch, a.call.queries, a.call.heads * a.call.channels};
  TORCH_CHECK(grad.sizes() == expected && out.sizes() == expected && out.scalar_type() == q.scalar_type() &&
                  stats.scalar_type() == at::kFloat && stats.numel() == 2 * a.call.batch * a.call.heads * a.call.queries &&
                  grad.device() == q.device() && out.device() == q.device() && stats.device() == q.device(),
              "cross_attention: the operands unpacked for the backward are not on the output's device or not of the "
              "sizes that were saved");
  Tensor grad_q = at::empty(q.sizes(), q.options()), grad_k = at::empty(k.sizes(), k.options()),
         grad_v = at::empty(v.sizes(), v.options());
  a.call.output = out.data_ptr();
  int64_t forward = 0, bytes = 0;
  check(g.attention_size(&a.call, &forward, &bytes));
  Tensor workspace;
  if (bytes) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
  check(g.attention_backward(&a.call, stats.data_ptr(), grad.data_ptr(), grad_q.data_ptr(), grad_k.data_ptr(),
                             grad_v.data_ptr(), bytes ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  return {grad_q, grad_k, grad_v};
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const std::optional<Tensor>& mask_in, const std::optional<Tensor>& lengths_in, double scale) {
    const Tensor mask = mask_in.value_or(Tensor()), lengths = lengths_in.value_or(Tensor());
    auto [out, stats] = attention_forward(q, k, v, mask, lengths, scale, true);
    ctx->save_for_backward({q, k, v, mask, lengths, out, stats});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list out(6);
    if (!grads[0].defined()) return out;
    refuse_foreign_accumulators("cross_attention", grads[0]);
    {
      const at::NoGradGuard no_grad;
      auto [q, k, v] = attention_backward(s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(), s[5], s[6], grads[0]);
      out[0] = q;
      out[1] = k;
      out[2] = v;
    }
    const variable_list three = once({out[0], out[1], out[2]}, grads[0]);
    return {three[0], three[1], three[2], Tensor(), Tensor(), Tensor()};
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask_in,
                       const std::optional<Tensor>& lengths_in, double scale) {
  const pybind11::gil_scoped_release no_gil;
  const Tensor mask = mask_in.value_or(Tensor()), lengths = lengths_in.value_or(Tensor());
  refuse_tangents("cross_attention", {&q, &k, &v, &mask});
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return CrossAttention::apply(q, k, v, mask_in, lengths_in, scale);
  const at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(attention_forward(q, k, v, mask, lengths, scale, false));
}

pybind11::object try_cross_attention(pybind11::handle q_in, pybind11::handle k_in, pybind11::handle v_in,
                                     pybind11::handle mask_in, pybind11::handle lengths_in, double scale) {
  Tensor q, k, v, mask, lengths;
  if (!plain(q_in, q) || !plain(k_in, k) || !plain(v_in, v) || !plain(mask_in, mask, true) ||
      !plain(lengths_in, lengths, true) || watched())
    return pybind11::none();
  if (!attention_agrees(q, k, v, mask, lengths) || (mask.defined() && mask.requires_grad())) return pybind11::none();
  if (scale == 0.0) scale = 1.0 / std::sqrt(double(q.size(3)));  // the default
  const float narrow = static_cast<float>(scale);
  if (!(narrow > 0.0f) || !std::isfinite(narrow)) return pybind11::none();
  return pybind11::cast(cross_attention(q, k, v, mask.defined() ? std::optional<Tensor>(mask) : std::nullopt,
                                        lengths.defined() ? std::optional<Tensor>(lengths) : std::nullopt, scale));
}

// ---------------------------------------------------------------------------
// Rotary positions.

int position_code(at::ScalarType t) {
  switch (t) {
    case at::kLong: return DEFORMOPS_POSITION_I64;
    case at::kInt: return DEFORMOPS_POSITION_I32;
    case at::kFloat: return DEFORMOPS_POSITION_F32;
    case at::kDouble: return DEFORMOPS_POSITION_F64;
    default: return -1;
  }
}

bool rotary_agrees(const Tensor& x, const Tensor& positions, const Tensor& frequencies, const std::vector<int64_t>& sections) {
  for (const Tensor* t : {&x, &positions, &frequencies})
    if (!on_gpu(*t) || t->device() != x.device()) return false;
  if (x.dim() != 4 || !kernel_dtype(x.scalar_type()) || position_code(positions.scalar_type()) < 0) return false;
  const int64_t axes = int64_t(sections.size()), p = positions.dim();
  if (p != 2 && p != 3) return false;
  if (axes < 1 || axes > 255 || positions.size(-1) != axes || positions.size(-2) != x.size(1)) return false;
  if (p == 3 && positions.size(0) != x.size(0) && positions.size(0) != 1) return false;
  int64_t pairs = 0;
  for (const int64_t n : sections) {
    if (n < 0 || n > 256) return false;
    pairs += n;
  }
  if (x.size(2) > 1 << 20 || x.size(3) > 1 << 20 || x.size(2) * x.size(3) > 1 << 20) return false;
  return pairs <= 256 && 2 * pairs <= x.size(3) && frequencies.dim() == 1 && frequencies.size(0) == pairs &&
         frequencies.scalar_type() == at::kFloat;
}

Tensor rotary_apply(const Tensor& x_in, const Tensor& positions, const Tensor& frequencies_in,
                    const std::vector<int64_t>& sections, bool interleaved, bool inverse) {
  TORCH_CHECK(rotary_agrees(x_in, positions, frequencies_in, sections),
              "rotary: the operands disagree in rank, size, dtype or device");
  const c10::OptionalDeviceGuard guard(x_in.device());
  const Tensor x = rows(x_in), frequencies = frequencies_in.contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  int64_t strides[3], p_strides[3] = {0, positions.stride(-2), positions.stride(-1)};
  for (int i = 0; i < 3; ++i) strides[i] = x.size(i) > 1 ? x.stride(i) : 0;
  if (positions.dim() == 3 && positions.size(0) > 1) p_strides[0] = positions.stride(0);
  check(g.rotary(x.data_ptr(), strides, y.data_ptr(), dtype_code(x.scalar_type()), positions.data_ptr(), p_strides,
                 position_code(positions.scalar_type()), frequencies.data_ptr(), sections.data(), int64_t(sections.size()),
                 x.size(0), x.size(1), x.size(2), x.size(3), interleaved, inverse, stream_of(x)));
  return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& frequencies,
                        const std::vector<int64_t>& sections, bool interleaved) {
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["dtype"] = x.scalar_type();
    return rotary_apply(x, positions, frequencies, sections, interleaved, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(5);
    refuse_foreign_accumulators("rotary", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    Tensor out;
    {
      const at::NoGradGuard no_grad;
      out = rotary_apply(grads[0].to(ctx->saved_data["dtype"].toScalarType()), s[0], s[1],
                         ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(), true);
    }
    return {once({out}, grads[0])[0], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor rotary(const Tensor& x, const Tensor& positions, const Tensor& frequencies, const std::vector<int64_t>& sections,
              bool interleaved) {
  const pybind11::gil_scoped_release no_gil;
  refuse_tangents("rotary", {&x, &positions, &frequencies});
  if (at::GradMode::is_enabled() && x.requires_grad()) return Rotary::apply(x, positions, frequencies, sections, interleaved);
  const at::AutoDispatchBelowADInplaceOrView below;
  return rotary_apply(x, positions, frequencies, sections, interleaved, false);
}

pybind11::object try_rotary(pybind11::handle x_in, pybind11::handle positions_in, pybind11::handle frequencies_in,
                            const std::vector<int64_t>& sections, bool interleaved) {
  Tensor x, positions, frequencies;
  if (!plain(x_in, x) || !plain(positions_in, positions) || !plain(frequencies_in, frequencies) || watched())
    return pybind11::none();
  if (!rotary_agrees(x, positions, frequencies, sections) || positions.requires_grad() || frequencies.requires_grad())
    return pybind11::none();
  return pybind11::cast(rotary(x, positions, frequencies, sections, interleaved));
}

// ---------------------------------------------------------------------------
// Dropout. The seed is a number, or an int64 tensor of one element on the GPU.

bool dropout_agrees(const Tensor& x, const Tensor& residual, const Tensor& seed_at) {
  if (!on_gpu(x) || !kernel_dtype(x.scalar_type())) return false;
  if (residual.defined() && (!on_gpu(residual) || residual.device() != x.device() || residual.sizes() != x.sizes() ||
                             residual.scalar_type() != x.scalar_type()))
    return false;
  return !seed_at.defined() || (on_gpu(seed_at) && seed_at.device() == x.device() && seed_at.numel() == 1 &&
                                seed_at.scalar_type() == at::kLong);
}

Tensor dropout_apply(const Tensor& x_in, double p, int64_t seed, const Tensor& seed_at, int64_t offset,
                     const Tensor& residual_in) {
  TORCH_CHECK(dropout_agrees(x_in, residual_in, seed_at), "dropout: the operands disagree in size, dtype or device");
  const c10::OptionalDeviceGuard guard(x_in.device());
  const Tensor x = x_in.contiguous(), residual = residual_in.defined() ? residual_in.contiguous() : Tensor();
  Tensor y = at::empty(x.sizes(), x.options());
  check(g.dropout(x.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr, y.data_ptr(),
                  dtype_code(x.scalar_type()), x.numel(), p, uint64_t(seed),
                  seed_at.defined() ? seed_at.data_ptr() : nullptr, uint64_t(offset), stream_of(x)));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed,
                        const std::optional<Tensor>& seed_at_in, int64_t offset, const std::optional<Tensor>& residual_in) {
    const Tensor seed_at = seed_at_in.value_or(Tensor()), residual = residual_in.value_or(Tensor());
    ctx->save_for_backward({seed_at});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["dtype"] = x.scalar_type();
    ctx->saved_data["residual"] = residual.defined();
    return dropout_apply(x, p, seed, seed_at, offset, residual);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    refuse_foreign_accumulators("dropout", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    if (ctx->needs_input_grad(0)) {
      const at::NoGradGuard no_grad;
      out[0] = dropout_apply(grads[0].to(ctx->saved_data["dtype"].toScalarType()), ctx->saved_data["p"].toDouble(),
                             ctx->saved_data["seed"].toInt(), s[0], ctx->saved_data["offset"].toInt(), Tensor());
    }
    if (out[0].defined()) out[0] = once({out[0]}, grads[0])[0];
    if (ctx->saved_data["residual"].toBool()) out[5] = grads[0];
    return out;
  }
};

Tensor dropout(const Tensor& x, double p, int64_t seed, const std::optional<Tensor>& seed_at_in, int64_t offset,
               const std::optional<Tensor>& residual_in) {
  const pybind11::gil_scoped_release no_gil;
  const Tensor seed_at = seed_at_in.value_or(Tensor()), residual = residual_in.value_or(Tensor());
  refuse_tangents("dropout", {&x, &residual});
  if (at::GradMode::is_enabled() && (x.requires_grad() || (residual.defined() && residual.requires_grad())))
    return Dropout::apply(x, p, seed, seed_at_in, offset, residual_in);
  const at::AutoDispatchBelowADInplaceOrView below;
  return dropout_apply(x, p, seed, seed_at, offset, residual);
}

pybind11::object try_dropout(pybind11::handle x_in, double p, int64_t seed, pybind11::handle seed_at_in, int64_t offset,
                             pybind11::handle residual_in) {
  Tensor x, seed_at, residual;
  if (!plain(x_in, x) || !plain(seed_at_in, seed_at, true) || !plain(residual_in, residual, true) || watched())
    return pybind11::none();
  if (!dropout_agrees(x, residual, seed_at) || !(p >= 0.0 && p <= 1.0)) return pybind11::none();
  return pybind11::cast(dropout(x, p, seed, seed_at.defined() ? std::optional<Tensor>(seed_at) : std::nullopt, offset,
                                residual.defined() ? std::optional<Tensor>(residual) : std::nullopt));
}

Tensor or_none(const std::optional<Tensor>& t) { return t.value_or(Tensor()); }

}  // namespace

void define_operators(pybind11::module_& m) {
  m.def("init_operators", &init_operators);
  m.def("cross_attention", &cross_attention);
  m.def("try_cross_attention", &try_cross_attention);
  m.def("cross_attention_forward",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
           const std::optional<Tensor>& lengths, double scale, bool training) {
          const pybind11::gil_scoped_release no_gil;
          return attention_forward(q, k, v, or_none(mask), or_none(lengths), scale, training);
        });
  m.def("cross_attention_backward",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
           const std::optional<Tensor>& lengths, double scale, const Tensor& out, const Tensor& stats, const Tensor& grad) {
          const pybind11::gil_scoped_release no_gil;
          return attention_backward(q, k, v, or_none(mask), or_none(lengths), scale, out, stats, grad);
        });
  m.def("rotary", &rotary);
  m.def("try_rotary", &try_rotary);
  m.def("rotary_apply", &rotary_apply, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("dropout", &dropout);
  m.def("try_dropout", &try_dropout);
  m.def("dropout_apply", [](const Tensor& x, double p, int64_t seed, const std::optional<Tensor>& seed_at, int64_t offset,
                            const std::optional<Tensor>& residual) {
    const pybind11::gil_scoped_release no_gil;
    return dropout_apply(x, p, seed, or_none(seed_at), offset, or_none(residual));
  });
}
