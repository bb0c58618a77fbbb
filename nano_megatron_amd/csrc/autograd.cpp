// Autograd nodes of the operators whose kernels take less time than an autograd Function in
// Python does: layer norm and rotary positions.
//
// A training call of these kernels is some tens of microseconds on the GPU.  A node in Python
// spends 38 us in the backward alone (8192 x 768 with residual: the kernels 25), on the
// autograd thread and under the interpreter's lock; these spend 12, and the checks of a call
// 2 instead of 6.  They call the C ABI of include/nmb.h as the Python bindings do, on the
// tensors' device and its current stream, with workspaces of torch's allocator.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <array>
#include <cmath>

#include "../../include/nmb.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status, const char* what) {
  if (status == NMB_OK) return;
  // as the Python bindings raise: bad arguments are ValueErrors
  TORCH_CHECK_VALUE(status != NMB_EINVAL && status != NMB_EUNSUPPORTED, what, ": ", nmb_last_error());
  TORCH_CHECK(false, what, ": ", nmb_last_error());
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return NMB_BF16;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "nano_megatron_amd kernels support float32 and bfloat16, got ",
                    t.scalar_type());
  return NMB_F32;
}

void require_gpu(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "nano_megatron_amd runs its kernels on the GPU only; got a tensor on ", t.device(),
                    " (there is no CPU fallback)");
}

bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// Whether a node has to stand behind the call: a gradient is wanted, or a forward-mode tangent
// would be lost (the node raises for it).
template <class... T>
bool needs_node(const T&... t) {
  const bool wanted = at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
  return wanted || (has_tangent(t) || ...);
}

// The gradients that `compute` forms outside of any graph; differentiated themselves they raise,
// instead of leaving out what the kernels computed.
template <class F>
variable_list once_differentiable(const variable_list& grads, const F& compute) {
  bool again = false;
  if (at::GradMode::is_enabled())
    for (const Tensor& g : grads) again = again || (g.defined() && g.requires_grad());
  const at::AutoGradMode off(false);
  variable_list out = compute();
  if (!again) return out;
  const at::AutoGradMode on(true);
  variable_list fake;
  for (const Tensor& t : out)
    if (t.defined()) fake.push_back(t.detach().requires_grad_(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      static_cast<int64_t>(fake.size()));
  fake = (*error)(std::move(fake));
  size_t n = 0;
  for (Tensor& t : out)
    if (t.defined()) t = fake[n++];
  return out;
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Tensors that may be missing: undefined here, and std::optional where a node takes them (it has
// no input, and so no place among those that needs_input_grad counts, for a missing one).
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

Tensor new_empty(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }

// ------------------------------------------------------------------ layer norm
// [rows, cols] with contiguous rows, copied only where the memory has none
Tensor rows_of(const Tensor& t, int64_t cols) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  return r.stride(1) == 1 || cols == 1 ? r : r.contiguous();
}

struct NormResult {
  Tensor y, h, rows, stats;  // h: the sum with the residual; rows: what was normalised
};

NormResult norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps,
                        bool keep) {
  const int64_t cols = weight.size(0);
  const Tensor x2 = rows_of(x, cols), r2 = residual.defined() ? rows_of(residual, cols) : Tensor();
  const int64_t rows = x2.size(0);
  NormResult out;
  out.y = new_empty(x.sizes(), x);
  if (r2.defined()) out.h = new_empty(x.sizes(), x);
  if (keep) out.stats = at::empty({2 * rows}, x.options().dtype(at::kFloat));
  check(nmb_layernorm_fwd(data(x2), x2.stride(0), data(r2), r2.defined() ? r2.stride(0) : 0, data(weight), data(bias),
                          data(out.y), data(out.h), static_cast<float*>(data(out.stats)), rows, cols,
                          static_cast<float>(eps), dtype_code(x), stream_of(x)),
        "nmb_layernorm_fwd");
  out.rows = out.h.defined() ? out.h : x2;
  return out;
}

// Saves what was normalised and a mean and a reciprocal deviation per row.
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias,
                               const Maybe& residual, double eps) {
    const NormResult r = norm_forward(x, weight, bias.value_or(Tensor()), residual.value_or(Tensor()), eps, true);
    ctx->save_for_backward({r.rows, weight, r.stats});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return r.h.defined() ? variable_list{r.y, r.h} : variable_list{r.y};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return once_differentiable(grads, [&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1),
               want_b = bias && ctx->needs_input_grad(2), want_r = residual && ctx->needs_input_grad(2 + bias);
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined()) {  // only the sum was used
      const Tensor zero_w = want_w && dh.defined() ? at::zeros_like(saved[1]) : Tensor();
      const Tensor zero_b = want_b && dh.defined() ? at::zeros_like(saved[1]) : Tensor();
      return {want_x ? dh : Tensor(), zero_w, zero_b, want_r ? dh : Tensor(), Tensor()};
    }
    // saved-tensor hooks may hand back tensors of another layout
    const Tensor weight = saved[1].contiguous(), stats = saved[2].contiguous();
    const int64_t cols = weight.size(0);
    const c10::OptionalDeviceGuard guard(weight.device());
    const Tensor h2 = rows_of(saved[0], cols), dy2 = rows_of(dy, cols), dh2 = dh.defined() ? rows_of(dh, cols) : Tensor();
    const int64_t rows = h2.size(0);
    const int code = dtype_code(weight);
    const Tensor dx = new_empty(ctx->saved_data["sizes"].toIntVector(), weight);
    Tensor sums, ws;
    size_t bytes = 0;
    if (want_w || want_b) {
      sums = new_empty({2, cols}, weight);
      check(nmb_layernorm_bwd_workspace_bytes(rows, cols, code, &bytes), "nmb_layernorm_bwd_workspace_bytes");
      ws = at::empty({static_cast<int64_t>(bytes)}, weight.options().dtype(at::kByte));
    }
    const Tensor dw = want_w ? sums.select(0, 0) : Tensor(), db = want_b ? sums.select(0, 1) : Tensor();
    check(nmb_layernorm_bwd(data(h2), h2.stride(0), static_cast<const float*>(data(stats)), data(weight), data(dy2),
                            dy2.stride(0), data(dh2), dh2.defined() ? dh2.stride(0) : 0, data(dx), data(dw), data(db),
                            data(ws), bytes, rows, cols, code, stream_of(weight)),
          "nmb_layernorm_bwd");
    return {want_x ? dx : Tensor(), dw, db, want_r ? dx : Tensor(), Tensor()};
  }
};

py::object layer_norm(const Tensor& x, const Tensor& weight_in, const Maybe& bias_in,
                      const Maybe& residual_in, double eps) {
  const Tensor bias_any = bias_in.value_or(Tensor()), residual = residual_in.value_or(Tensor());
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight_in.dim() == 1 && weight_in.size(0) == x.size(-1) && weight_in.size(0) >= 1,
                    "expected the last dimension to be that of the weight ", weight_in.sizes(), ", got ", x.sizes());
  TORCH_CHECK_VALUE(!bias_any.defined() || bias_any.sizes() == weight_in.sizes(), "bias ", bias_any.sizes(),
                    " does not match the weight ", weight_in.sizes());
  TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == x.sizes(), "residual ", residual.sizes(),
                    " does not match x ", x.sizes());
  TORCH_CHECK_VALUE(eps > 0 && std::isfinite(eps), "eps must be positive and finite, got ", eps);
  for (const Tensor& t : {weight_in, bias_any, residual})
    TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == x.scalar_type() && t.device() == x.device()),
                      "x, weight, bias and residual must have one dtype and one device, got ", x.scalar_type(), " on ",
                      x.device(), " and ", t.scalar_type(), " on ", t.device());
  require_gpu(x);
  variable_list out;
  {
    const py::gil_scoped_release release;
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor weight = weight_in.contiguous(), bias = bias_any.defined() ? bias_any.contiguous() : bias_any;
    if (needs_node(x, weight, bias, residual)) {
      out = LayerNorm::apply(x, weight, maybe(bias), maybe(residual), eps);
    } else {
      NormResult r = norm_forward(x, weight, bias, residual, eps, false);
      out.push_back(std::move(r.y));
      if (r.h.defined()) out.push_back(std::move(r.h));
    }
  }
  if (out.size() == 1) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

// ------------------------------------------------------------------ rotary positions
struct RotaryMeta {
  int64_t offset;
  bool interleaved;
  double magnitude;
};

std::array<int64_t, 3> strides_of(const Tensor& t) {  // (batch, token, head) of [B, H, S, D]
  return {t.stride(0), t.stride(2), t.stride(1)};
}

Tensor head_rows(const Tensor& t) {
  return t.stride(3) == 1 || t.size(3) == 1 ? t : t.transpose(1, 2).contiguous().transpose(1, 2);
}

// q and k, either undefined, rotated into new [B, S, H, D] memory
std::array<Tensor, 2> rotate(const Tensor& q, const Tensor& k, const Tensor& frequencies, const Tensor& positions,
                             const Tensor& offsets, const RotaryMeta& meta, bool inverse) {
  const Tensor& first = q.defined() ? q : k;
  const int64_t b = first.size(0), s = first.size(2), d = first.size(3);
  std::array<Tensor, 2> in, out;
  std::array<std::array<int64_t, 3>, 2> is{}, os{};
  std::array<int64_t, 2> heads{};
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = i == 0 ? q : k;
    if (!t.defined()) continue;
    in[i] = head_rows(t);
    heads[i] = t.size(1);
    out[i] = at::empty_strided({b, heads[i], s, d}, {s * heads[i] * d, d, heads[i] * d, 1}, t.options());
    is[i] = strides_of(in[i]);
    os[i] = strides_of(out[i]);
  }
  int64_t pos_b = 0, pos_s = 0;
  if (positions.defined()) {
    pos_s = positions.stride(-1);
    pos_b = positions.dim() == 2 ? positions.stride(0) : 0;
  }
  check(nmb_rotary(data(in[0]), is[0].data(), data(out[0]), os[0].data(), heads[0], data(in[1]), is[1].data(),
                   data(out[1]), os[1].data(), heads[1], static_cast<const double*>(data(frequencies)),
                   2 * frequencies.size(0), data(positions),
                   positions.defined() ? static_cast<int>(positions.element_size()) : 4, pos_b, pos_s,
                   static_cast<const int32_t*>(data(offsets)), meta.offset, b, s, d, meta.interleaved, inverse,
                   static_cast<float>(meta.magnitude), dtype_code(first), stream_of(first)),
        "nmb_rotary");
  return out;
}

// The backward turns by the negative angles; saves the frequencies and positions.
struct RotaryPositions : torch::autograd::Function<RotaryPositions> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k_in, const Tensor& frequencies,
                               const Maybe& positions_in, const Maybe& offsets_in, int64_t offset, bool interleaved,
                               double magnitude) {
    const Tensor k = k_in.value_or(Tensor()), positions = positions_in.value_or(Tensor()),
                 offsets = offsets_in.value_or(Tensor());
    ctx->save_for_backward({frequencies, positions, offsets});
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->set_materialize_grads(false);
    const auto out = rotate(q, k, frequencies, positions, offsets, RotaryMeta{offset, interleaved, magnitude}, false);
    return k.defined() ? variable_list{out[0], out[1]} : variable_list{out[0]};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return once_differentiable(grads, [&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(8);
    const Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor();
    const Tensor gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    if (!gq.defined() && !gk.defined()) return out;
    const c10::OptionalDeviceGuard guard(saved[0].device());
    const RotaryMeta meta{ctx->saved_data["offset"].toInt(), ctx->saved_data["interleaved"].toBool(),
                          ctx->saved_data["magnitude"].toDouble()};
    const auto turned = rotate(gq, gk, saved[0].contiguous(), saved[1], saved[2].defined() ? saved[2].contiguous() : saved[2],
                               meta, true);
    out[0] = turned[0];
    out[1] = turned[1];
    return out;
  }
};

py::object rotary_positions(const Tensor& q, const Maybe& k_in, const Tensor& frequencies_in,
                            const Maybe& positions_in, const Maybe& offsets_in,
                            int64_t offset, bool interleaved, double magnitude) {
  const Tensor k = k_in.value_or(Tensor()), positions = positions_in.value_or(Tensor());
  TORCH_CHECK_VALUE(q.dim() == 4 && (!k.defined() || k.dim() == 4),
                    "q and k must have [batch, heads, sequence, head_dim] shape");
  const int64_t b = q.size(0), s = q.size(2), d = q.size(3);
  if (k.defined()) {
    TORCH_CHECK_VALUE(k.size(0) == b && k.size(2) == s && k.size(3) == d, "q ", q.sizes(), " and k ", k.sizes(),
                      " must agree in all but their heads");
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.device() == q.device(),
                      "q and k must have one dtype and one device");
  }
  TORCH_CHECK_VALUE(frequencies_in.scalar_type() == at::kDouble && frequencies_in.dim() == 1 &&
                        frequencies_in.size(0) >= 1 && 2 * frequencies_in.size(0) <= d,
                    "frequencies must be a float64 [pairs] tensor of up to ", d / 2, " pairs, got ",
                    frequencies_in.scalar_type(), " ", frequencies_in.sizes());
  TORCH_CHECK_VALUE(!(frequencies_in.requires_grad() && at::GradMode::is_enabled()) && !has_tangent(frequencies_in),
                    "frequencies get no gradient; pass them detached");
  TORCH_CHECK_VALUE(std::isfinite(magnitude) && std::fabs(magnitude) <= 1e30,
                    "magnitude must be finite and within 1e30, got ", magnitude);
  require_gpu(q);
  TORCH_CHECK_VALUE(frequencies_in.device() == q.device(), "frequencies must be on the queries' device ", q.device(),
                    ", got ", frequencies_in.device());
  TORCH_CHECK_VALUE(offset >= -(int64_t{1} << 40) && offset <= (int64_t{1} << 40),
                    "sequence_offset must lie within 2^40 of 0, got ", offset);
  if (offsets_in.has_value())
    TORCH_CHECK_VALUE(offsets_in->scalar_type() == at::kInt && offsets_in->dim() == 1 && offsets_in->size(0) == b &&
                          offsets_in->device() == q.device(),
                      "sequence_offset must be an int32 [", b, "] tensor on the query's device, got ",
                      offsets_in->scalar_type(), " ", offsets_in->sizes(), " on ", offsets_in->device());
  if (positions.defined()) {
    TORCH_CHECK_VALUE(!offsets_in.has_value() && offset == 0, "positions and a sequence_offset exclude each other");
    const bool shape = (positions.dim() == 1 && positions.size(0) == s) ||
                       (positions.dim() == 2 && positions.size(0) == b && positions.size(1) == s);
    TORCH_CHECK_VALUE(shape && (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
                          positions.device() == q.device(),
                      "positions must be an integer [", s, "] or [", b, ", ", s, "] tensor on the queries' device, got ",
                      positions.scalar_type(), " ", positions.sizes(), " on ", positions.device());
  }
  std::array<Tensor, 2> out;
  {
    const py::gil_scoped_release release;
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor frequencies = frequencies_in.contiguous(), offsets = offsets_in.has_value() ? offsets_in->contiguous() : Tensor();
    if (needs_node(q, k)) {
      const variable_list r = RotaryPositions::apply(q, maybe(k), frequencies, maybe(positions), maybe(offsets), offset,
                                                     interleaved, magnitude);
      out[0] = r[0];
      if (r.size() > 1) out[1] = r[1];
    } else {
      out = rotate(q, k, frequencies, positions, offsets, RotaryMeta{offset, interleaved, magnitude}, false);
    }
  }
  if (!k.defined()) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("rotary_positions", &rotary_positions);
  m.def("abi_version", &nmb_abi_version);
}
