// Autograd nodes of the operators whose kernels can take less time than an autograd Function in
// Python does: layer norm, rotary positions, the head's loss against a teacher.
//
// A training call of these kernels is some tens of microseconds on the GPU.  A node in Python
// spends 38 us in the backward alone (8192 x 768 with residual: the kernels 25), on the
// autograd thread and under the interpreter's lock; these spend 12, and the checks of a call
// 2 instead of 6.  They call the C ABI of include/nmb.h as the Python bindings do, on the
// tensors' device and its current stream, with workspaces of torch's allocator.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <algorithm>
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

// The gradients that `compute` forms outside of any graph.  Where they are differentiated
// themselves they raise, instead of leaving out what the kernels computed: the purpose and the message
// of torch's Python decorator once_differentiable.  That looks at the incoming gradients alone and
// raises only where nothing else is asked for; these depend on the node's inputs too (but where
// they are `linear`: in the incoming gradients, and in nothing else), so the error stands between
// them and both, on the way to whatever is differentiated by.
template <class F>
variable_list once_differentiable(const variable_list& grads, bool linear, const F& compute) {
  torch::autograd::edge_list edges;
  bool again = false;
  if (at::GradMode::is_enabled()) {
    for (const Tensor& g : grads) again = again || (g.defined() && g.requires_grad());
    if (again) edges = torch::autograd::collect_next_edges(grads);
    if (!linear) {
      again = true;
      const auto& own = torch::autograd::get_current_node()->next_edges();
      edges.insert(edges.end(), own.begin(), own.end());
    }
  }
  const at::AutoGradMode off(false);
  variable_list out = compute();
  if (!again) return out;
  const auto error = std::make_shared<torch::autograd::Error>(
      "trying to differentiate twice a function that was marked with @once_differentiable", std::move(edges));
  for (Tensor& t : out)
    if (t.defined()) {
      t = t.detach();  // (one of them may stand in two places)
      torch::autograd::set_history(t, error);
    }
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
    if (!grads[0].defined()) return gradients(ctx, grads);  // the sum's own, as it came in
    return once_differentiable(grads, false, [&] { return gradients(ctx, grads); });
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
    Tensor dw, db, ws;
    size_t bytes = 0;
    if (want_w) dw = new_empty({cols}, weight);
    if (want_b) db = new_empty({cols}, weight);
    if (want_w || want_b) {
      check(nmb_layernorm_bwd_workspace_bytes(rows, cols, code, &bytes), "nmb_layernorm_bwd_workspace_bytes");
      ws = at::empty({static_cast<int64_t>(bytes)}, weight.options().dtype(at::kByte));
    }
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
    return once_differentiable(grads, true, [&] { return gradients(ctx, grads); });
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

// ------------------------------------------------------------------ the head against a teacher
// The embedding's TiedGrad, to which the table's gradient goes; a Python object.
struct Tie : torch::CustomClassHolder {
  py::object tie;
  explicit Tie(py::object t) : tie(std::move(t)) {}
  ~Tie() override {
    const py::gil_scoped_acquire gil;
    tie = py::object();
  }
};
using TiePtr = c10::intrusive_ptr<Tie>;

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

enum Reduction : int64_t { kNone, kSum, kMean };

struct DistillMeta {
  int64_t chunk, ignore_index;
  double temperature, weight;
  int64_t reduction;
};

// The teacher of the rows from `first` on.
nmb_teacher teacher_at(const Tensor& values, const Tensor& ids, const Tensor& targets, int64_t first, const DistillMeta& m) {
  nmb_teacher t{};
  t.ld = values.stride(0);
  t.ldi = ids.stride(0);
  t.logits = static_cast<const char*>(data(values)) + values.element_size() * t.ld * first;
  t.ids = static_cast<const char*>(data(ids)) + ids.element_size() * t.ldi * first;
  t.targets = targets.defined() ? static_cast<const int64_t*>(data(targets)) + first : nullptr;
  t.ignore_index = m.ignore_index;
  t.top = values.size(1);
  t.logits_dtype = dtype_code(values);
  t.id_bytes = static_cast<int>(ids.element_size());
  t.temperature = static_cast<float>(m.temperature);
  t.target_weight = static_cast<float>(m.weight);
  return t;
}

Tensor workspace(int64_t bytes, const Tensor& like) {
  return at::empty({std::max<int64_t>(bytes, 16)}, like.options().dtype(at::kByte));
}

template <class F, class... Args>
int64_t bytes_of(const F& query, const char* what, Args... args) {
  int64_t bytes = 0;
  check(query(args..., &bytes), what);
  return bytes;
}

// use(first row, rows) for the one or two calls that a bf16 product of m rows takes
template <class F>
void in_calls(int la, int lb, int64_t m, int64_t n, int64_t k, const F& use) {
  const int64_t first = bytes_of(nmb_gemm_bf16_first_rows, "nmb_gemm_bf16_first_rows", la, lb, m, n, k);
  if (first > 0) use(int64_t{0}, first);
  use(first, m - first);
}

int64_t gemm_f32_bytes(int64_t m, int64_t n, int64_t k) {
  return bytes_of(nmb_gemm_f32_workspace_bytes, "nmb_gemm_f32_workspace_bytes", m, n, k);
}

// Row-major fp32 products: a [m, k] or, transposed, [k, m]; b [n, k] or, plain, [k, n].
void gemm_f32(int la, int lb, int64_t m, int64_t n, int64_t k, const float* a, int64_t lda, const float* b, int64_t ldb,
              float beta, float* d, const Tensor& ws, hipStream_t stream) {
  check(nmb_gemm_f32_split(la, lb, m, n, k, 1.f, a, lda, b, ldb, beta, beta != 0.f ? d : nullptr, n, d, n, data(ws),
                           ws.numel(), stream),
        "nmb_gemm_f32_split");
}

struct DistillResult {
  Tensor loss, stats, picked;
  Tensor total, over;  // of "sum" and "mean": the result, and what it was divided by
  const Tensor& result() const { return total.defined() ? total : loss; }
};

// The losses of the rows
DistillResult distill_rows(const Tensor& x, const Tensor& weight, const Tensor& values, const Tensor& ids,
                              const Tensor& targets, const DistillMeta& m) {
  const int64_t rows = x.size(0), hidden = x.size(1), vocab = weight.size(0);
  const int64_t entries = values.size(1) + targets.defined();
  const auto f32 = x.options().dtype(at::kFloat);
  DistillResult out{at::empty({rows}, f32), at::empty({4, rows}, f32), at::empty({rows, entries}, f32)};
  if (rows == 0) return out;
  const hipStream_t stream = stream_of(x);
  const int code = dtype_code(x);
  float *loss = out.loss.data_ptr<float>(), *stats = out.stats.data_ptr<float>(), *picked = out.picked.data_ptr<float>();
  const auto own_bytes = [&](int64_t n) {
    return bytes_of(nmb_distill_workspace_bytes, "nmb_distill_workspace_bytes", n, vocab, code);
  };
  if (code == NMB_BF16) {
    const Tensor ws = workspace(own_bytes(rows), x);
    const nmb_teacher t = teacher_at(values, ids, targets, 0, m);
    check(nmb_distill_fwd(data(x), hidden, data(weight), hidden, rows, vocab, hidden, &t, loss, stats, rows, picked,
                          data(ws), ws.numel(), stream),
          "nmb_distill_fwd");
    return out;
  }
  const float *xp = x.data_ptr<float>(), *wp = weight.data_ptr<float>();
  const Tensor buf = at::empty({std::min(m.chunk, rows), vocab}, f32);
  for (int64_t s = 0; s < rows; s += m.chunk) {
    const int64_t n = std::min(m.chunk, rows - s);
    const Tensor ws = workspace(std::max(gemm_f32_bytes(n, vocab, hidden), own_bytes(n)), x);
    gemm_f32(0, 0, n, vocab, hidden, xp + hidden * s, hidden, wp, hidden, 0.f, buf.data_ptr<float>(), ws, stream);
    const nmb_teacher t = teacher_at(values, ids, targets, s, m);
    check(nmb_distill_rows_fwd(buf.data_ptr<float>(), vocab, n, vocab, &t, loss + s, stats + s, rows, picked + entries * s,
                               data(ws), ws.numel(), stream),
          "nmb_distill_rows_fwd");
  }
  return out;
}

DistillResult distill_forward(const Tensor& x, const Tensor& weight, const Tensor& values, const Tensor& ids,
                              const Tensor& targets, const DistillMeta& m) {
  DistillResult out = distill_rows(x, weight, values, ids, targets, m);
  if (m.reduction == kNone) return out;
  out.total = at::empty({}, out.loss.options());
  out.over = at::empty({}, out.loss.options());
  const int64_t rows = x.size(0);
  const int64_t bytes = bytes_of(nmb_distill_total_workspace_bytes, "nmb_distill_total_workspace_bytes", rows);
  const Tensor ws = bytes ? workspace(bytes, x) : Tensor();
  check(nmb_distill_total(static_cast<const float*>(data(out.loss)), static_cast<const float*>(data(out.stats)), rows,
                          static_cast<const int64_t*>(data(targets)), m.ignore_index, rows, m.reduction == kMean,
                          out.total.data_ptr<float>(), out.over.data_ptr<float>(), data(ws), bytes, stream_of(x)),
        "nmb_distill_total");
  return out;
}

// The logits are formed once for the loss and again for their gradient G, a chunk of rows at a
// time (bf16: the forward in one go), then dx = G W and dW = G^T x, added up over the chunks.
// Saves four numbers of each row and the logits of its entries, and what a mean divides by.
struct Distillation : torch::autograd::Function<Distillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& values,
                        const Tensor& ids, const Maybe& targets, int64_t chunk, int64_t ignore_index, double temperature,
                        double target_weight, int64_t reduction, const TiePtr& tie) {
    const Tensor t = targets.value_or(Tensor());
    const DistillResult r = distill_forward(
        x, weight, values, ids, t, DistillMeta{chunk, ignore_index, temperature, target_weight, reduction});
    ctx->save_for_backward({x, weight, values, ids, t, r.stats, r.picked, r.over});
    ctx->saved_data["chunk"] = chunk;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["target_weight"] = target_weight;
    ctx->saved_data["reduction"] = reduction;
    if (tie) ctx->saved_data["tie"] = c10::IValue::make_capsule(tie);
    return r.result();
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return once_differentiable(grads, false, [&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list saved = ctx->get_saved_variables();
    // saved-tensor hooks may hand back tensors of another layout
    for (Tensor& t : saved)
      if (t.defined()) t = t.contiguous();
    const Tensor &x = saved[0], &weight = saved[1], &values = saved[2], &ids = saved[3], &targets = saved[4],
                 &stats_t = saved[5], &picked_t = saved[6];
    auto& meta = ctx->saved_data;
    DistillMeta m{meta["chunk"].toInt(), meta["ignore_index"].toInt(), meta["temperature"].toDouble(),
                  meta["target_weight"].toDouble(), meta["reduction"].toInt()};
    const bool tied = meta.count("tie") != 0;
    const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1) || tied;
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t rows = x.size(0), hidden = x.size(1), vocab = weight.size(0), entries = picked_t.size(1);
    Tensor up = grads[0].to(at::kFloat);
    if (m.reduction == kMean) up = up / saved[7];
    up = up.expand({rows}).contiguous();
    const bool bf16 = x.scalar_type() == at::kBFloat16;
    const int64_t cols = bf16 ? round8(vocab) : vocab, size = bf16 ? 2 : 4;
    // of dw's product: 32-bit byte offsets into the chunk's gradients and hidden states
    if (bf16) m.chunk = std::max<int64_t>(1, std::min(m.chunk, ((int64_t{1} << 30) - 1) / std::max(cols, hidden)));
    // one chunk writes the table gradient rounded; several add it up in fp32 first
    const bool several = rows > m.chunk;
    Tensor dx, dw, buf, kept;
    if (want_dx) dx = at::empty_like(x);
    if (want_dw) {
      const auto options = weight.options().dtype(several ? at::kFloat : weight.scalar_type());
      dw = rows ? at::empty({cols, hidden}, options) : at::zeros({cols, hidden}, options);
    }
    if (rows) buf = new_empty({std::min(m.chunk, rows), cols}, x);
    // the chunk's x without the rows that have no part, for dw
    if (rows && want_dw) kept = new_empty({std::min(m.chunk, rows), hidden}, x);
    const hipStream_t stream = stream_of(x);
    const float *stats = stats_t.data_ptr<float>(), *picked = picked_t.data_ptr<float>(), *g_up = up.data_ptr<float>();
    void* g = data(buf);
    for (int64_t s = 0; s < rows; s += m.chunk) {
      const int64_t n = std::min(m.chunk, rows - s);
      char* xs = static_cast<char*>(data(x)) + size * hidden * s;
      char* dxs = want_dx ? static_cast<char*>(data(dx)) + size * hidden * s : nullptr;
      const float beta = s == 0 ? 0.f : 1.f;
      const nmb_teacher t = teacher_at(values, ids, targets, s, m);
      if (bf16) {
        int64_t ws_bytes = 0;
        if (want_dx)
          in_calls(0, 1, n, hidden, vocab, [&](int64_t, int64_t count) {
            ws_bytes = std::max(ws_bytes, bytes_of(nmb_head_loss_dx_workspace_bytes, "nmb_head_loss_dx_workspace_bytes",
                                                   count, vocab, hidden, hidden));
          });
        if (want_dw)
          in_calls(1, 1, cols, hidden, n, [&](int64_t, int64_t count) {
            ws_bytes = std::max(ws_bytes, bytes_of(nmb_gemm_bf16_workspace_bytes, "nmb_gemm_bf16_workspace_bytes", 1, 1,
                                                   count, hidden, n));
          });
        const Tensor ws = workspace(ws_bytes, x);
        check(nmb_distill_grad(xs, hidden, data(weight), hidden, n, vocab, hidden, &t, stats + s, rows,
                               picked + entries * s, g_up + s, g, cols, data(kept), stream),
              "nmb_distill_grad");
        auto* gb = static_cast<at::BFloat16*>(g);
        if (want_dx)
          in_calls(0, 1, n, hidden, vocab, [&](int64_t at, int64_t count) {
            check(nmb_head_loss_dx(gb + at * cols, cols, data(weight), hidden, count, vocab, hidden,
                                   reinterpret_cast<at::BFloat16*>(dxs) + at * hidden, hidden, data(ws), ws.numel(), stream),
                  "nmb_head_loss_dx");
          });
        if (want_dw)
          in_calls(1, 1, cols, hidden, n, [&](int64_t at, int64_t count) {
            if (several)
              check(nmb_gemm_bf16_f32out(1, 1, count, hidden, n, 1.f, gb + at, cols, data(kept), hidden, beta,
                                         dw.data_ptr<float>() + at * hidden, hidden, data(ws), ws.numel(), stream),
                    "nmb_gemm_bf16_f32out");
            else
              check(nmb_gemm_bf16(1, 1, count, hidden, n, 1.f, gb + at, cols, data(kept), hidden, 0.f, nullptr, hidden,
                                  dw.data_ptr<at::BFloat16>() + at * hidden, hidden, data(ws), ws.numel(), stream),
                    "nmb_gemm_bf16");
          });
      } else {
        float *gf = static_cast<float*>(g), *xf = reinterpret_cast<float*>(xs), *wf = weight.data_ptr<float>();
        const Tensor ws = workspace(std::max({gemm_f32_bytes(n, vocab, hidden), gemm_f32_bytes(n, hidden, vocab),
                                              gemm_f32_bytes(vocab, hidden, n)}), x);
        gemm_f32(0, 0, n, vocab, hidden, xf, hidden, wf, hidden, 0.f, gf, ws, stream);
        float* kf = static_cast<float*>(data(kept));
        check(nmb_distill_rows_grad(gf, vocab, n, vocab, &t, stats + s, rows, picked + entries * s, g_up + s, xf, hidden,
                                    hidden, kf, stream),
              "nmb_distill_rows_grad");
        if (want_dx) gemm_f32(0, 1, n, hidden, vocab, gf, vocab, wf, hidden, 0.f, reinterpret_cast<float*>(dxs), ws, stream);
        if (want_dw) gemm_f32(1, 1, vocab, hidden, n, gf, vocab, kf, hidden, beta, dw.data_ptr<float>(), ws, stream);
      }
    }
    if (want_dw) {
      if (cols != vocab) dw = dw.narrow(0, 0, vocab);
      dw = dw.to(weight.scalar_type());
    }
    if (tied) {  // the embedding's backward adds it to its own gradient
      const py::gil_scoped_acquire gil;
      static_cast<Tie*>(meta["tie"].toCapsule().get())->tie.attr("put")(dw);
      dw = Tensor();
    }
    variable_list out(11);
    out[0] = dx;
    out[1] = dw;
    return out;
  }
};

void check_distillation(const Tensor& hidden, const Tensor& weight, const Tensor& values, const Tensor& ids,
                        const Maybe& targets, double temperature, double target_weight) {
  TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.scalar_type() == weight.scalar_type() &&
                        hidden.size(-1) == weight.size(1),
                    "hidden ", hidden.sizes(), " ", hidden.scalar_type(), " and weight ", weight.sizes(), " ",
                    weight.scalar_type(), " must have one dtype and one hidden size");
  const auto is_int = [](const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; };
  TORCH_CHECK_VALUE((values.scalar_type() == at::kFloat || values.scalar_type() == at::kBFloat16) && is_int(ids),
                    "teacher_logits must be float32 or bfloat16 and teacher_ids int32 or int64, got ",
                    values.scalar_type(), " and ", ids.scalar_type());
  const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
  TORCH_CHECK_VALUE(values.sizes() == ids.sizes() && ids.dim() == hidden.dim() &&
                        ids.sizes().slice(0, ids.dim() - 1) == lead,
                    "teacher_logits ", values.sizes(), " and teacher_ids ", ids.sizes(), " must both be [..., K] for hidden ",
                    hidden.sizes());
  TORCH_CHECK_VALUE(ids.size(-1) >= 1 && ids.size(-1) <= 1024, "1 to 1024 teacher logits a token, got ", ids.size(-1));
  TORCH_CHECK_VALUE(!targets.has_value() || (targets->sizes() == lead && is_int(*targets)),
                    "targets must be integers that match hidden ", hidden.sizes(), " in all but the last dimension");
  TORCH_CHECK_VALUE(temperature >= 1e-2 && temperature <= 1e2, "temperature must lie within 0.01 and 100, got ", temperature);
  TORCH_CHECK_VALUE(target_weight >= 0 && target_weight <= 1e30, "target_weight must lie within 0 and 1e30, got ",
                    target_weight);
  TORCH_CHECK_VALUE(!(values.requires_grad() && at::GradMode::is_enabled()) && !has_tangent(values),
                    "teacher_logits get no gradient; pass them detached");
  TORCH_CHECK_VALUE(hidden.scalar_type() != at::kBFloat16 || hidden.size(-1) % 8 == 0,
                    "the head in bf16 needs a hidden size that is a multiple of 8, got ", hidden.size(-1));
  for (const Tensor& t : {weight, values, ids, targets.value_or(weight)})
    TORCH_CHECK_VALUE(t.device() == hidden.device(), "hidden, weight, the teacher and targets must be on one device, got ",
                      hidden.device(), " and ", t.device());
  require_gpu(hidden);
}

Tensor lm_head_distillation(const Tensor& hidden, const Tensor& weight, const Tensor& values_in, const Tensor& ids_in,
                            const Maybe& targets_in, double temperature, double target_weight, int64_t ignore_index,
                            std::optional<int64_t> chunk_in, const py::object& tie_in, const std::string& reduction_name) {
  check_distillation(hidden, weight, values_in, ids_in, targets_in, temperature, target_weight);
  TORCH_CHECK_VALUE(chunk_in.value_or(1) >= 1, "chunk must be at least 1, got ", chunk_in.value_or(1));
  const TiePtr tie = tie_in.is_none() ? TiePtr() : c10::make_intrusive<Tie>(tie_in);
  const py::gil_scoped_release release;
  const c10::OptionalDeviceGuard guard(hidden.device());
  const int64_t vocab = weight.size(0), top = ids_in.size(-1);
  const bool bf16 = hidden.scalar_type() == at::kBFloat16;
  if (at::GradMode::is_enabled()) {  // what the gradients' products cannot address
    TORCH_CHECK_VALUE(!(bf16 && hidden.requires_grad() && round8(vocab) >= (1 << 22)),
                      "the gradient of the hidden states in bf16 needs a vocabulary below 2^22, got ", vocab);
    TORCH_CHECK_VALUE(bf16 || !(weight.requires_grad() || tie) || vocab <= 65535 * 64,
                      "the gradient of the table in fp32 needs a vocabulary of at most ", 65535 * 64, ", got ", vocab);
  }
  // 16-byte rows need a 16-byte start, which a contiguous view may lack
  const auto dense = [](const Tensor& t) {
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
  };
  const Tensor x = dense(hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)})), w = dense(weight);
  const Tensor values = rows_of(values_in, top), ids = rows_of(ids_in, top);
  const Tensor targets = targets_in.has_value() ? targets_in->reshape({-1}).to(at::kLong).contiguous() : Tensor();
  // rows whose gradients are in memory at a time; bf16: what 1 GiB holds, in whole 256-row tiles
  // (and no more than a launch takes)
  const int64_t chunk = std::min(int64_t{1} << 21, chunk_in.value_or(
      bf16 ? std::max<int64_t>(256, (int64_t{1} << 30) / (2 * round8(vocab)) / 256 * 256) : 2048));
  const int64_t reduction = reduction_name == "none" ? kNone : reduction_name == "sum" ? kSum : kMean;
  const DistillMeta m{chunk, ignore_index, temperature, target_weight, reduction};
  const Tensor loss = needs_node(x, w) ? Distillation::apply(x, w, values, ids, maybe(targets), chunk, ignore_index,
                                                             temperature, target_weight, reduction, tie)
                                       : distill_forward(x, w, values, ids, targets, m).result();
  return hidden.dim() == 2 || reduction != kNone ? loss : loss.view(hidden.sizes().slice(0, hidden.dim() - 1));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("rotary_positions", &rotary_positions);
  m.def("check_distillation", &check_distillation);
  m.def("lm_head_distillation", &lm_head_distillation);
  m.attr("abi_version") = NMB_ABI_VERSION;  // of the header that these nodes follow
}
