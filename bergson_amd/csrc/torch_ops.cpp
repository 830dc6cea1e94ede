// The model operators as native autograd functions: argument checks, allocation, and the calls of the C ABI of
// include/bergson_amd.h, without the interpreter in either pass.
//
// A Python autograd function of the same calls took 114 us for a forward and backward pass of a small layer norm on
// an MI355X host, this takes 64, of which 40 are the engine's own (x * 2 and its gradient): the backward pass runs on
// the engine's thread, where every step of a Python function competes for the interpreter.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>

#include "bergson_amd.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t MAX_NORM_WIDTH = 16384;  // elements of a row the layer norm kernels hold
constexpr int64_t MAX_HEAD_DIM = 128;
constexpr int64_t MAX_TEACHER_ENTRIES = 1024;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BGX_F32;
    case at::kHalf: return BGX_F16;
    case at::kBFloat16: return BGX_BF16;
    default:
      C10_THROW_ERROR(TypeError, c10::str("unsupported dtype ", t, "; the kernels take float32, float16 and bfloat16"));
  }
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, ": ", bgx_last_error());
}

void need_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor: bergson_amd has no CPU path (got device ", t.device(), ")");
}

// The kernels form no tangents, and an output without one is a derivative of zero to forward mode.  A gradient recorded
// for the backward pass refuses by itself; a call that records none (frozen parameters, no_grad) would not.
void no_tangent(const Tensor& t, const char* name) {
  if (t.defined() && t._fw_grad(/*level=*/0).defined())
    C10_THROW_ERROR(NotImplementedError, c10::str(name, " carries a tangent: forward-mode derivatives are not supported"));
}

void same_device(const Tensor& ref, const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.device() == ref.device(), name, " lives on ", t.device(), ", the input on ", ref.device());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool wants_graph(std::initializer_list<Tensor> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// The kernels' results carry no graph: differentiating them again is an error, not a zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list live;
  for (Tensor& g : grads)
    if (g.defined()) live.push_back(g.detach().requires_grad_());
  if (live.empty()) return grads;
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "bergson_amd's operators are differentiable once", (int)live.size());
  variable_list marked = (*refuse)(std::move(live));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// [rows, d] with rows at least d elements apart and contiguous elements, copied only where x is not that
Tensor as_rows(const Tensor& x, int64_t d) {
  Tensor rows = x.dim() == 2 ? x : x.reshape({-1, d});
  if (x.numel() == 0) return rows;
  if ((d > 1 && rows.stride(1) != 1) || (rows.size(0) > 1 && rows.stride(0) < d)) rows = rows.contiguous();
  return rows;
}
int64_t row_stride(const Tensor& rows) { return std::max(rows.stride(0), rows.size(1)); }

// ---- layer norm -------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor& x, const Tensor& rows, const Tensor& weight, const Tensor& bias, double eps,
                    const Tensor& stats) {
  const int64_t n = rows.size(0), d = rows.size(1);
  Tensor y = at::empty(x.sizes(), x.options());
  float* mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
  check(bgx_layernorm_forward(ptr(rows), row_stride(rows), ptr(weight), ptr(bias), dtype_code(weight.scalar_type()), n,
                              (int32_t)d, dtype_code(x.scalar_type()), (float)eps, out_ptr(y), d, mean,
                              mean == nullptr ? nullptr : mean + n, stream_of(x)),
        "bgx_layernorm_forward");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight_in,
                        const optional<Tensor>& bias_in, double eps) {
    const Tensor rows = as_rows(x, x.size(-1)), weight = weight_in.contiguous();
    const Tensor bias = bias_in.has_value() ? bias_in->contiguous() : Tensor();
    const Tensor stats = at::empty({2, rows.size(0)}, x.options().dtype(at::kFloat));
    Tensor y = norm_forward(x, rows, weight, bias, eps, stats);
    ctx->save_for_backward({rows, weight, stats});
    ctx->saved_data["shape"] = x.sizes();
    ctx->saved_data["bias"] = bias.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &weight = saved[1], &stats = saved[2];
    const int64_t n = rows.size(0), d = rows.size(1);
    const c10::DeviceGuard guard(rows.device());
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), 
               want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    const Tensor dy = as_rows(grads[0], d);
    Tensor dx, dw, db, ws;
    if (want_x) dx = at::empty(ctx->saved_data["shape"].toIntVector(), rows.options());
    if (want_w) dw = at::empty({d}, weight.options());
    if (want_b) db = at::empty({d}, weight.options());
    size_t nbytes = 0;
    if (want_w || want_b) {
      nbytes = bgx_layernorm_backward_workspace_bytes(n, (int32_t)d);
      if (nbytes) ws = at::empty({(int64_t)nbytes}, rows.options().dtype(at::kByte));
    }
    const float* mean = stats.data_ptr<float>();
    check(bgx_layernorm_backward(ptr(dy), row_stride(dy), ptr(rows), row_stride(rows), ptr(weight),
                                 dtype_code(weight.scalar_type()), mean, mean + n, n, (int32_t)d,
                                 dtype_code(rows.scalar_type()), out_ptr(dx), d, out_ptr(dw), out_ptr(db), out_ptr(ws),
                                 nbytes, stream_of(rows)),
          "bgx_layernorm_backward");
    return once({dx, dw, db, Tensor()});
  }
};

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight_in, const optional<Tensor>& bias_in, double eps) {
  const int64_t d = x.dim() ? x.size(-1) : 0;
  dtype_code(x.scalar_type());
  TORCH_CHECK_VALUE(d >= 1 && d <= MAX_NORM_WIDTH, "layer_norm takes rows of 1 to ", MAX_NORM_WIDTH, " elements, got ",
                    x.sizes());
  TORCH_CHECK_VALUE(weight_in.has_value(), "layer_norm needs a weight");
  const Tensor weight = *weight_in, bias = bias_in.value_or(Tensor());
  auto vector = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == d, name, " ", t.sizes(), " does not match rows of ", d, " elements");
    TORCH_CHECK_TYPE((t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat) &&
                         t.scalar_type() == weight.scalar_type(),
                     name, " is ", t.scalar_type(), "; weight and bias share x's dtype (", x.scalar_type(),
                     ") or float32");
  };
  vector(weight, "weight");
  if (bias.defined()) vector(bias, "bias");
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < INFINITY, "eps=", eps, " must be finite and not negative");
  no_tangent(x, "x");
  no_tangent(weight, "weight");
  no_tangent(bias, "bias");
  need_gpu(x, "x");
  same_device(x, weight, "weight");
  if (bias.defined()) same_device(x, bias, "bias");
  const c10::DeviceGuard guard(x.device());
  if (wants_graph({x, weight, bias})) return LayerNorm::apply(x, weight, bias_in, eps);
  return norm_forward(x, as_rows(x, d), weight.contiguous(), bias.defined() ? bias.contiguous() : bias, eps, Tensor());
}

// ---- causal attention -------------------------------------------------------------------------------------------
// elements contiguous, positions ascending, apart, and at most 8 MiB so
bool direct(const Tensor& t) {
  const int64_t tok = t.stride(-3), dim = t.size(-1);
  return (dim == 1 || t.stride(-1) == 1) && (t.size(-3) == 1 || (tok >= dim && tok * t.element_size() <= (1 << 23)));
}
Tensor operand(const Tensor& t) { return direct(t) ? t : t.contiguous(); }

bgx_attention_rows rows_of(const Tensor& t) {
  const int64_t tok = t.size(-3) == 1 ? t.size(-1) : t.stride(-3);  // the stride of a single position means nothing
  return {t.data_ptr(), t.dim() == 4 ? t.stride(0) : 0, tok, t.stride(-2)};
}

// a gradient's buffer in the layout of its input, where that has every element once
Tensor gradient_like(const Tensor& t) {
  Tensor g = at::empty_like(t);
  return direct(g) ? g : at::empty(t.sizes(), t.options());
}

// Packed calls of one sequence, or of at most 64 and too few tiles for their order to matter, need no plan: a launch
// less (48 documents of up to 96 tokens, 12 heads: 13 us with it, 7.3 without).
bool needs_plan(const Tensor& q, int64_t n_seqs) {
  return n_seqs > 1 && (n_seqs > 64 || (q.size(0) / 128 + n_seqs) * q.size(1) > 1024);
}

// plan: the plan, or the boundaries themselves (int32), or undefined for the batch layout
bgx_attention_shape shape_of(const Tensor& q, const Tensor& k, const Tensor& plan, const Tensor& lengths, int64_t n_seqs,
                             double scale) {
  bgx_attention_shape s{};
  if (plan.defined() && plan.scalar_type() == at::kInt)
    s.cu_seqlens_dev = plan.data_ptr<int32_t>();
  else
    s.plan_dev = ptr(plan);
  s.lengths_dev = lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr;
  s.rows = q.dim() == 4 ? q.size(0) * q.size(1) : q.size(0);
  s.n_seqs = (int32_t)n_seqs;
  s.heads = (int32_t)q.size(-2);
  s.kv_heads = (int32_t)k.size(-2);
  s.head_dim = (int32_t)q.size(-1);
  s.dtype = dtype_code(q.scalar_type());
  s.scale = (float)scale;
  return s;
}

struct AttentionCall {
  Tensor out, plan, saved;
  int64_t n_seqs;
};

AttentionCall attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, const Tensor& lengths,
                                double scale, bool keep) {
  AttentionCall r;
  r.out = at::empty(q.sizes(), q.options());
  r.n_seqs = q.dim() == 4 ? q.size(0) : cu.size(0) - 1;
  void* stream = stream_of(q);
  const auto bytes = q.options().dtype(at::kByte);
  if (q.dim() == 3 && !needs_plan(q, r.n_seqs)) {
    r.plan = cu;
  } else if (q.dim() == 3) {
    const size_t n = bgx_attention_plan_bytes(q.size(0), (int32_t)r.n_seqs);
    r.plan = at::empty({(int64_t)n}, bytes);
    check(bgx_attention_plan(cu.data_ptr<int32_t>(), (int32_t)r.n_seqs, q.size(0), out_ptr(r.plan), n, stream),
          "bgx_attention_plan");
  }
  const bgx_attention_shape shape = shape_of(q, k, r.plan, lengths, r.n_seqs, scale);
  if (keep) r.saved = at::empty({(int64_t)bgx_attention_saved_bytes(&shape)}, bytes);
  const bgx_attention_rows rq = rows_of(q), rk = rows_of(k), rv = rows_of(v), ro = rows_of(r.out);
  check(bgx_attention_forward(&shape, &rq, &rk, &rv, &ro, out_ptr(r.saved), stream), "bgx_attention_forward");
  return r;
}

struct CausalAttention : torch::autograd::Function<CausalAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                        const optional<Tensor>& cu, const optional<Tensor>& lengths, double scale) {
    const Tensor q = operand(q_in), k = operand(k_in), v = operand(v_in);
    AttentionCall r = attention_forward(q, k, v, cu.value_or(Tensor()), lengths.value_or(Tensor()), scale, true);
    ctx->save_for_backward({q, k, v, r.out, r.saved, r.plan, lengths.value_or(Tensor())});
    ctx->saved_data["n_seqs"] = r.n_seqs;
    ctx->saved_data["scale"] = scale;
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &kept = saved[4];
    const c10::DeviceGuard guard(q.device());
    const bgx_attention_shape shape =
        shape_of(q, k, saved[5], saved[6], ctx->saved_data["n_seqs"].toInt(), ctx->saved_data["scale"].toDouble());
    const Tensor grad = operand(grads[0]);
    Tensor dq = gradient_like(q), dk = gradient_like(k), dv = gradient_like(v);
    const size_t nbytes = bgx_attention_backward_workspace_bytes(&shape);
    const Tensor ws = at::empty({(int64_t)nbytes}, q.options().dtype(at::kByte));
    const bgx_attention_rows rq = rows_of(q), rk = rows_of(k), rv = rows_of(v), ro = rows_of(out), rg = rows_of(grad),
                             rdq = rows_of(dq), rdk = rows_of(dk), rdv = rows_of(dv);
    check(bgx_attention_backward(&shape, &rq, &rk, &rv, &ro, ptr(kept), &rg, &rdq, &rdk, &rdv, out_ptr(ws), nbytes,
                                 stream_of(q)),
          "bgx_attention_backward");
    return once({dq, dk, dv, Tensor(), Tensor(), Tensor()});
  }
};

Tensor causal_attention(const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& cu_in,
                        const optional<Tensor>& lengths_in, optional<double> scale_in) {
  dtype_code(q.scalar_type());
  TORCH_CHECK_VALUE((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim() && v.dim() == q.dim(), "q ", q.sizes(), ", k ",
                    k.sizes(), ", v ", v.sizes(), " must all be [N, S, heads, D] or all [T, heads, D]");
  bool match = k.sizes() == v.sizes() && k.size(-1) == q.size(-1);
  for (int64_t i = 0; i < q.dim() - 2; ++i) match = match && k.size(i) == q.size(i);
  TORCH_CHECK_VALUE(match, "q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not match");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k and v share one dtype; got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  const int64_t heads = q.size(-2), kv_heads = k.size(-2), dim = q.size(-1);
  TORCH_CHECK_VALUE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, heads, " query heads on ", kv_heads,
                    " key/value heads");
  TORCH_CHECK_VALUE(dim >= 1 && dim <= MAX_HEAD_DIM, "head dimension ", dim, "; supported are 1 to ", MAX_HEAD_DIM);
  const double scale = scale_in.value_or(1.0 / std::sqrt((double)dim));
  TORCH_CHECK_VALUE((float)scale > 0.f && (float)scale < INFINITY, "scale=", scale, " must be positive and finite");
  const Tensor cu = cu_in.value_or(Tensor()), lengths = lengths_in.value_or(Tensor());
  if (q.dim() == 3) {
    TORCH_CHECK_VALUE(cu.defined() && !lengths.defined(), "packed sequences come with cu_seqlens (and without lengths)");
  } else {
    TORCH_CHECK_VALUE(!cu.defined(),
                      "cu_seqlens go with packed [T, heads, D] inputs; a batch [N, S, heads, D] takes lengths");
  }
  no_tangent(q, "q");
  no_tangent(k, "k");
  no_tangent(v, "v");
  need_gpu(q, "q");
  same_device(q, k, "k");
  same_device(q, v, "v");
  auto index_vector = [&](const Tensor& t, const char* name, int64_t size) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (size < 0 || t.size(0) == size),
                      name, " must be a contiguous int32 vector", size < 0 ? std::string() : c10::str(" of ", size, " elements"),
                      ", got ", t.scalar_type(), " ", t.sizes());
    need_gpu(t, name);
    TORCH_CHECK_VALUE(t.device() == q.device(), name, " lives on ", t.device(), ", the queries on ", q.device());
  };
  if (cu.defined()) {
    index_vector(cu, "cu_seqlens", -1);
    TORCH_CHECK_VALUE(cu.size(0) >= 1, "cu_seqlens needs at least one element");
  }
  if (lengths.defined()) index_vector(lengths, "lengths", q.size(0));
  // nothing to attend to: a plain zero of the inputs, which keeps their graph
  if (q.numel() == 0) return (q.sum() + k.sum() + v.sum()) * at::zeros(q.sizes(), q.options());
  const c10::DeviceGuard guard(q.device());
  // heads of a ragged width are padded with zeros to whole 16-byte pieces: zeros change no score and no sum
  const int64_t piece = 16 / q.element_size(), pad = (piece - dim % piece) % piece;
  if (pad) {
    auto wide = [&](const Tensor& t) { return at::constant_pad_nd(t, {0, pad}); };
    return causal_attention(wide(q), wide(k), wide(v), cu_in, lengths_in, scale).narrow(-1, 0, dim).contiguous();
  }
  if (wants_graph({q, k, v})) return CausalAttention::apply(q, k, v, cu_in, lengths_in, scale);
  return attention_forward(operand(q), operand(k), operand(v), cu, lengths, scale, false).out;
}

// ---- distillation -----------------------------------------------------------------------------------------------
Tensor distill_forward(const Tensor& logits, const Tensor& rows, const Tensor& ids, const Tensor& teacher,
                       const Tensor& valid, double temperature, const Tensor& stats) {
  Tensor losses = at::empty(logits.sizes().slice(0, logits.dim() - 1), logits.options().dtype(at::kFloat));
  check(bgx_distill_forward(ptr(rows), row_stride(rows), rows.size(0), (int32_t)rows.size(1),
                            dtype_code(rows.scalar_type()), ids.data_ptr<int64_t>(), ptr(teacher),
                            dtype_code(teacher.scalar_type()), (int32_t)ids.size(1),
                            valid.defined() ? (const uint8_t*)valid.data_ptr() : nullptr, (float)temperature,
                            losses.data_ptr<float>(), stats.defined() ? stats.data_ptr<float>() : nullptr,
                            stream_of(logits)),
        "bgx_distill_forward");
  return losses;
}

struct TopkDistillation : torch::autograd::Function<TopkDistillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& teacher,
                        const optional<Tensor>& valid, double temperature) {
    const Tensor rows = as_rows(logits, logits.size(-1));
    const Tensor stats = at::empty({rows.size(0), 2}, logits.options().dtype(at::kFloat));
    Tensor losses = distill_forward(logits, rows, ids, teacher, valid.value_or(Tensor()), temperature, stats);
    ctx->save_for_backward({rows, ids, teacher, stats});
    ctx->saved_data["shape"] = logits.sizes();
    ctx->saved_data["temperature"] = temperature;
    return losses;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &ids = saved[1], &teacher = saved[2], &stats = saved[3];
    const c10::DeviceGuard guard(rows.device());
    const Tensor grad = grads[0].reshape({-1}).contiguous();
    Tensor dlogits = at::empty(ctx->saved_data["shape"].toIntVector(), rows.options());
    check(bgx_distill_backward(ptr(rows), row_stride(rows), rows.size(0), (int32_t)rows.size(1),
                               dtype_code(rows.scalar_type()), ids.data_ptr<int64_t>(), ptr(teacher),
                               dtype_code(teacher.scalar_type()), (int32_t)ids.size(1),
                               (float)ctx->saved_data["temperature"].toDouble(), stats.data_ptr<float>(),
                               grad.data_ptr<float>(), out_ptr(dlogits), rows.size(1), stream_of(rows)),
          "bgx_distill_backward");
    return once({dlogits, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor topk_distillation(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits,
                         double temperature, const optional<Tensor>& valid_in) {
  dtype_code(logits.scalar_type());
  dtype_code(teacher_logits.scalar_type());
  TORCH_CHECK_VALUE(logits.dim() >= 1 && teacher_ids.dim() == logits.dim() && logits.size(-1) >= 1, "logits ",
                    logits.sizes(), " and teacher_ids ", teacher_ids.sizes(), " must be [..., V] and [..., K]");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(teacher_ids.sizes() == teacher_logits.sizes() && teacher_ids.sizes().slice(0, logits.dim() - 1) == lead,
                    "teacher_ids ", teacher_ids.sizes(), " and teacher_logits ", teacher_logits.sizes(),
                    " do not match logits ", logits.sizes());
  const int64_t K = teacher_ids.size(-1);
  TORCH_CHECK_VALUE(K >= 1 && K <= MAX_TEACHER_ENTRIES, K, " teacher entries per token; supported are 1 to ",
                    MAX_TEACHER_ENTRIES);
  TORCH_CHECK_VALUE(logits.size(-1) <= INT32_MAX - 64, "a vocabulary of ", logits.size(-1));
  TORCH_CHECK_TYPE(teacher_ids.scalar_type() == at::kLong, "teacher_ids must be int64, got ", teacher_ids.scalar_type());
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && teacher_logits.requires_grad()),
                    "teacher_logits are constants of the loss: detach them");
  TORCH_CHECK_VALUE((float)temperature > 0.f && (float)temperature < INFINITY, "temperature=", temperature,
                    " must be positive and finite");
  const Tensor valid = valid_in.value_or(Tensor());
  if (valid.defined())
    TORCH_CHECK_VALUE(valid.scalar_type() == at::kBool && valid.sizes() == lead, "valid must be bool ", lead, ", got ",
                      valid.scalar_type(), " ", valid.sizes());
  no_tangent(logits, "logits");
  no_tangent(teacher_logits, "teacher_logits");
  need_gpu(logits, "logits");
  same_device(logits, teacher_ids, "teacher_ids");
  same_device(logits, teacher_logits, "teacher_logits");
  if (valid.defined()) same_device(logits, valid, "valid");
  const c10::DeviceGuard guard(logits.device());
  // the graph keeps the teacher's entries as they are now
  const Tensor ids = teacher_ids.reshape({-1, K}).contiguous(), teacher = teacher_logits.reshape({-1, K}).contiguous();
  optional<Tensor> mask;
  if (valid.defined()) mask = valid.reshape({-1}).contiguous();
  if (wants_graph({logits})) return TopkDistillation::apply(logits, ids, teacher, mask, temperature);
  return distill_forward(logits, as_rows(logits, logits.size(-1)), ids, teacher, mask.value_or(Tensor()), temperature, Tensor());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("causal_attention", &causal_attention, py::call_guard<py::gil_scoped_release>());
  m.def("topk_distillation", &topk_distillation, py::call_guard<py::gil_scoped_release>());
}
