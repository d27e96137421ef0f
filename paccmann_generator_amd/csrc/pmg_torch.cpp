// PyTorch operators of the namespace `pmg` over include/pmg_lm.h: schemas, argument checks, autograd.
//
// In C++ because the calls are short: an update of the decoder's 13 tensors is about 20 us on the device, and
// from Python the checks and pointer lists of four times 13 tensors take longer than that; a backward in
// Python also runs on autograd's own thread, which has to be handed the interpreter first (about 100 us a
// call).  Every message begins with "pmg" (lm_ops.py turns such errors into PmgError).
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/pmg_lm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PMG_F32;
    case at::kBFloat16: return PMG_BF16;
    case at::kHalf: return PMG_F16;
    default: TORCH_CHECK(false, "pmg: fp32, bf16 or fp16 tensors required, got ", t.scalar_type());
  }
}

int id_bits_of(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, "pmg: token ids must be int64 or int32, got ",
              t.scalar_type());
  return t.scalar_type() == at::kLong ? 64 : 32;
}

void need_device(const Tensor& t, const at::Device& d) {
  TORCH_CHECK(t.is_cuda(), "pmg: tensors must live on the GPU (there is no CPU path)");
  TORCH_CHECK(t.device() == d, "pmg: the tensors of one call must live on one device, got ", d, " and ", t.device());
}

void need_device(at::TensorList ts, const at::Device& d) {
  for (const Tensor& t : ts) need_device(t, d);
}

// The device of a call, current while it lives, and that device's stream.
struct On {
  c10::DeviceGuard guard;
  pmg_stream stream;
  explicit On(const at::Device& d)
      : guard(d), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream()) {}
};

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, ": ", pmg_strerror(rc), " (code ", rc, ")");
}

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}

Tensor fp32(at::IntArrayRef size, const Tensor& like) {
  return at::empty(size, like.options().dtype(at::kFloat).requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
}

bool same_layout(const Tensor& a, const Tensor& b) {
  return a.sizes() == b.sizes() && ((a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides());
}

void changed(at::TensorList ts) {
  for (const Tensor& t : ts)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// `t` [..., width] as rows of contiguous elements; copied where it is not such rows (a stride of 0 of an expanded
// tensor among them).  ld: elements from one row to the next.
Tensor rows_of(const Tensor& t, int64_t width, int64_t* ld) {
  Tensor r = t.reshape({-1, width});
  const bool one = r.size(0) <= 1;
  if ((width > 1 && r.stride(1) != 1) || (!one && r.stride(0) < width)) r = r.contiguous();
  *ld = one ? width : r.stride(0);
  return r;
}

// A gradient formed with create_graph: it is right, a backward through it to what it was made from is refused (and not
// taken for zero).
struct NotTwice : torch::autograd::Function<NotTwice> {
  static Tensor forward(AutogradContext*, const Tensor& grad, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                        const OptTensor&) {
    return grad.view_as(grad);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "pmg: gradients of this operator are not differentiable");
  }
};

Tensor last(const Tensor& grad, const OptTensor& a, const OptTensor& b = {}, const OptTensor& c = {}, const OptTensor& d = {},
            const OptTensor& e = {}) {
  return at::GradMode::is_enabled() && grad.defined() ? NotTwice::apply(grad, a, b, c, d, e) : grad;
}

// ------------------------------------------------------------------------------------------ embedding
Tensor embedding(const Tensor& weight, const Tensor& ids, double scale, int64_t padding_idx) {
  need_device({weight, ids}, weight.device());
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "pmg::embedding: a table [V, E] required, got ",
              weight.sizes());
  const int64_t V = weight.size(0), E = weight.size(1);
  TORCH_CHECK(padding_idx >= -1 && padding_idx < V, "pmg::embedding: padding_idx must lie in [0, ", V, ") or be -1 (none)");
  const int dtype = dtype_of(weight), bits = id_bits_of(ids);
  int64_t ld;
  const Tensor w = rows_of(weight, E, &ld), flat = ids.contiguous();
  auto size = ids.sizes().vec();
  size.push_back(E);
  Tensor out = at::empty(size, weight.options().requires_grad(false));
  On on(weight.device());
  check(pmg_embedding_fwd(w.data_ptr(), ld, flat.data_ptr(), bits, flat.numel(), V, E, dtype, (float)scale, out.data_ptr(),
                          on.stream),
        "pmg_embedding_fwd");
  return out;
}

Tensor embedding_bwd(const Tensor& grad, const Tensor& ids, int64_t vocab_size, double scale, int64_t padding_idx) {
  need_device({grad, ids}, grad.device());
  TORCH_CHECK(grad.dim() >= 1 && grad.size(-1) > 0 && grad.sizes().slice(0, grad.dim() - 1) == ids.sizes(),
              "pmg::embedding_bwd: gradient ", grad.sizes(), " for ids ", ids.sizes());
  const int64_t E = grad.size(-1);
  const int dtype = dtype_of(grad), bits = id_bits_of(ids);
  int64_t ld;
  const Tensor g = rows_of(grad, E, &ld), flat = ids.contiguous();
  size_t need = 0;
  check(pmg_embedding_bwd_workspace(flat.numel(), vocab_size, E, dtype, &need), "pmg_embedding_bwd_workspace");
  const Tensor ws = bytes(need, grad);
  Tensor out = at::empty({vocab_size, E}, grad.options().requires_grad(false));
  On on(grad.device());
  check(pmg_embedding_bwd(g.data_ptr(), ld, flat.data_ptr(), bits, flat.numel(), vocab_size, E, dtype, (float)scale, padding_idx,
                          out.data_ptr(), ws.data_ptr(), on.stream),
        "pmg_embedding_bwd");
  return out;
}

Tensor call_embedding(const Tensor& weight, const Tensor& ids, double scale, int64_t padding_idx) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pmg::embedding", "").typed<decltype(embedding)>();
  return op.call(weight, ids, scale, padding_idx);
}

Tensor call_embedding_bwd(const Tensor& grad, const Tensor& ids, int64_t vocab_size, double scale, int64_t padding_idx) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pmg::embedding_bwd", "").typed<decltype(embedding_bwd)>();
  return op.call(grad, ids, vocab_size, scale, padding_idx);
}

struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({ids});
    ctx->saved_data["v"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = padding_idx;
    return call_embedding(weight, ids, scale, padding_idx);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto saved = ctx->get_saved_variables();
    Tensor dw;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      dw = call_embedding_bwd(grad[0], saved[0], ctx->saved_data["v"].toInt(), ctx->saved_data["scale"].toDouble(),
                              ctx->saved_data["pad"].toInt());
    }
    return {last(dw, grad[0]), Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding_autograd(const Tensor& weight, const Tensor& ids, double scale, int64_t padding_idx) {
  return EmbeddingGrad::apply(weight, ids, scale, padding_idx);
}

// --------------------------------------------------------------------------- linear cross entropy
// The C call's arguments without the outputs; holds the tensors they point into.
struct CeCall {
  pmg_linear_ce a = {};
  Tensor x, w, t, b, r;
  CeCall(const Tensor& hidden, const Tensor& weight, const OptTensor& bias, const Tensor& targets, const OptTensor& row_weight,
         int64_t ignore_index, double logit_scale, int64_t reduction) {
    const at::Device d = hidden.device();
    need_device({hidden, weight, targets}, d);
    if (bias) need_device(*bias, d);
    if (row_weight) need_device(*row_weight, d);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0,
                "pmg::linear_cross_entropy: weight must be [V, H], got ", weight.sizes());
    a.V = weight.size(0);
    a.H = weight.size(1);
    TORCH_CHECK(hidden.dim() >= 1 && hidden.size(-1) == a.H && hidden.sizes().slice(0, hidden.dim() - 1) == targets.sizes(),
                "pmg::linear_cross_entropy: hidden [..., ", a.H, "] and targets [...] required, got ", hidden.sizes(), " and ",
                targets.sizes());
    TORCH_CHECK(hidden.scalar_type() == weight.scalar_type() && (!bias || bias->scalar_type() == weight.scalar_type()) &&
                    (weight.scalar_type() == at::kFloat || weight.scalar_type() == at::kBFloat16),
                "pmg::linear_cross_entropy: hidden, weight and bias must all be fp32 or all be bf16 (the slopes of the logits "
                "leave the range of fp16)");
    TORCH_CHECK(!bias || (bias->dim() == 1 && bias->size(0) == a.V), "pmg::linear_cross_entropy: bias must be [", a.V, "]");
    TORCH_CHECK(!row_weight || (row_weight->scalar_type() == at::kFloat && row_weight->sizes() == targets.sizes()),
                "pmg::linear_cross_entropy: row_weight must be fp32, one value per target");
    x = rows_of(hidden, a.H, &a.ld_hidden);
    w = rows_of(weight, a.H, &a.ld_weight);
    t = targets.contiguous();
    if (bias) b = bias->contiguous();
    if (row_weight) r = row_weight->contiguous();
    a.N = t.numel();
    a.dtype = dtype_of(weight);
    a.id_bits = id_bits_of(t);
    a.reduction = (int)reduction;
    a.logit_scale = (float)logit_scale;
    a.ignore_index = ignore_index;
    a.hidden = x.data_ptr();
    a.weight = w.data_ptr();
    a.targets = t.data_ptr();
    a.bias = b.defined() ? b.data_ptr() : nullptr;
    a.row_weight = r.defined() ? (const float*)r.data_ptr() : nullptr;
  }
  Tensor workspace(int backward) const {
    size_t need = 0;
    check(pmg_linear_ce_workspace(&a, backward, &need), "pmg_linear_ce_workspace");
    return bytes(need, x);
  }
};

// The logits too where `keep` says so (else an empty tensor).
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_ce_keep(const Tensor& hidden, const Tensor& weight, const OptTensor& bias,
                                                          const Tensor& targets, const OptTensor& row_weight,
                                                          int64_t ignore_index, double logit_scale, int64_t reduction,
                                                          bool keep) {
  CeCall c(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction);
  const bool none = reduction == PMG_REDUCE_NONE;
  Tensor loss = fp32(none ? targets.sizes() : at::IntArrayRef(), hidden), lse = fp32(targets.sizes(), hidden);
  Tensor count = none ? fp32({0}, hidden) : fp32({}, hidden);
  Tensor logits = fp32({keep ? c.a.N : 0, (c.a.V + 3) / 4 * 4}, hidden);
  if (c.a.N == 0) return {loss.zero_(), lse, count.zero_(), logits};
  c.a.logits = keep ? (float*)logits.data_ptr() : nullptr;
  const Tensor ws = c.workspace(0);
  c.a.loss = (float*)loss.data_ptr();
  c.a.lse = (float*)lse.data_ptr();
  c.a.count = none ? nullptr : (float*)count.data_ptr();
  On on(hidden.device());
  check(pmg_linear_ce_fwd(&c.a, ws.data_ptr(), on.stream), "pmg_linear_ce_fwd");
  return {loss, lse, count, logits};
}

std::tuple<Tensor, Tensor, Tensor> linear_ce(const Tensor& hidden, const Tensor& weight, const OptTensor& bias,
                                             const Tensor& targets, const OptTensor& row_weight, int64_t ignore_index,
                                             double logit_scale, int64_t reduction) {
  auto [loss, lse, count, logits] =
      linear_ce_keep(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction, false);
  return {loss, lse, count};
}

std::tuple<Tensor, Tensor, Tensor> linear_ce_bwd(const OptTensor& grad_loss, const OptTensor& grad_lse, const Tensor& hidden,
                                                 const Tensor& weight, const OptTensor& bias, const Tensor& targets,
                                                 const OptTensor& row_weight, const Tensor& lse, const Tensor& count,
                                                 int64_t ignore_index, double logit_scale, int64_t reduction,
                                                 std::array<bool, 3> wanted, const OptTensor& logits) {
  CeCall c(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction);
  TORCH_CHECK(!wanted[2] || bias, "pmg::linear_cross_entropy_bwd: there is no bias");
  const auto out = [&](bool want, at::IntArrayRef size) {
    return at::empty(want ? size : at::IntArrayRef({0}),
                     weight.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  };
  Tensor dx = out(wanted[0], hidden.sizes()), dw = out(wanted[1], weight.sizes()), db = out(wanted[2], {c.a.V});
  if (c.a.N == 0) return {dx, dw.zero_(), db.zero_()};
  const bool none = reduction == PMG_REDUCE_NONE;
  need_device({lse, count}, hidden.device());
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.sizes() == targets.sizes() && lse.is_contiguous() &&
                  count.scalar_type() == at::kFloat && (none || count.numel() == 1),
              "pmg::linear_cross_entropy_bwd: lse and count must be those of the forward call");
  if (logits && logits->numel()) {
    need_device(*logits, hidden.device());
    TORCH_CHECK(logits->scalar_type() == at::kFloat && logits->is_contiguous() && logits->dim() == 2 &&
                    logits->size(0) == c.a.N && logits->size(1) == (c.a.V + 3) / 4 * 4,
                "pmg::linear_cross_entropy_bwd: logits must be those of the forward call");
    c.a.logits = (float*)logits->data_ptr();
  }
  Tensor slope[2];
  for (int k = 0; k < 2; ++k) {
    const OptTensor& g = k == 0 ? grad_loss : grad_lse;
    if (!g || !g->defined()) continue;
    need_device(*g, hidden.device());
    TORCH_CHECK(k == 0 && !none ? g->numel() == 1 : g->sizes() == targets.sizes(),
                "pmg::linear_cross_entropy_bwd: a slope for every element of loss and lse required, got ", g->sizes());
    slope[k] = g->to(at::kFloat).contiguous();
  }
  c.a.grad_loss = slope[0].defined() ? (const float*)slope[0].data_ptr() : nullptr;
  c.a.grad_lse = slope[1].defined() ? (const float*)slope[1].data_ptr() : nullptr;
  c.a.lse = (float*)lse.data_ptr();
  c.a.count = none ? nullptr : (float*)count.data_ptr();
  c.a.grad_hidden = wanted[0] ? dx.data_ptr() : nullptr;
  c.a.grad_weight = wanted[1] ? dw.data_ptr() : nullptr;
  c.a.grad_bias = wanted[2] ? db.data_ptr() : nullptr;
  const Tensor ws = c.workspace(1);
  On on(hidden.device());
  check(pmg_linear_ce_bwd(&c.a, ws.data_ptr(), on.stream), "pmg_linear_ce_bwd");
  return {dx, dw, db};
}

struct LinearCeGrad : torch::autograd::Function<LinearCeGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const OptTensor& bias,
                               const Tensor& targets, const OptTensor& row_weight, int64_t ignore_index, double logit_scale,
                               int64_t reduction, bool keep) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pmg::linear_cross_entropy_keep", "").typed<decltype(linear_ce_keep)>();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, lse, count, logits] = op.call(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction, keep);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({count});
    ctx->save_for_backward({hidden, weight, bias.value_or(Tensor()), targets, row_weight.value_or(Tensor()), lse, count,
                            logits});
    ctx->saved_data["wanted"] =
        c10::List<bool>({hidden.requires_grad(), weight.requires_grad(), bias && bias->defined() && bias->requires_grad()});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["scale"] = logit_scale;
    ctx->saved_data["reduction"] = reduction;
    return {loss, lse, count};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    static auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("pmg::linear_cross_entropy_bwd", "").typed<decltype(linear_ce_bwd)>();
    variable_list out(9);
    const auto wanted = ctx->saved_data["wanted"].toBoolList();
    if (!grad[0].defined() && !grad[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto [dx, dw, db] = [&] {
      at::AutoDispatchBelowADInplaceOrView below;
      return op.call(opt(grad[0]), opt(grad[1]), s[0], s[1], opt(s[2]), s[3], opt(s[4]), s[5], s[6],
                                ctx->saved_data["ignore"].toInt(), ctx->saved_data["scale"].toDouble(),
                                ctx->saved_data["reduction"].toInt(), {wanted.get(0), wanted.get(1), wanted.get(2)}, s[7]);
    }();
    const OptTensor from[5] = {opt(grad[0]), opt(grad[1]), s[0], s[1], opt(s[2])};
    if (wanted.get(0)) out[0] = last(dx, from[0], from[1], from[2], from[3], from[4]);
    if (wanted.get(1)) out[1] = last(dw, from[0], from[1], from[2], from[3], from[4]);
    if (wanted.get(2)) out[2] = last(db, from[0], from[1], from[2], from[3], from[4]);
    return out;
  }
};

// Whether training keeps the logits, in fp32, rather than form them again.
//   - a row of them takes at most a quarter of the bytes of the hidden row it is made of: reading them (and their slopes) is
//     cheaper than reading the hidden rows once more, before any product (524288 rows of 512 fp32 over 60: 1146 us a step,
//     1544 without)
//   - all of them take 4 MB: forming few takes the latency of a product (5 rows of 1024 bf16 over 50000: 5 us to read them,
//     18 to form them)
//   - all of them take 256 MB, no more than the backward's own scratch, and the hidden size is long enough for writing and
//     reading 8 bytes to take less than 2 H operations (bf16 8000
//     rows of 1024 over 8000: 108 us to write and read them, 142 to form them; 2000 of 4096 over 32000: 136 and 466; fp32
//     30000 of 136 over 2000: 132 and 198)
bool keep_logits(const c10::SymInt& n, const c10::SymInt& v, const c10::SymInt& h, int64_t size) {
  const c10::SymInt all = n * v;
  return v * 16 <= h * size || all <= (1 << 20) || (all <= (64 << 20) && h >= (size == 4 ? 128 : 1024));
}

std::tuple<Tensor, Tensor, Tensor> linear_ce_autograd(const Tensor& hidden, const Tensor& weight, const OptTensor& bias,
                                                      const Tensor& targets, const OptTensor& row_weight, int64_t ignore_index,
                                                      double logit_scale, int64_t reduction) {
  const bool grads = at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()));
  const bool keep = grads && weight.dim() == 2 && keep_logits(targets.sym_numel(), weight.sym_size(0), weight.sym_size(1), weight.element_size());
  auto out = LinearCeGrad::apply(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction, keep);
  return {out[0], out[1], out[2]};
}

// --------------------------------------------------------------------------------- norm and clipping
Tensor norm_call(at::TensorList grads, const double* max_norm) {
  TORCH_CHECK(!grads.empty(), "pmg: no gradients");
  const at::Device d = grads[0].device();
  const int n = (int)grads.size();
  std::vector<const void*> ptr(n);
  std::vector<int64_t> numel(n);
  std::vector<int> dtype(n);
  std::vector<Tensor> copies;
  for (int i = 0; i < n; ++i) {
    const Tensor& g = grads[i];
    need_device(g, d);
    dtype[i] = dtype_of(g);
    numel[i] = g.numel();
    ptr[i] = g.data_ptr();
    if (!g.is_non_overlapping_and_dense()) {
      TORCH_CHECK(!max_norm, "pmg::clip_grad_norm_: gradients must be dense (no gaps, no repeated elements)");
      copies.push_back(g.contiguous());
      ptr[i] = copies.back().data_ptr();
    }
  }
  size_t need = 0;
  check(pmg_grad_norm_workspace(numel.data(), n, &need), "pmg_grad_norm_workspace");
  const Tensor ws = bytes(need, grads[0]);
  Tensor norm = fp32({}, grads[0]);
  On on(d);
  float* to = (float*)norm.data_ptr();
  // what the clipping would refuse is refused before the norm is launched
  if (max_norm)
    check(pmg_grad_clip_check((void* const*)ptr.data(), numel.data(), dtype.data(), n, (float)*max_norm), "pmg_grad_clip");
  check(pmg_grad_norm(ptr.data(), numel.data(), dtype.data(), n, to, ws.data_ptr(), on.stream), "pmg_grad_norm");
  if (max_norm)
    check(pmg_grad_clip((void* const*)ptr.data(), numel.data(), dtype.data(), n, to, (float)*max_norm, on.stream), "pmg_grad_clip");
  return norm;
}

Tensor grad_norm(at::TensorList grads) { return norm_call(grads, nullptr); }

Tensor clip_grad_norm(at::TensorList grads, double max_norm) {
  TORCH_CHECK(max_norm > 0, "pmg::clip_grad_norm_: max_norm must be positive");
  Tensor norm = norm_call(grads, &max_norm);
  changed(grads);
  return norm;
}

// ------------------------------------------------------------------------------------------- AdamW
void adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avg, at::TensorList exp_avg_sq,
                at::TensorList top_m, at::TensorList top_v, at::TensorList master, const Tensor& step, const OptTensor& lr_tensor,
                const OptTensor& norm, double lr, double beta1, double beta2, double eps, double weight_decay, double max_norm,
                bool decoupled) {
  const size_t n = params.size();
  TORCH_CHECK(n > 0, "pmg::adamw_step_: no parameters");
  const bool q = !top_m.empty() || !top_v.empty(), copy = !master.empty();
  TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n && (!q || (top_m.size() == n && top_v.size() == n)) &&
                  (!copy || master.size() == n),
              "pmg::adamw_step_: lists of different lengths");
  const at::Device d = step.device();
  for (at::TensorList list : {params, grads, exp_avg, exp_avg_sq, top_m, top_v, master}) need_device(list, d);
  need_device(step, d);
  TORCH_CHECK(step.scalar_type() == at::kLong && step.numel() == 1, "pmg::adamw_step_: step must be one int64 value");
  for (const OptTensor* t : {&lr_tensor, &norm}) {
    if (!t->has_value()) continue;
    need_device(**t, d);
    TORCH_CHECK((*t)->scalar_type() == at::kFloat && (*t)->numel() == 1,
                "pmg::adamw_step_: learning rate and norm must be one fp32 value each");
  }
  const auto p_type = params[0].scalar_type(), g_type = grads[0].scalar_type();
  const auto m_type = q ? at::kChar : at::kFloat, v_type = q ? at::kByte : at::kFloat;
  std::vector<int64_t> numel(n);
  std::vector<void*> ptr(n * 6, nullptr);
  std::vector<const void*> grad(n);
  std::vector<Tensor> laid;
  void **pp = ptr.data(), **pm = pp + n, **pv = pm + n, **pmt = pv + n, **pvt = pmt + n, **pw = pvt + n;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &g = grads[i], &m = exp_avg[i], &v = exp_avg_sq[i];
    TORCH_CHECK(p.scalar_type() == p_type && g.scalar_type() == g_type && m.scalar_type() == m_type && v.scalar_type() == v_type,
                "pmg::adamw_step_: one element type per list: parameters, gradients, fp32 states (or int8 and uint8 codes); got ",
                p.scalar_type(), ", ", g.scalar_type(), ", ", m.scalar_type(), ", ", v.scalar_type());
    TORCH_CHECK(p.sizes() == g.sizes(), "pmg::adamw_step_: gradient of shape ", g.sizes(), " for a parameter ", p.sizes());
    TORCH_CHECK(p.is_non_overlapping_and_dense() && same_layout(p, m) && same_layout(p, v),
                "pmg::adamw_step_: parameters must be dense (no gaps, no repeated elements) and states must have their shape and "
                "strides");
    numel[i] = p.numel();
    pp[i] = p.data_ptr();
    pm[i] = m.data_ptr();
    pv[i] = v.data_ptr();
    if (copy) {
      TORCH_CHECK(master[i].scalar_type() == at::kFloat && same_layout(p, master[i]),
                  "pmg::adamw_step_: 32-bit copies must be fp32 and have the shape and strides of their parameter");
      pw[i] = master[i].data_ptr();
    }
    if (q) {
      const int64_t blocks = (p.numel() + PMG_STATE_BLOCK - 1) / PMG_STATE_BLOCK;
      for (const Tensor* s : {&top_m[i], &top_v[i]})
        TORCH_CHECK(s->scalar_type() == at::kFloat && s->numel() == blocks && s->is_contiguous(), "pmg::adamw_step_: ", blocks,
                    " contiguous fp32 scales required for a state of ", p.numel(), " values");
      pmt[i] = top_m[i].data_ptr();
      pvt[i] = top_v[i].data_ptr();
    }
    if (same_layout(p, g)) {
      grad[i] = g.data_ptr();
    } else {  // a gradient of another memory order than its parameter's is brought into that order
      laid.push_back(at::empty_like(p, p.options().dtype(g_type).requires_grad(false)).copy_(g));
      grad[i] = laid.back().data_ptr();
    }
  }
  pmg_adamw a = {};
  a.n = (int)n;
  a.dtype = dtype_of(params[0]);
  a.grad_dtype = dtype_of(grads[0]);
  a.state_bits = q ? 8 : 32;
  a.decoupled = decoupled;
  a.numel = numel.data();
  a.param = pp;
  a.grad = grad.data();
  a.m = pm;
  a.v = pv;
  a.m_top = q ? (float* const*)pmt : nullptr;
  a.v_top = q ? (float* const*)pvt : nullptr;
  a.master = copy ? (float* const*)pw : nullptr;
  a.step = (int64_t*)step.data_ptr();
  a.lr_dev = lr_tensor ? (const float*)lr_tensor->data_ptr() : nullptr;
  a.norm = norm ? (const float*)norm->data_ptr() : nullptr;
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.max_norm = max_norm;
  const Tensor ws = bytes(PMG_ADAMW_WS, step);
  On on(d);
  check(pmg_adamw_step(&a, ws.data_ptr(), on.stream), "pmg_adamw_step");
  for (at::TensorList list : {params, exp_avg, exp_avg_sq, top_m, top_v, master}) changed(list);
  changed({step});
}

Tensor adamw_state_values(const Tensor& code, const Tensor& top) {
  need_device({code, top}, code.device());
  TORCH_CHECK((code.scalar_type() == at::kChar || code.scalar_type() == at::kByte) && top.scalar_type() == at::kFloat,
              "pmg::adamw_state_values: int8 or uint8 codes and fp32 scales required");
  TORCH_CHECK(code.is_non_overlapping_and_dense() && top.is_contiguous() &&
                  top.numel() == (code.numel() + PMG_STATE_BLOCK - 1) / PMG_STATE_BLOCK,
              "pmg::adamw_state_values: dense codes with one scale per ", PMG_STATE_BLOCK, " required");
  Tensor out = at::empty_like(code, code.options().dtype(at::kFloat));
  On on(code.device());
  check(pmg_adamw_values(code.data_ptr(), (const float*)top.data_ptr(), code.numel(), code.scalar_type() == at::kChar,
                         (float*)out.data_ptr(), on.stream),
        "pmg_adamw_values");
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pmg, m) {
  m.def("embedding(Tensor weight, Tensor ids, float scale, int padding_idx) -> Tensor");
  m.def("embedding_bwd(Tensor grad, Tensor ids, int vocab_size, float scale, int padding_idx) -> Tensor");
  m.def(
      "linear_cross_entropy(Tensor hidden, Tensor weight, Tensor? bias, Tensor targets, Tensor? row_weight, int ignore_index, "
      "float logit_scale, int reduction) -> (Tensor, Tensor, Tensor)");
  m.def(
      "linear_cross_entropy_keep(Tensor hidden, Tensor weight, Tensor? bias, Tensor targets, Tensor? row_weight, int ignore_index, "
      "float logit_scale, int reduction, bool keep) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "linear_cross_entropy_bwd(Tensor? grad_loss, Tensor? grad_lse, Tensor hidden, Tensor weight, Tensor? bias, Tensor targets, "
      "Tensor? row_weight, Tensor lse, Tensor count, int ignore_index, float logit_scale, int reduction, bool[3] wanted, Tensor? logits=None) -> "
      "(Tensor, Tensor, Tensor)");
  m.def("grad_norm(Tensor[] grads) -> Tensor");
  m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor");
  m.def(
      "adamw_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, Tensor(d!)[] exp_avg_top, "
      "Tensor(e!)[] exp_avg_sq_top, Tensor(f!)[] master, Tensor(g!) step, Tensor? lr_tensor, Tensor? grad_norm, float lr, "
      "float beta1, float beta2, float eps, float weight_decay, float max_norm, bool decoupled) -> ()");
  m.def("adamw_state_values(Tensor code, Tensor top) -> Tensor");
}

TORCH_LIBRARY_IMPL(pmg, CUDA, m) {
  m.impl("embedding", embedding);
  m.impl("embedding_bwd", embedding_bwd);
  m.impl("linear_cross_entropy", linear_ce);
  m.impl("linear_cross_entropy_keep", linear_ce_keep);
  m.impl("linear_cross_entropy_bwd", linear_ce_bwd);
  m.impl("grad_norm", grad_norm);
  m.impl("clip_grad_norm_", clip_grad_norm);
  m.impl("adamw_step_", adamw_step);
  m.impl("adamw_state_values", adamw_state_values);
}

TORCH_LIBRARY_IMPL(pmg, Autograd, m) {
  m.impl("embedding", embedding_autograd);
  m.impl("linear_cross_entropy", linear_ce_autograd);
}
