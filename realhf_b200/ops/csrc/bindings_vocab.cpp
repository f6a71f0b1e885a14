// torch bindings for the operators on rows of logits: token statistics, top alternatives, distillation.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <torch/types.h>

#include <algorithm>
#include <atomic>
#include <vector>

using at::Tensor;
using OptT = c10::optional<Tensor>;

bool gradient_goes_past(const Tensor& leaf, bool own_hook);      // bindings.cpp
void check_capture(const Tensor& leaf, c10::string_view op);     // bindings.cpp
void attn_check();      // bindings_attn.cpp: an error once a bounded wait of an earlier kernel has run out

// kernels launched where Python does not see them (in a native backward pass, or one or two of them in a call), since the last question
static std::atomic<int64_t> unseen_launches{0};

extern "C" {
int rb_token_stats(const void*, int64_t, const int64_t*, const uint8_t*, int64_t, float*, float*, float*, int64_t, int, float, int, cudaStream_t);
int rb_token_stats_bwd(const void*, int64_t, const int64_t*, const uint8_t*, int64_t, const float*, const float*, const float*, const float*, void*, int64_t,
                       int64_t, int, float, int, cudaStream_t);
int rb_top_logprobs_max();
int rb_top_logprobs(const void*, int64_t, const int64_t*, const uint8_t*, int64_t, float*, float*, float*, int64_t*, float*, int64_t, int, int, float, int,
                    cudaStream_t);
int64_t rb_head_stats_scratch(int);
int rb_head_stats(const void*, const void*, int64_t, int64_t, const int64_t*, const uint8_t*, int64_t, float*, void*, int64_t, float*, float*, float*, int, int, int,
                  float, int, int, int, cudaStream_t);
int rb_head_grad(const void*, int64_t, const float*, const int64_t*, const uint8_t*, int64_t, const float*, const float*, const float*, const float*, const uint32_t*,
                 void*, int64_t, int, int, int, int, float, int, cudaStream_t);
int rb_head_grad_peak(const int64_t*, const float*, const float*, const float*, uint32_t*, int, float, cudaStream_t);
int rb_head_stats_bwd(const void*, const void*, int64_t, int64_t, const int64_t*, const uint8_t*, int64_t, const float*, const float*, const float*, const float*,
                      const uint32_t*, void*, int64_t, int, int, int, float, int, int, int, cudaStream_t);
int rb_head_dhidden_splits(int, int, int, int);
int rb_head_dhidden(const void*, const void*, int64_t, int64_t, const uint32_t*, float*, void*, int, int, int, int, int, int, cudaStream_t);
int rb_gemm_tcgen05(const void*, const void*, void*, const void*, int, int, int, int64_t, int64_t, int64_t, int, int, int, int, int, int, int, int, cudaStream_t);
int rb_head_dweight(const void*, const void*, int64_t, int64_t, const uint32_t*, void*, int, int, int, int, int, int, int, cudaStream_t);
int rb_distill_max_listed();
int64_t rb_distill_max_vocab();
int rb_distill_fwd(const void*, int64_t, const int64_t*, const float*, const float*, int, float*, float*, float*, float*, int*, int64_t, int, int, float, int,
                   cudaStream_t);
int rb_distill_peak(const float*, const float*, const float*, uint32_t*, int64_t, int, float, cudaStream_t);
int rb_distill_bwd(const void*, int64_t, const float*, const float*, const float*, const int*, const float*, const uint32_t*, void*, int64_t, int64_t, int, int, float, int,
                   int, cudaStream_t);
}

namespace {

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type(), " (float32, bfloat16 or float16)");
  }
}

bool good_factor(double inv_temp) { return inv_temp >= 1e-30 && inv_temp <= 1e30; }

void check_logits(const Tensor& logits, const char* op, double inv_temp) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, op, ": logits are a CUDA matrix [rows, vocabulary] with unit inner stride");
  TORCH_CHECK_VALUE(logits.size(1) > 0 && logits.size(1) <= 0x7ffe0000LL && logits.size(0) <= 0x7fffffffLL, op, ": bad size ", logits.sizes());
  TORCH_CHECK_VALUE(good_factor(inv_temp), op, ": the inverse temperature lies between 1e-30 and 1e30, not at ", inv_temp);
}

// a contiguous tensor of this device, of one value a row (or [rows, k])
const void* row_values(const OptT& t, at::ScalarType type, const Tensor& logits, int64_t k, const char* op, const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_VALUE(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() && (k < 0 ? t->dim() == 1 : t->dim() == 2 && t->size(1) == k) &&
                  t->size(0) == logits.size(0),
              op, ": ", name, " has to be contiguous, of type ", type, ", on the logits' device and of ", logits.size(0), " rows");
  return t->data_ptr();
}

const uint8_t* mask_rows(const OptT& mask, const Tensor& logits, const char* op) {
  if (!mask.has_value()) return nullptr;
  TORCH_CHECK_VALUE(mask->device() == logits.device() && mask->scalar_type() == at::kByte && mask->dim() == 2 && mask->is_contiguous() &&
                  mask->size(0) == logits.size(0) && mask->size(1) * 8 >= logits.size(1),
              op, ": the mask is a packed uint8 matrix [rows, at least vocabulary / 8] on the logits' device");
  return mask->data_ptr<uint8_t>();
}

int64_t mask_bytes(const OptT& mask) { return mask.has_value() ? mask->size(1) : 0; }

// the gradient's destination: a new matrix, or `out` (the logits themselves, or one like them)
Tensor gradient_like(const Tensor& logits, const OptT& out, const char* op, bool any_type = false) {
  if (!out.has_value()) return at::empty({logits.size(0), logits.size(1)}, logits.options());
  TORCH_CHECK(out->device() == logits.device() && (any_type || out->scalar_type() == logits.scalar_type()) && out->sizes() == logits.sizes() && out->stride(1) == 1, op,
              ": the gradient's destination is like the logits");
  return *out;
}

// the bound that gradients in fp16 are scaled by (`head_grad_peak`, `distill_peak`), or none
const uint32_t* peak_of(const OptT& peak, const Tensor& like, const char* op) {
  if (!peak.has_value()) return nullptr;
  TORCH_CHECK(peak->device() == like.device() && peak->scalar_type() == at::kFloat && peak->numel() == 1, op, ": the peak is one fp32 number");
  return static_cast<const uint32_t*>(peak->data_ptr());
}
Tensor new_peak(const Tensor& like) { return at::zeros({1}, like.options().dtype(at::kFloat)); }

// whole numbers as contiguous int64
Tensor whole_numbers(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), op, ": ", name, " are whole numbers, not ", t.scalar_type());
  return t.to(at::kLong).contiguous();
}
Tensor fp32(const Tensor& t) { return t.to(at::kFloat).contiguous(); }
OptT fp32(const OptT& t) { return t.has_value() ? OptT(fp32(*t)) : t; }
OptT packed(const OptT& t) { return t.has_value() ? OptT(t->contiguous()) : t; }
// rows with unit inner stride (`contiguous()` keeps a single column as it lies)
Tensor unit_rows(const Tensor& x) { return x.dim() != 2 || x.stride(1) == 1 ? x : x.clone(at::MemoryFormat::Contiguous); }

std::vector<Tensor> token_stats(const Tensor& logits, const Tensor& labels, const OptT& mask, double inv_temp) {
  check_logits(logits, "token_stats", inv_temp);
  const int64_t rows = logits.size(0);
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, logits, -1, "token_stats", "labels"));
  c10::cuda::CUDAGuard guard(logits.device());
  auto f = logits.options().dtype(at::kFloat);
  Tensor logp = at::empty({rows}, f), entropy = at::empty({rows}, f), lse = at::empty({rows}, f);
  const int rc = rb_token_stats(logits.data_ptr(), logits.stride(0), lab, mask_rows(mask, logits, "token_stats"), mask_bytes(mask), logp.data_ptr<float>(),
                                entropy.data_ptr<float>(), lse.data_ptr<float>(), rows, (int)logits.size(1), (float)inv_temp, dtype_code(logits), stream());
  TORCH_CHECK(rc == 0, "token_stats failed with code ", rc);
  return {logp, entropy, lse};
}

Tensor token_stats_bwd(const Tensor& logits, const Tensor& labels, const OptT& mask, const Tensor& lse, const Tensor& entropy, const OptT& g_logp,
                       const OptT& g_entropy, double inv_temp, const OptT& out) {
  const char* op = "token_stats_bwd";
  check_logits(logits, op, inv_temp);
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, logits, -1, op, "labels"));
  const auto* l = static_cast<const float*>(row_values(lse, at::kFloat, logits, -1, op, "lse"));
  const auto* h = static_cast<const float*>(row_values(entropy, at::kFloat, logits, -1, op, "entropy"));
  const auto* gl = static_cast<const float*>(row_values(g_logp, at::kFloat, logits, -1, op, "the log-probability's gradient"));
  const auto* ge = static_cast<const float*>(row_values(g_entropy, at::kFloat, logits, -1, op, "the entropy's gradient"));
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor d = gradient_like(logits, out, op);
  const int rc = rb_token_stats_bwd(logits.data_ptr(), logits.stride(0), lab, mask_rows(mask, logits, op), mask_bytes(mask), l, h, gl, ge, d.data_ptr(),
                                    d.stride(0), logits.size(0), (int)logits.size(1), (float)inv_temp, dtype_code(logits), stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  return d;
}

std::vector<Tensor> top_logprobs(const Tensor& logits_in, int64_t k, const OptT& labels_in, const OptT& mask_in, double inv_temp) {
  const char* op = "top_logprobs_from_logits";
  const Tensor logits = unit_rows(logits_in);
  const OptT labels = labels_in.has_value() ? OptT(whole_numbers(*labels_in, op, "labels")) : labels_in, mask = packed(mask_in);
  check_logits(logits, op, inv_temp);
  const int64_t rows = logits.size(0), V = logits.size(1);
  TORCH_CHECK_VALUE(k >= 1 && k <= V && k <= rb_top_logprobs_max(), op, ": between 1 and min(vocabulary, ", rb_top_logprobs_max(), ") alternatives, not ", k);
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, logits, -1, op, "labels"));
  c10::cuda::CUDAGuard guard(logits.device());
  auto f = logits.options().dtype(at::kFloat);
  Tensor entropy = at::empty({rows}, f), rest = at::empty({rows}, f), top = at::empty({rows, k}, f), ids = at::empty({rows, k}, f.dtype(at::kLong));
  Tensor logp = labels.has_value() ? at::empty({rows}, f) : Tensor();
  const int rc = rb_top_logprobs(logits.data_ptr(), logits.stride(0), lab, mask_rows(mask, logits, op), mask_bytes(mask),
                                 labels.has_value() ? logp.data_ptr<float>() : nullptr, entropy.data_ptr<float>(), top.data_ptr<float>(), ids.data_ptr<int64_t>(),
                                 rest.data_ptr<float>(), rows, (int)V, (int)k, (float)inv_temp, dtype_code(logits), stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  std::vector<Tensor> r{top, ids, rest, entropy};
  if (labels.has_value()) r.push_back(logp);
  return r;
}

void check_teacher(const Tensor& logits, const Tensor& ids, const Tensor& t, const OptT& rest, bool reverse, const char* op) {
  TORCH_CHECK_VALUE(ids.dim() == 2 && ids.sizes() == t.sizes() && ids.size(1) >= 1 && ids.size(1) <= rb_distill_max_listed(), op,
                    ": the teacher's tokens and their log-probabilities are matrices [rows, 1 .. ", rb_distill_max_listed(), "], not ", ids.sizes(), " and ", t.sizes());
  TORCH_CHECK_VALUE(logits.size(1) <= rb_distill_max_vocab(), op, ": a vocabulary of at most ", rb_distill_max_vocab(), " tokens");
  TORCH_CHECK_VALUE(!reverse || rest.has_value(), op, ": the reverse divergence needs the teacher's rest (a token that the teacher gives nothing costs infinitely much)");
  row_values(ids, at::kLong, logits, ids.size(1), op, "the teacher's tokens");
  row_values(t, at::kFloat, logits, ids.size(1), op, "the tokens' log-probabilities");
  row_values(rest, at::kFloat, logits, -1, op, "the rest's log-probability");
}

std::vector<Tensor> distill_fwd(const Tensor& logits, const Tensor& ids, const Tensor& top_logp, const OptT& rest_logp, bool reverse, double inv_temp,
                                bool need_grad) {
  const char* op = "distill_fwd";
  check_logits(logits, op, inv_temp);
  const int64_t rows = logits.size(0), V = logits.size(1);
  check_teacher(logits, ids, top_logp, rest_logp, reverse, op);
  const int64_t k = ids.size(1);
  const auto* id = ids.data_ptr<int64_t>();
  const auto *t = top_logp.data_ptr<float>(), *tr = rest_logp.has_value() ? rest_logp->data_ptr<float>() : nullptr;
  c10::cuda::CUDAGuard guard(logits.device());
  auto f = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({rows}, f), lse_rest, g_rest, g_listed, ids_out;
  if (need_grad) {
    lse_rest = at::empty({rows}, f);
    g_rest = at::empty({rows}, f);
    g_listed = at::empty({rows, k}, f);
    ids_out = at::empty({rows, k}, f.dtype(at::kInt));
  }
  const int rc = rb_distill_fwd(logits.data_ptr(), logits.stride(0), id, t, tr, reverse, loss.data_ptr<float>(), need_grad ? lse_rest.data_ptr<float>() : nullptr,
                                need_grad ? g_rest.data_ptr<float>() : nullptr, need_grad ? g_listed.data_ptr<float>() : nullptr,
                                need_grad ? ids_out.data_ptr<int>() : nullptr, rows, (int)V, (int)k, (float)inv_temp, dtype_code(logits), stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  if (!need_grad) return {loss};
  return {loss, lse_rest, g_rest, g_listed, ids_out};
}

// a bound of all gradients of the logits
Tensor distill_peak(const Tensor& g_rest, const Tensor& g_listed, const Tensor& g_loss, double inv_temp) {
  const char* op = "distill_peak";
  TORCH_CHECK(g_rest.is_cuda() && g_listed.dim() == 2, op, ": gradients of rows on a CUDA device");
  const int64_t k = g_listed.size(1);
  const auto* gk = static_cast<const float*>(row_values(g_listed, at::kFloat, g_rest, k, op, "the tokens' gradients"));
  const auto* gr = static_cast<const float*>(row_values(g_rest, at::kFloat, g_rest, -1, op, "the rest's gradient"));
  const auto* g = static_cast<const float*>(row_values(g_loss, at::kFloat, g_rest, -1, op, "the loss's gradient"));
  c10::cuda::CUDAGuard guard(g_rest.device());
  Tensor peak = new_peak(g_rest);
  const int rc = rb_distill_peak(gr, gk, g, static_cast<uint32_t*>(peak.data_ptr()), g_rest.size(0), (int)k, (float)inv_temp, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  return peak;
}

Tensor distill_bwd(const Tensor& logits, const Tensor& lse_rest, const Tensor& g_rest, const Tensor& g_listed, const Tensor& ids, const Tensor& g_loss,
                   double inv_temp, const OptT& out, const OptT& peak) {
  const char* op = "distill_bwd";
  check_logits(logits, op, inv_temp);
  TORCH_CHECK(ids.dim() == 2, op, ": the tokens are a matrix");
  const int64_t k = ids.size(1);
  const auto* id = static_cast<const int*>(row_values(ids, at::kInt, logits, k, op, "the tokens"));
  const auto* gk = static_cast<const float*>(row_values(g_listed, at::kFloat, logits, k, op, "the tokens' gradients"));
  const auto* lr = static_cast<const float*>(row_values(lse_rest, at::kFloat, logits, -1, op, "lse_rest"));
  const auto* gr = static_cast<const float*>(row_values(g_rest, at::kFloat, logits, -1, op, "the rest's gradient"));
  const auto* g = static_cast<const float*>(row_values(g_loss, at::kFloat, logits, -1, op, "the loss's gradient"));
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor d = gradient_like(logits, out, op, logits.scalar_type() == at::kFloat);
  const int rc = rb_distill_bwd(logits.data_ptr(), logits.stride(0), lr, gr, gk, id, g, peak_of(peak, logits, op), d.data_ptr(), d.stride(0), logits.size(0),
                                (int)logits.size(1), (int)k, (float)inv_temp, dtype_code(logits), dtype_code(d), stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  return d;
}

void check_head(const Tensor& h, const Tensor& w, const char* op, double inv_temp) {
  TORCH_CHECK(h.is_cuda() && w.device() == h.device() && h.dim() == 2 && w.dim() == 2 && h.size(1) == w.size(1) && h.stride(1) == 1 && w.stride(1) == 1, op,
              ": hidden states [rows, H] and a head [vocabulary, H] on one CUDA device, unit inner stride");
  attn_check();
  TORCH_CHECK(h.scalar_type() == w.scalar_type() && h.element_size() == 2, op, ": 16-bit operands of one type");
  TORCH_CHECK(w.size(0) > 0 && w.size(0) <= 0x7ffe0000LL && h.size(0) <= 0x7ffe0000LL && good_factor(inv_temp), op, ": bad sizes or temperature");
}

// A first derivative that is asked for with a graph (create_graph) and then differentiated again is an error, not a zero.
Tensor once(const Tensor& d, const char* op) {
  if (!at::GradMode::is_enabled()) return d;
  Tensor t = d.detach();
  t.set_requires_grad(true);
  return (*std::make_shared<torch::autograd::DelayedError>(std::string(op) + " has no second derivative", 1))({t})[0];
}

// Native, as short batches wait for the host: as Python functions forward and backward of 16 x 32000 logits took 75 (statistics) and 100 us (distillation).
class LogprobEntropy : public torch::autograd::Function<LogprobEntropy> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const OptT& mask, double inv_temp) {
    auto r = token_stats(logits, labels, mask, inv_temp);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, labels, mask.has_value() ? *mask : Tensor(), r[2], r[1]});
    ctx->saved_data["inv_temp"] = inv_temp;
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    auto given = [](const Tensor& t) { return t.defined() ? OptT(t) : OptT(); };
    ++unseen_launches;
    return {once(token_stats_bwd(s[0], s[1], given(s[2]), s[3], s[4], fp32(given(g[0])), fp32(given(g[1])), ctx->saved_data["inv_temp"].toDouble(), OptT()),
                 "logprob_entropy_from_logits"), Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> logprob_entropy(const Tensor& logits_in, const Tensor& labels_in, const OptT& mask, double inv_temp) {
  const char* op = "logprob_entropy_from_logits";
  const Tensor logits = unit_rows(logits_in), labels = whole_numbers(labels_in, op, "labels");
  check_logits(logits, op, inv_temp);
  row_values(labels, at::kLong, logits, -1, op, "labels");
  const OptT m = packed(mask);
  mask_rows(m, logits, op);
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    check_capture(logits, op);
    return LogprobEntropy::apply(logits, labels, m, inv_temp);
  }
  auto r = token_stats(logits, labels, m, inv_temp);
  r.pop_back();
  return r;
}

class DistillLoss : public torch::autograd::Function<DistillLoss> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& t, const OptT& rest, bool reverse, double inv_temp) {
    auto r = distill_fwd(logits, ids, t, rest, reverse, inv_temp, true);
    ctx->save_for_backward({logits, r[1], r[2], r[3], r[4]});
    ctx->saved_data["inv_temp"] = inv_temp;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto s = ctx->get_saved_variables();
    ++unseen_launches;
    return {once(distill_bwd(s[0], s[1], s[2], s[3], s[4], fp32(g[0]), ctx->saved_data["inv_temp"].toDouble(), OptT(), OptT()), "distill_loss_from_logits"), Tensor(), Tensor(),
            Tensor(), Tensor(), Tensor()};
  }
};

Tensor distill_loss(const Tensor& logits_in, const Tensor& ids_in, const Tensor& t_in, const OptT& rest_in, bool reverse, double inv_temp) {
  const char* op = "distill_loss_from_logits";
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(t_in.requires_grad() || (rest_in.has_value() && rest_in->requires_grad())), op,
                    ": the teacher's log-probabilities get no gradient (detach them)");
  const Tensor logits = unit_rows(logits_in), ids = whole_numbers(ids_in, op, "the teacher's tokens"), t = fp32(t_in);
  const OptT rest = fp32(rest_in);
  check_logits(logits, op, inv_temp);
  check_teacher(logits, ids, t, rest, reverse, op);
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    check_capture(logits, op);
    return DistillLoss::apply(logits, ids, t, rest, reverse, inv_temp);
  }
  return distill_fwd(logits, ids, t, rest, reverse, inv_temp, false)[0];
}

// mask rows beside hidden states: [rows, at least vocabulary / 8]
const uint8_t* head_mask(const OptT& mask, const Tensor& h, int64_t V, const char* op) {
  if (!mask.has_value()) return nullptr;
  TORCH_CHECK(mask->device() == h.device() && mask->scalar_type() == at::kByte && mask->dim() == 2 && mask->is_contiguous() && mask->size(0) == h.size(0) &&
                  mask->size(1) * 8 >= V, op, ": the mask is a packed uint8 matrix [rows, at least vocabulary / 8]");
  return mask->data_ptr<uint8_t>();
}

// keep: also the weights fp16 [rows, vocabulary] and the maxima that they stand against, for head_grad
std::vector<Tensor> head_stats(const Tensor& h, const Tensor& w, const Tensor& labels, const OptT& mask, double inv_temp, bool keep, int64_t num_sms,
                               bool rounded) {
  const char* op = "head_stats";
  check_head(h, w, op, inv_temp);
  const int64_t rows = h.size(0), V = w.size(0);
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, h, -1, op, "labels"));
  c10::cuda::CUDAGuard guard(h.device());
  auto f = h.options().dtype(at::kFloat);
  Tensor logp = at::empty({rows}, f), entropy = at::empty({rows}, f), lse = at::empty({rows}, f), scratch = at::empty({rows * rb_head_stats_scratch((int)V)}, f);
  const int64_t pitch = (V + 7) / 8 * 8;
  Tensor kept = keep ? at::empty({rows, pitch}, f.dtype(at::kHalf)) : Tensor();
  const int rc = rb_head_stats(h.data_ptr(), w.data_ptr(), h.stride(0), w.stride(0), lab, head_mask(mask, h, V, op), mask_bytes(mask), scratch.data_ptr<float>(),
                               keep ? kept.data_ptr() : nullptr, pitch, logp.data_ptr<float>(), entropy.data_ptr<float>(), lse.data_ptr<float>(), (int)rows, (int)V, (int)h.size(1), (float)inv_temp,
                               rounded, dtype_code(h), (int)num_sms, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  if (!keep) return {logp, entropy, lse};
  return {logp, entropy, lse, kept, scratch.slice(0, 0, rows * ((V + 255) / 256 * 2)).clone()};
}

// a bound of all d logits
Tensor head_grad_peak(const Tensor& labels, const Tensor& entropy, const OptT& g_logp, const OptT& g_entropy, double inv_temp) {
  const char* op = "head_grad_peak";
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, entropy, -1, op, "labels"));
  const auto* e = static_cast<const float*>(row_values(entropy, at::kFloat, entropy, -1, op, "entropy"));
  const auto* gl = static_cast<const float*>(row_values(g_logp, at::kFloat, entropy, -1, op, "the log-probability's gradient"));
  const auto* ge = static_cast<const float*>(row_values(g_entropy, at::kFloat, entropy, -1, op, "the entropy's gradient"));
  c10::cuda::CUDAGuard guard(entropy.device());
  Tensor peak = new_peak(entropy);
  const int rc = rb_head_grad_peak(lab, e, gl, ge, static_cast<uint32_t*>(peak.data_ptr()), (int)entropy.size(0), (float)inv_temp, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  return peak;
}

// d logits of rows [row0, row0 + out.size(0)) from what head_stats kept
void head_grad(const Tensor& kept, const Tensor& maxima, const Tensor& labels, const OptT& mask, const Tensor& lse, const Tensor& entropy, const OptT& g_logp,
               const OptT& g_entropy, double inv_temp, Tensor out, int64_t row0, const OptT& peak) {
  const char* op = "head_grad";
  const int64_t all = kept.size(0), rows = out.size(0), V = out.size(1);
  TORCH_CHECK(kept.is_cuda() && kept.dim() == 2 && kept.is_contiguous() && kept.scalar_type() == at::kHalf && kept.size(1) == (V + 7) / 8 * 8 && row0 >= 0 &&
                  row0 + rows <= all, op, ": the kept weights are fp16 rows of the vocabulary");
  TORCH_CHECK(out.device() == kept.device() && out.element_size() == 2 && out.dim() == 2 && out.stride(1) == 1, op, ": a 16-bit destination");
  TORCH_CHECK(maxima.device() == kept.device() && maxima.scalar_type() == at::kFloat && maxima.numel() == all * ((V + 255) / 256 * 2), op, ": bad maxima");
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, kept, -1, op, "labels"));
  const auto* l = static_cast<const float*>(row_values(lse, at::kFloat, kept, -1, op, "lse"));
  const auto* e = static_cast<const float*>(row_values(entropy, at::kFloat, kept, -1, op, "entropy"));
  const auto* gl = static_cast<const float*>(row_values(g_logp, at::kFloat, kept, -1, op, "the log-probability's gradient"));
  const auto* ge = static_cast<const float*>(row_values(g_entropy, at::kFloat, kept, -1, op, "the entropy's gradient"));
  c10::cuda::CUDAGuard guard(kept.device());
  const int rc = rb_head_grad(kept.data_ptr<at::Half>() + row0 * kept.size(1), kept.size(1), maxima.data_ptr<float>(), lab, head_mask(mask, kept, V, op), mask_bytes(mask),
                              l, e, gl, ge, peak_of(peak, kept, op), out.data_ptr(), out.stride(0), (int)row0, (int)rows, (int)all, (int)V, (float)inv_temp, dtype_code(out),
                              stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
}

void head_stats_bwd(const Tensor& h, const Tensor& w, const Tensor& labels, const OptT& mask, const Tensor& lse, const Tensor& entropy, const OptT& g_logp,
                    const OptT& g_entropy, double inv_temp, Tensor out, int64_t num_sms, const OptT& peak, bool rounded) {
  const char* op = "head_stats_bwd";
  check_head(h, w, op, inv_temp);
  const int64_t rows = h.size(0), V = w.size(0);
  const auto* lab = static_cast<const int64_t*>(row_values(labels, at::kLong, h, -1, op, "labels"));
  const auto* l = static_cast<const float*>(row_values(lse, at::kFloat, h, -1, op, "lse"));
  const auto* e = static_cast<const float*>(row_values(entropy, at::kFloat, h, -1, op, "entropy"));
  const auto* gl = static_cast<const float*>(row_values(g_logp, at::kFloat, h, -1, op, "the log-probability's gradient"));
  const auto* ge = static_cast<const float*>(row_values(g_entropy, at::kFloat, h, -1, op, "the entropy's gradient"));
  TORCH_CHECK(out.device() == h.device() && out.scalar_type() == h.scalar_type() && out.dim() == 2 && out.size(0) == rows && out.size(1) == V &&
                  out.stride(1) == 1, op, ": the destination is [rows, vocabulary] of the operands' type");
  c10::cuda::CUDAGuard guard(h.device());
  const int rc = rb_head_stats_bwd(h.data_ptr(), w.data_ptr(), h.stride(0), w.stride(0), lab, head_mask(mask, h, V, op), mask_bytes(mask), l, e, gl, ge,
                                   peak_of(peak, h, op), out.data_ptr(), out.stride(0), (int)rows, (int)V, (int)h.size(1), (float)inv_temp, rounded, dtype_code(h),
                                   (int)num_sms, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
}

// out [rows, H] = d [rows, vocabulary] x w [vocabulary, H], the sum in `splits` parts; peak: taken back from the scale of d
void head_dhidden(const Tensor& d, const Tensor& w, Tensor out, int64_t splits, int64_t num_sms, const OptT& peak) {
  const char* op = "head_dhidden";
  TORCH_CHECK(d.is_cuda() && w.device() == d.device() && out.device() == d.device() && d.dim() == 2 && w.dim() == 2 && d.size(1) == w.size(0) && d.stride(1) == 1 &&
                  w.stride(1) == 1 && out.is_contiguous() && out.dim() == 2 && out.size(0) == d.size(0) && out.size(1) == w.size(1), op, ": bad shapes");
  TORCH_CHECK(d.scalar_type() == w.scalar_type() && out.scalar_type() == w.scalar_type() && w.element_size() == 2, op, ": 16-bit operands of one type");
  c10::cuda::CUDAGuard guard(d.device());
  Tensor parts = at::empty({splits > 1 ? splits : 0, d.size(0), w.size(1)}, d.options().dtype(at::kFloat));
  const int rc = rb_head_dhidden(d.data_ptr(), w.data_ptr(), d.stride(0), w.stride(0), peak_of(peak, d, op), parts.data_ptr<float>(), out.data_ptr(), (int)d.size(0),
                                 (int)w.size(1), (int)d.size(1), (int)splits, dtype_code(d), (int)num_sms, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
  unseen_launches += splits > 1 ? 2 : 1;
}

// out [vocabulary, H], of the operands' type or fp32, = or with `add` += d^T x h, fp16, taken back from the scale of d
void head_dweight(const Tensor& d, const Tensor& h, Tensor out, bool add, int64_t num_sms, const Tensor& peak) {
  const char* op = "head_dweight";
  TORCH_CHECK(d.is_cuda() && h.device() == d.device() && out.device() == d.device() && d.dim() == 2 && h.dim() == 2 && d.size(0) == h.size(0) && d.stride(1) == 1 &&
                  h.stride(1) == 1 && out.is_contiguous() && out.dim() == 2 && out.size(0) == d.size(1) && out.size(1) == h.size(1), op, ": bad shapes");
  TORCH_CHECK(d.scalar_type() == at::kHalf && h.scalar_type() == at::kHalf, op, ": fp16 operands");
  c10::cuda::CUDAGuard guard(d.device());
  const int rc = rb_head_dweight(d.data_ptr(), h.data_ptr(), d.stride(0), h.stride(0), peak_of(peak, d, op), out.data_ptr(), (int)d.size(0), (int)h.size(1), (int)d.size(1),
                                 dtype_code(d), dtype_code(out), add, (int)num_sms, stream());
  TORCH_CHECK(rc == 0, op, " failed with code ", rc);
}

// rows that a TMA descriptor can describe: unit inner stride, 16-byte aligned rows
Tensor tma_rows(const Tensor& x) {
  if (x.stride(1) != 1 || x.stride(0) % 8 != 0 || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15)) return x.clone(at::MemoryFormat::Contiguous);
  return x;
}

// The gradient buffer in a leaf's .grad that products can be added to, if its gradient may go past autograd's own accumulation
Tensor flat_gradient(const Tensor& w, bool flat) {
  if (!flat || !w.is_leaf()) return Tensor();
  const Tensor g = w.grad();
  const bool fits = g.defined() && g.device() == w.device() && g.sizes() == w.sizes() && g.is_contiguous() && (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15) == 0 &&
                    (g.scalar_type() == at::kFloat || g.scalar_type() == w.scalar_type());
  return fits && gradient_goes_past(w, false) ? g : Tensor();
}

// Native for the same reason as the functions on logits: a step of few rows waits for the host (64 rows forward and backward 190 us as a Python function).
class HeadLogprobEntropy : public torch::autograd::Function<HeadLogprobEntropy> {
 public:
  // log-probability, entropy, log-sum-exp and, where kept, the weights and the maxima that they stand against
  static std::vector<Tensor> statistics(const Tensor& hidden, const Tensor& weight, const Tensor& labels, const OptT& mask, double inv_temp, int64_t chunk, bool keep,
                                        bool rounded, int64_t num_sms) {
    const char* op = "lm_head_logprobs_entropy";
    const int64_t T = hidden.size(0), H = hidden.size(1), V = weight.size(0), mask_row = mask_bytes(mask);
    c10::cuda::CUDAGuard guard(hidden.device());
    const Tensor h = tma_rows(hidden);
    const int64_t step = keep ? T : std::min(chunk, std::max<int64_t>(T, 1)), pitch = (V + 7) / 8 * 8;
    auto f = h.options().dtype(at::kFloat);
    Tensor logp = at::empty({T}, f), entropy = at::empty({T}, f), lse = at::empty({T}, f), scratch = at::empty({step * rb_head_stats_scratch((int)V)}, f);
    const Tensor kept = keep ? at::empty({T, pitch}, f.dtype(at::kHalf)) : Tensor();
    const uint8_t* m = head_mask(mask, h, V, op);
    for (int64_t s = 0; s < T; s += step) {
      const int rc = rb_head_stats(static_cast<const char*>(h.data_ptr()) + s * h.stride(0) * 2, weight.data_ptr(), h.stride(0), weight.stride(0),
                                   labels.data_ptr<int64_t>() + s, m ? m + s * mask_row : nullptr, mask_row, scratch.data_ptr<float>(),
                                   keep ? kept.data_ptr() : nullptr, pitch, logp.data_ptr<float>() + s, entropy.data_ptr<float>() + s, lse.data_ptr<float>() + s,
                                   (int)std::min(step, T - s), (int)V, (int)H, (float)inv_temp, rounded, dtype_code(h), (int)num_sms, stream());
      TORCH_CHECK(rc == 0, op, " failed with code ", rc);
    }
    if (!keep) return {logp, entropy, lse, Tensor(), Tensor()};
    return {logp, entropy, lse, kept, scratch.slice(0, 0, T * ((V + 255) / 256 * 2)).clone()};
  }
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& labels, const OptT& mask,
                                                double inv_temp, int64_t chunk, int64_t keep_bytes, bool flat, bool rounded, int64_t num_sms) {
    // keep the weights from width 1024 on: forming and reading them costs what the product of width 512 does (us, both passes up to d logits, kept / formed again:
    // 8192 x 4096 x 32000 1583 / 2715, 2047 x 1024 x 50257 352 / 408, 8192 x 512 x 32000 484 / 486)
    const int64_t T = hidden.size(0);
    const bool keep = T > 256 && hidden.size(1) >= 1024 && 2 * T * weight.size(0) <= keep_bytes;
    const auto r = statistics(hidden, weight, labels, mask, inv_temp, chunk, keep, rounded, num_sms);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({hidden, weight, labels, mask.has_value() ? *mask : Tensor(), r[2], r[1], r[3], r[4]});
    ctx->saved_data["inv_temp"] = inv_temp;
    ctx->saved_data["chunk"] = chunk;
    ctx->saved_data["flat"] = flat;
    ctx->saved_data["rounded"] = rounded;
    ctx->saved_data["num_sms"] = num_sms;
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const char* op = "lm_head_logprobs_entropy";
    torch::autograd::variable_list out(10);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor h = tma_rows(saved[0]), w = saved[1], labels = saved[2], mask = saved[3], lse = saved[4], entropy = saved[5], kept = saved[6], maxima = saved[7];
    const double inv_temp = ctx->saved_data["inv_temp"].toDouble();
    const int num_sms = (int)ctx->saved_data["num_sms"].toInt(), rounded = ctx->saved_data["rounded"].toBool();
    const int64_t T = h.size(0), H = h.size(1), V = w.size(0), pitch = (V + 7) / 8 * 8, mask_row = mask.defined() ? mask.size(1) : 0;
    const int64_t step = std::min<int64_t>(ctx->saved_data["chunk"].toInt(), std::max<int64_t>(T, 1));
    const int dt = dtype_code(h);
    c10::cuda::CUDAGuard guard(h.device());
    attn_check();
    const Tensor gl = g[0].defined() ? fp32(g[0]) : Tensor(), ge = g[1].defined() ? fp32(g[1]) : Tensor();
    const Tensor d = at::empty({std::min(step, T), pitch}, h.options());
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const int64_t* lab = labels.data_ptr<int64_t>();
    // in fp16 d logits leave scaled by their largest size, as those of a mean lie below its smallest number: the products are taken back from it in fp32
    const Tensor peak = dt == 2 && T > 0 ? new_peak(h) : Tensor();
    const uint32_t* pk = peak.defined() ? static_cast<const uint32_t*>(peak.data_ptr()) : nullptr;
    Tensor dh = need_h ? at::empty({T, H}, h.options()) : Tensor(), dw, buffer, parts;
    if (need_w) {
      buffer = flat_gradient(w, ctx->saved_data["flat"].toBool());
      if (buffer.defined() && buffer.scalar_type() != at::kFloat && T > step) buffer = Tensor();      // (16 bits would be rounded once a chunk)
      dw = buffer.defined()   ? buffer
           : T > step || T == 0 ? at::zeros({V, H}, h.options().dtype(at::kFloat))
                                : at::empty({V, H}, h.options());
    }
    const bool add = need_w && (buffer.defined() || dw.scalar_type() == at::kFloat);
    const uint8_t* m = mask.defined() ? mask.data_ptr<uint8_t>() : nullptr;
    auto at_row = [](const Tensor& t, int64_t s) { return t.defined() ? t.data_ptr<float>() + s : nullptr; };
    if (pk) {
      const int rc = rb_head_grad_peak(lab, at_row(entropy, 0), at_row(gl, 0), at_row(ge, 0), static_cast<uint32_t*>(peak.data_ptr()), (int)T, (float)inv_temp, stream());
      TORCH_CHECK(rc == 0, op, ": the gradients' peak failed with code ", rc);
      ++unseen_launches;
    }
    for (int64_t s = 0; s < T; s += step) {
      const int64_t n = std::min(step, T - s);
      const char* hs = static_cast<const char*>(h.data_ptr()) + s * h.stride(0) * 2;
      int rc;
      if (kept.defined())
        rc = rb_head_grad(kept.data_ptr<at::Half>() + s * pitch, pitch, maxima.data_ptr<float>(), lab, m, mask_row, at_row(lse, 0), at_row(entropy, 0), at_row(gl, 0),
                          at_row(ge, 0), pk, d.data_ptr(), pitch, (int)s, (int)n, (int)T, (int)V, (float)inv_temp, dt, stream());
      else
        rc = rb_head_stats_bwd(hs, w.data_ptr(), h.stride(0), w.stride(0), lab + s, m ? m + s * mask_row : nullptr, mask_row, at_row(lse, s), at_row(entropy, s),
                               at_row(gl, s), at_row(ge, s), pk, d.data_ptr(), pitch, (int)n, (int)V, (int)H, (float)inv_temp, rounded, dt, num_sms, stream());
      TORCH_CHECK(rc == 0, op, ": d logits failed with code ", rc);
      ++unseen_launches;
      if (need_h) {       // [n, V] x [V, H]
        void* to = static_cast<char*>(dh.data_ptr()) + s * H * 2;
        const int splits = rb_head_dhidden_splits((int)n, (int)H, (int)V, num_sms);
        if (splits > 1 || pk) {
          if (splits > 1 && (!parts.defined() || parts.numel() < splits * n * H)) parts = at::empty({splits * n * H}, h.options().dtype(at::kFloat));
          rc = rb_head_dhidden(d.data_ptr(), w.data_ptr(), pitch, w.stride(0), pk, splits > 1 ? parts.data_ptr<float>() : nullptr, to, (int)n, (int)H, (int)V, splits, dt, num_sms, stream());
        } else {
          rc = rb_gemm_tcgen05(d.data_ptr(), w.data_ptr(), to, nullptr, (int)n, (int)H, (int)V, pitch, w.stride(0), H, 0, 1, dt, dt, 0, 0, num_sms, -1, stream());
        }
        TORCH_CHECK(rc == 0, op, ": d hidden failed with code ", rc);
        unseen_launches += splits > 1 ? 2 : 1;
      }
      if (need_w) {       // [n, V]^T x [n, H]
        if (pk)
          rc = rb_head_dweight(d.data_ptr(), hs, pitch, h.stride(0), pk, dw.data_ptr(), (int)n, (int)H, (int)V, dt, dtype_code(dw), add, num_sms, stream());
        else
          rc = rb_gemm_tcgen05(d.data_ptr(), hs, dw.data_ptr(), nullptr, (int)V, (int)H, (int)n, pitch, h.stride(0), H, 1, 1, dt, dtype_code(dw), add, 0, num_sms, -1,
                               stream());
        TORCH_CHECK(rc == 0, op, ": d weight failed with code ", rc);
        ++unseen_launches;
      }
    }
    if (need_h) out[0] = once(dh, op);
    if (need_w && !buffer.defined()) out[1] = once(dw.scalar_type() == w.scalar_type() ? dw : dw.to(w.scalar_type()), op);
    return out;
  }
};

// For 16-bit operands as a TMA descriptor takes them; flat: the weight's gradient buffer is its .grad
torch::autograd::variable_list head_logprob_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& labels_in, const OptT& mask_in, double inv_temp, int64_t chunk,
                                                    int64_t keep_bytes, bool flat, int64_t num_sms, bool rounded) {
  const char* op = "lm_head_logprobs_entropy";
  TORCH_CHECK_VALUE(good_factor(inv_temp) && chunk >= 1, op, ": the temperature lies between 1e-30 and 1e30 and a chunk is one row at least");
  TORCH_CHECK_VALUE(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1) && weight.size(0) > 0 && hidden.device() == weight.device() &&
                        hidden.scalar_type() == weight.scalar_type(), op, ": hidden states [T, H] and a head [V, H] of one type and device");
  TORCH_CHECK(weight.element_size() == 2 && weight.stride(1) == 1 && weight.stride(0) % 8 == 0 && hidden.size(1) % 8 == 0 && weight.size(0) <= 0x7ffe0000LL &&
                  hidden.size(0) <= 0x7ffe0000LL && (reinterpret_cast<uintptr_t>(weight.data_ptr()) & 15) == 0, op, ": operands that the products cannot take");
  attn_check();
  const Tensor labels = whole_numbers(labels_in, op, "labels");
  const OptT mask = packed(mask_in);
  row_values(labels, at::kLong, hidden, -1, op, "labels");
  TORCH_CHECK_VALUE(!mask.has_value() || (mask->device() == hidden.device() && mask->scalar_type() == at::kByte && mask->dim() == 2 && mask->size(0) == hidden.size(0) &&
                                          mask->size(1) * 8 >= weight.size(0)), op, ": the mask is a packed uint8 matrix [rows, at least vocabulary / 8]");
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad())) {
    check_capture(hidden, op);
    check_capture(weight, op);
    return HeadLogprobEntropy::apply(hidden, weight, labels, mask, inv_temp, chunk, keep_bytes, flat, rounded, num_sms);
  }
  const auto r = HeadLogprobEntropy::statistics(hidden, weight, labels, mask, inv_temp, chunk, false, rounded, num_sms);
  return {r[0], r[1]};
}

}  // namespace

void register_vocab_ops(torch::Library& m) {
  m.def("native_vocab_launches() -> int", []() -> int64_t { return unseen_launches.exchange(0); });
  m.def("logprob_entropy(Tensor logits, Tensor labels, Tensor? mask, float inv_temp) -> Tensor[]", &logprob_entropy);
  m.def("distill_loss(Tensor logits, Tensor ids, Tensor top_logp, Tensor? rest_logp, bool reverse, float inv_temp) -> Tensor", &distill_loss);
  m.def("token_stats(Tensor logits, Tensor labels, Tensor? mask, float inv_temp) -> Tensor[]", &token_stats);
  m.def("token_stats_bwd(Tensor logits, Tensor labels, Tensor? mask, Tensor lse, Tensor entropy, Tensor? g_logp, Tensor? g_entropy, float inv_temp, "
        "Tensor(a!)? out) -> Tensor", &token_stats_bwd);
  m.def("top_logprobs(Tensor logits, int k, Tensor? labels, Tensor? mask, float inv_temp) -> Tensor[]", &top_logprobs);
  m.def("head_logprob_entropy(Tensor hidden, Tensor weight, Tensor labels, Tensor? mask, float inv_temp, int chunk, int keep_bytes, bool flat, int num_sms, "
        "bool rounded=False) -> Tensor[]",
        &head_logprob_entropy);
  m.def("head_stats(Tensor h, Tensor w, Tensor labels, Tensor? mask, float inv_temp, bool keep, int num_sms, bool rounded=False) -> Tensor[]", &head_stats);
  m.def("head_grad(Tensor kept, Tensor maxima, Tensor labels, Tensor? mask, Tensor lse, Tensor entropy, Tensor? g_logp, Tensor? g_entropy, float inv_temp, Tensor(a!) out, "
        "int row0, Tensor? peak=None) -> ()", &head_grad);
  m.def("head_grad_peak(Tensor labels, Tensor entropy, Tensor? g_logp, Tensor? g_entropy, float inv_temp) -> Tensor", &head_grad_peak);
  m.def("head_dweight(Tensor d, Tensor h, Tensor(a!) out, bool add, int num_sms, Tensor peak) -> ()", &head_dweight);
  m.def("head_stats_bwd(Tensor h, Tensor w, Tensor labels, Tensor? mask, Tensor lse, Tensor entropy, Tensor? g_logp, Tensor? g_entropy, float inv_temp, "
        "Tensor(a!) out, int num_sms, Tensor? peak=None, bool rounded=False) -> ()", &head_stats_bwd);
  m.def("head_dhidden(Tensor d, Tensor w, Tensor(a!) out, int splits, int num_sms, Tensor? peak=None) -> ()", &head_dhidden);
  m.def("head_dhidden_splits(int rows, int width, int vocab, int num_sms) -> int",
        [](int64_t m, int64_t n, int64_t v, int64_t sms) -> int64_t { return rb_head_dhidden_splits((int)m, (int)n, (int)v, (int)sms); });
  m.def("distill_fwd(Tensor logits, Tensor ids, Tensor top_logp, Tensor? rest_logp, bool reverse, float inv_temp, bool need_grad) -> Tensor[]", &distill_fwd);
  m.def("distill_bwd(Tensor logits, Tensor lse_rest, Tensor g_rest, Tensor g_listed, Tensor ids, Tensor g_loss, float inv_temp, Tensor(a!)? out, "
        "Tensor? peak=None) -> Tensor", &distill_bwd);
  m.def("distill_peak(Tensor g_rest, Tensor g_listed, Tensor g_loss, float inv_temp) -> Tensor", &distill_peak);
}
