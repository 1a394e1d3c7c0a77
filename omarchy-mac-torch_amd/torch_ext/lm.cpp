// torch.ops.omt.*: both ends of a language model's training step (embedding and its gradient, losses on logits with theirs,
// AdamW with states in 8 bits or 32) over libomt_hip.so, on tensors of the device and on torch.cuda tensors alike. No counterpart
// in the reference. The Python entry points are omarchy_mac_torch.hip_ops (functions), omarchy_mac_torch.lm (differentiable
// functions) and omarchy_mac_torch.optim (the optimizer).
//
// Arguments are checked here: a wrong type or device raises TypeError, a wrong shape or value ValueError, sizes that no
// kernel covers NotImplementedError.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <algorithm>
#include <utility>

#include "operands.h"

namespace omt {

namespace {

constexpr int64_t kBlock = 128;
constexpr at::ScalarType kFp8 = at::kFloat8_e4m3fn;

Tensor take_tokens(const Tensor& t) {
  TORCH_CHECK_TYPE(t.defined() && on_gpu(t) && (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt),
                   "tokens: expected int64 or int32 on the HIP device, got ", t.scalar_type(), " on ", t.device());
  return t.contiguous();
}
int token_dtype(const Tensor& t) { return t.scalar_type() == at::kLong ? OMT_DT_I64 : OMT_DT_I32; }

Tensor embedding(const Tensor& tokens_, const Tensor& weight_, double scale) {
  OMT_OP("embedding");
  Tensor weight = take(weight_, "weight", real_type(weight_, "weight"));
  Tensor tokens = take_tokens(tokens_);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0, "weight: expected a matrix, got ", weight.sizes());
  TORCH_CHECK_VALUE(tokens.device() == weight.device(), "tokens: on ", tokens.device(), ", the weight on ", weight.device());
  auto shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  Site at(weight);
  Tensor y = make(weight, shape, weight.scalar_type());
  ok(omt_embedding_fwd(dtype_of(weight), token_dtype(tokens), tokens.numel(), weight.size(0), weight.size(1), raw(tokens),
                       raw(weight), (float)scale, raw(y), at.stream),
     "embedding");
  return y;
}

Tensor embedding_backward(const Tensor& gy_, const Tensor& tokens_, int64_t vocab, double scale, int64_t padding_idx) {
  OMT_OP("embedding_backward");
  Tensor gy = take(gy_, "gy", real_type(gy_, "gy"));
  Tensor tokens = take_tokens(tokens_);
  TORCH_CHECK_VALUE(tokens.device() == gy.device(), "tokens: on ", tokens.device(), ", gy on ", gy.device());
  TORCH_CHECK_VALUE(gy.dim() == tokens.dim() + 1 && gy.size(-1) >= 1 &&
                        gy.sizes().slice(0, tokens.dim()).equals(tokens.sizes()),
                    "gy: expected the tokens' shape ", tokens.sizes(), " and a last dimension, got ", gy.sizes());
  TORCH_CHECK_VALUE(vocab >= 1, "vocab: expected at least 1, got ", vocab);
  const int64_t n = tokens.numel(), dim = gy.size(-1);
  Site at(gy);
  Tensor gw = make(gy, {vocab, dim}, gy.scalar_type());
  const size_t need = omt_embedding_bwd_workspace(n, vocab, dim);
  void* ws = at.scratch(gy, need);
  ok(omt_embedding_bwd(dtype_of(gy), token_dtype(tokens), n, vocab, dim, raw(gy), raw(tokens), padding_idx, (float)scale,
                       raw(gw), ws, need, at.stream),
     "embedding_backward");
  return gw;
}

// Logits [sequences, length, vocab] as they lie, if each row is dense, and their labels.
struct Logits {
  Tensor x, labels;
  omt_logits q;
};
Logits take_logits(const Tensor& x_, const Tensor& labels_, int64_t ignore_index) {
  Logits l;
  const at::ScalarType type = real_type(x_, "logits");
  TORCH_CHECK_TYPE(on_gpu(x_), "logits: expected ", type, " on the HIP device, got ", x_.device());
  TORCH_CHECK_VALUE(x_.dim() == 3 && x_.size(2) >= 1, "logits: expected [sequences, length, vocab], got ", x_.sizes());
  l.x = x_.stride(2) == 1 || x_.size(2) == 1 ? x_ : x_.contiguous();
  l.labels = take(labels_, "labels", at::kLong, &l.x, l.x.sizes().slice(0, 2));
  l.q = omt_logits{raw(l.x),       (const int64_t*)raw(l.labels), ignore_index,  l.x.size(0),  l.x.size(1),
                   l.x.size(2),    l.x.stride(0),                 l.x.stride(1), dtype_of(l.x)};
  return l;
}
Tensor make_gradient(const Logits& l, bool asked) { return asked ? make(l.x, l.x.sizes(), l.x.scalar_type()) : Tensor(); }

std::tuple<Tensor, Tensor> token_logps(const Tensor& logits, const Tensor& labels, int64_t ignore_index, bool lse64) {
  OMT_OP("token_logps");
  const Logits l = take_logits(logits, labels, ignore_index);
  Site at(l.x);
  Tensor logps = make(l.x, l.labels.sizes(), at::kFloat), lse = make(l.x, l.labels.sizes(), lse64 ? at::kDouble : at::kFloat);
  ok(lse64 ? omt_token_logps_fwd64(&l.q, rawf(logps), (double*)raw(lse), at.stream)
           : omt_token_logps_fwd(&l.q, rawf(logps), rawf(lse), at.stream),
     "token_logps");
  return {logps, lse};
}

Tensor token_logps_backward(const Tensor& g_, const Tensor& logits, const Tensor& labels, const Tensor& lse_,
                            int64_t ignore_index) {
  OMT_OP("token_logps_backward");
  const Logits l = take_logits(logits, labels, ignore_index);
  const bool lse64 = lse_.defined() && lse_.scalar_type() == at::kDouble;
  Tensor g = take(g_, "g", at::kFloat, &l.x, l.labels.sizes());
  Tensor lse = take(lse_, "lse", lse64 ? at::kDouble : at::kFloat, &l.x, l.labels.sizes());
  Site at(l.x);
  Tensor gx = make_gradient(l, true);
  ok(lse64 ? omt_token_logps_bwd64(&l.q, (const double*)raw(lse), rawf(g), raw(gx), at.stream)
           : omt_token_logps_bwd(&l.q, rawf(lse), rawf(g), raw(gx), at.stream),
     "token_logps_backward");
  return gx;
}

// (loss, rewards, the logits' gradient, undefined where it is not asked for)
std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& labels, const Tensor& reference_,
                                                   double beta, int64_t kind, double smoothing, bool average,
                                                   int64_t ignore_index, bool grad) {
  OMT_OP("preference_loss");
  const Logits l = take_logits(logits, labels, ignore_index);
  TORCH_CHECK_VALUE(l.q.sequences >= 2 && l.q.sequences % 2 == 0, "logits: expected pairs of sequences, got ", l.q.sequences);
  TORCH_CHECK_VALUE(beta > 0, "beta: expected over 0, got ", beta);
  TORCH_CHECK_VALUE(smoothing >= 0 && smoothing <= 1, "smoothing: expected from 0 to 1, got ", smoothing);
  TORCH_CHECK_VALUE(kind == OMT_PREFERENCE_SIGMOID || smoothing == 0, "smoothing: of the sigmoid loss only, got ", smoothing);
  Tensor reference = take(reference_, "reference", at::kFloat, &l.x, IntArrayRef{l.q.sequences});
  Site at(l.x);
  Tensor loss = make(l.x, {}, at::kFloat), rewards = make(l.x, {l.q.sequences}, at::kFloat), gx = make_gradient(l, grad);
  const size_t need = omt_preference_workspace(l.q.sequences, l.q.length);
  void* ws = at.scratch(l.x, need);
  ok(omt_preference_loss(&l.q, rawf(reference), (int)kind, beta, smoothing, average, rawf(loss), rawf(rewards), raw(gx), ws,
                         need, at.stream),
     "preference_loss");
  return {loss, rewards, gx};
}

// (loss, KL term, logps, the logits' gradient, undefined where it is not asked for)
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& labels, const Tensor& old_,
                                                       const Tensor& advantages_, const OptTensor& reference_, double clip_low,
                                                       double clip_high, double kl_weight, bool by_sequence,
                                                       int64_t ignore_index, bool grad) {
  OMT_OP("policy_loss");
  const Logits l = take_logits(logits, labels, ignore_index);
  const IntArrayRef rows = l.labels.sizes();
  Tensor old = take(old_, "old_logps", at::kFloat, &l.x, rows);
  Tensor reference = defined(reference_) ? take(*reference_, "reference", at::kFloat, &l.x, rows) : Tensor();
  TORCH_CHECK_VALUE(clip_low >= 0 && clip_high >= 0, "clip: expected at least 0, got ", clip_low, " and ", clip_high);
  TORCH_CHECK_VALUE(advantages_.dim() == 1 || advantages_.dim() == 2, "advantages: expected [sequences] or [sequences, length], got ",
                    advantages_.sizes());
  const bool each = advantages_.dim() == 2;
  Tensor advantages = take(advantages_, "advantages", at::kFloat, &l.x, each ? rows : rows.slice(0, 1));
  Site at(l.x);
  Tensor loss = make(l.x, {}, at::kFloat), kl = make(l.x, {}, at::kFloat), logps = make(l.x, rows, at::kFloat);
  Tensor gx = make_gradient(l, grad);
  const size_t need = omt_policy_workspace(l.q.sequences, l.q.length, by_sequence);
  void* ws = at.scratch(l.x, need);
  ok(omt_policy_loss(&l.q, rawf(old), rawf(reference), rawf(advantages), each ? l.q.length : 1, each, clip_low, clip_high,
                     kl_weight, by_sequence, rawf(loss), rawf(kl), rawf(logps), raw(gx), ws, need, at.stream),
     "policy_loss");
  return {loss, kl, logps, gx};
}

// after an operator has written t in place: autograd then refuses what it saved of it before
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void scale_by_(const Tensor& x, const Tensor& factor) {
  OMT_OP("scale_by_");
  real_type(x, "x");
  TORCH_CHECK_VALUE(on_gpu(x) && x.is_contiguous(), "x: expected a contiguous tensor on the HIP device");
  Tensor f = take(factor, "factor", at::kFloat, &x);
  TORCH_CHECK_VALUE(f.numel() == 1, "factor: expected one element, got ", f.sizes());
  const char *begin = (const char*)raw(x), *of = (const char*)raw(f);
  if (of >= begin && of < begin + x.nbytes()) f = f.clone();  // an element of x: some threads would read it scaled
  Site at(x);
  ok(omt_scale_by(dtype_of(x), x.numel(), raw(x), rawf(f), at.stream), "scale_by_");
  written(x);
}

// whether two tensors' elements lie in the same order
bool same_layout(const Tensor& a, const Tensor& b) {
  if (!a.sizes().equals(b.sizes())) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}
void check_state(const Tensor& t, const char* name, size_t i, at::ScalarType type, const Tensor& p) {
  TORCH_CHECK_TYPE(t.defined() && t.scalar_type() == type && t.device() == p.device(), name, " ", i, ": expected ", type, " on ",
                   p.device(), ", got ", t.scalar_type(), " on ", t.device());
  TORCH_CHECK_VALUE(same_layout(t, p), name, " ", i, ": expected the parameter's shape and order ", p.sizes(), ", got ", t.sizes(),
                    " with strides ", t.strides());
}
float* check_scale(const Tensor& t, const char* name, size_t i, const Tensor& p) {
  TORCH_CHECK_TYPE(t.defined() && t.scalar_type() == at::kFloat && t.device() == p.device(), name, " ", i,
                   ": expected float32 on ", p.device(), ", got ", t.scalar_type(), " on ", t.device());
  const int64_t blocks = (p.numel() + kBlock - 1) / kBlock;
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == blocks && t.is_contiguous(), name, " ", i, ": expected [", blocks, "], got ",
                    t.sizes());
  return rawf(t);
}
const float* check_scalar(const OptTensor& t, const char* name, const Tensor& p) {
  if (!defined(t)) return nullptr;
  TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat && t->device() == p.device(), name, ": expected float32 on ", p.device(), ", got ",
                   t->scalar_type(), " on ", t->device());
  TORCH_CHECK_VALUE(t->numel() == 1, name, ": expected one element, got ", t->sizes());
  return rawf(*t);
}

// The memory of one call's tensors: what one of them is written to, no other of them may hold.
struct Ranges {
  c10::SmallVector<std::pair<uintptr_t, uintptr_t>, 128> all;  // begin, and twice the end, odd where the memory is only read
  void add(const void* p, int64_t bytes, bool read = false) {
    if (p) all.emplace_back((uintptr_t)p, ((uintptr_t)p + bytes) << 1 | read);
  }
  bool overlap() {
    std::sort(all.begin(), all.end(), [](const auto& a, const auto& b) { return a.first < b.first; });
    uintptr_t any = 0, written = 0;  // where those before end
    for (const auto& [begin, end] : all) {
      if (begin < (end & 1 ? written : any)) return true;
      any = std::max(any, end >> 1);
      if (!(end & 1)) written = std::max(written, end >> 1);
    }
    return false;
  }
};

void adamw_(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
            at::TensorList steps, at::TensorList exp_avg_scales, at::TensorList exp_avg_sq_scales, at::TensorList masters,
            double lr, const OptTensor& lr_dev, double beta1, double beta2, double eps, double weight_decay,
            const OptTensor& grad_scale, const OptTensor& found_inf, bool maximize) {
  OMT_OP("adamw_");
  const size_t n = params.size();
  const bool fp8 = !exp_avg_scales.empty() || !exp_avg_sq_scales.empty();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && steps.size() == n &&
                        (!fp8 || (exp_avg_scales.size() == n && exp_avg_sq_scales.size() == n)) &&
                        (masters.empty() || masters.size() == n),
                    "adamw: lists of one length are needed");
  if (n == 0) return;
  TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas: expected from 0 to below 1, got ", beta1, ", ", beta2);
  const Tensor& first = params[0];
  const at::ScalarType type = real_type(first, "parameter 0"), held = fp8 ? kFp8 : at::kFloat;
  TORCH_CHECK_TYPE(on_gpu(first), "parameter 0: expected a tensor on the HIP device, got one on ", first.device());
  TORCH_CHECK_TYPE(masters.empty() || type == at::kBFloat16, "masters: of bfloat16 parameters only");
  std::vector<omt_adamw_tensor> ts(n);
  Ranges memory;
  std::vector<Tensor> copies;  // gradients whose elements lie in another order
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    TORCH_CHECK_TYPE(p.scalar_type() == type && p.device() == first.device(), "parameter ", i, ": expected ", type, " on ",
                     first.device(), " as the first, got ", p.scalar_type(), " on ", p.device());
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "parameter ", i, ": expected dense, got strides ", p.strides());
    Tensor g = grads[i];
    TORCH_CHECK_TYPE(g.defined() && g.scalar_type() == type && g.device() == p.device() && g.layout() == at::kStrided, "gradient ", i,
                     ": expected dense ", type, " on ", p.device(), " as the parameter, got ", g.scalar_type(), " on ", g.device());
    TORCH_CHECK_VALUE(g.sizes().equals(p.sizes()), "gradient ", i, ": expected ", p.sizes(), ", got ", g.sizes());
    if (!same_layout(g, p)) copies.push_back(g = at::empty_like(p).copy_(g));
    check_state(exp_avgs[i], "exp_avg", i, held, p);
    check_state(exp_avg_sqs[i], "exp_avg_sq", i, held, p);
    if (!masters.empty()) check_state(masters[i], "master", i, at::kFloat, p);
    ts[i] = omt_adamw_tensor{raw(p),
                             raw(g),
                             masters.empty() ? nullptr : rawf(masters[i]),
                             raw(exp_avgs[i]),
                             fp8 ? check_scale(exp_avg_scales[i], "exp_avg_scale", i, p) : nullptr,
                             raw(exp_avg_sqs[i]),
                             fp8 ? check_scale(exp_avg_sq_scales[i], "exp_avg_sq_scale", i, p) : nullptr,
                             check_scalar(steps[i], "step", p),
                             p.numel()};
    TORCH_CHECK_VALUE(ts[i].step, "step ", i, ": expected a tensor");
    const omt_adamw_tensor& t = ts[i];
    if (t.numel == 0) continue;
    const int64_t size = type == at::kFloat ? 4 : 2, held_size = fp8 ? 1 : 4, scales = (t.numel + kBlock - 1) / kBlock * 4;
    memory.add(t.param, t.numel * size);
    memory.add(t.master, t.numel * 4);
    memory.add(t.exp_avg, t.numel * held_size);
    memory.add(t.exp_avg_sq, t.numel * held_size);
    memory.add(t.exp_avg_scale, scales);
    memory.add(t.exp_avg_sq_scale, scales);
    // (a parameter that is its own gradient: each element is read before it is written, by one thread)
    if (t.grad != t.param) memory.add(t.grad, t.numel * size, true);
  }
  TORCH_CHECK_VALUE(!memory.overlap(), "adamw: a parameter, a gradient or a state is given twice, or overlaps another");
  const omt_adamw_params hp{lr,
                            beta1,
                            beta2,
                            weight_decay,
                            eps,
                            check_scalar(lr_dev, "lr", first),
                            check_scalar(grad_scale, "grad_scale", first),
                            check_scalar(found_inf, "found_inf", first),
                            maximize};
  Site at(first);
  ok(omt_adamw(type == at::kFloat ? OMT_DT_F32 : OMT_DT_BF16, fp8 ? 8 : 32, &hp, ts.data(), (int)n, at.stream), "adamw");
  for (auto list : {params, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters})
    for (const Tensor& t : list) written(t);
}

}  // namespace

// The same functions for omarchy_mac_torch.hip_ops, without the dispatcher's way
void bind_lm(pybind11::module_& m) {
  auto f = m.def_submodule("lm");
  f.def("embedding", torch::wrap_pybind_function(&embedding));
  f.def("embedding_backward", torch::wrap_pybind_function(&embedding_backward));
  f.def("token_logps", torch::wrap_pybind_function(&token_logps));
  f.def("token_logps_backward", torch::wrap_pybind_function(&token_logps_backward));
  f.def("preference_loss", torch::wrap_pybind_function(&preference_loss));
  f.def("policy_loss", torch::wrap_pybind_function(&policy_loss));
  f.def("scale_by_", torch::wrap_pybind_function(&scale_by_));
  using List = const std::vector<Tensor>&;
  f.def("adamw_", torch::wrap_pybind_function(+[](List p, List g, List m, List v, List steps, List ms, List vs, List masters, double lr,
                                                  const OptTensor& lr_dev, double b1, double b2, double eps, double wd,
                                                  const OptTensor& scale, const OptTensor& inf, bool maximize) {
          adamw_(p, g, m, v, steps, ms, vs, masters, lr, lr_dev, b1, b2, eps, wd, scale, inf, maximize);
        }));
}

TORCH_LIBRARY_FRAGMENT(omt, m) {
  m.def("embedding(Tensor tokens, Tensor weight, float scale) -> Tensor");
  m.def("embedding_backward(Tensor gy, Tensor tokens, int vocab, float scale, int padding_idx) -> Tensor");
  m.def("token_logps(Tensor logits, Tensor labels, int ignore_index, bool lse64=False) -> (Tensor, Tensor)");
  m.def("token_logps_backward(Tensor g, Tensor logits, Tensor labels, Tensor lse, int ignore_index) -> Tensor");
  m.def("preference_loss(Tensor logits, Tensor labels, Tensor reference, float beta, int kind, float smoothing, bool average, "
        "int ignore_index, bool grad) -> (Tensor, Tensor, Tensor)");
  m.def("policy_loss(Tensor logits, Tensor labels, Tensor old_logps, Tensor advantages, Tensor? reference, float clip_low, "
        "float clip_high, float kl_weight, bool by_sequence, int ignore_index, bool grad) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("scale_by_(Tensor(a!) x, Tensor factor) -> ()");
  m.def("adamw_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, Tensor[] steps, "
        "Tensor(d!)[] exp_avg_scales, Tensor(e!)[] exp_avg_sq_scales, Tensor(f!)[] masters, float lr, Tensor? lr_dev, float beta1, "
        "float beta2, float eps, float weight_decay, Tensor? grad_scale, Tensor? found_inf, bool maximize) -> ()");
}
// Under every backend, so that an operand elsewhere meets the check above, with its name, rather than the dispatcher's.
TORCH_LIBRARY_IMPL(omt, CompositeExplicitAutograd, m) {
  m.impl("embedding", &embedding);
  m.impl("embedding_backward", &embedding_backward);
  m.impl("token_logps", &token_logps);
  m.impl("token_logps_backward", &token_logps_backward);
  m.impl("preference_loss", &preference_loss);
  m.impl("policy_loss", &policy_loss);
  m.impl("scale_by_", &scale_by_);
  m.impl("adamw_", &adamw_);
}

}  // namespace omt
