// torch.ops.omt.*: the feed-forward sublayer's operators (residual RMS norm, 8-bit quantization and matrix products, the
// gated block and its backward) over libomt_hip.so, on tensors of the device and on torch.cuda tensors alike. No
// counterpart in the reference. The Python entry points are omarchy_mac_torch.hip_ops (functions) and
// omarchy_mac_torch.ffn (differentiable functions and modules).
//
// Arguments are checked here: a wrong type or device raises TypeError, a wrong shape or value ValueError, sizes that no
// kernel covers NotImplementedError. Operands that are not contiguous, or not on 16 bytes, are copied first.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include "omt_torch.h"

namespace omt {

namespace {

using OptTensor = std::optional<Tensor>;
constexpr int64_t kBlock = 128;
constexpr at::ScalarType kFp8 = at::kFloat8_e4m3fn;

int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
bool on_gpu(const Tensor& t) { return t.device().type() == kDev || t.device().is_cuda(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? OMT_DT_F32 : OMT_DT_BF16; }

// t, contiguous and on 16 bytes, after checking it against a type, and the device and shape of the other operands
Tensor take(const Tensor& t, const char* name, at::ScalarType type, const Tensor* beside = nullptr,
            at::OptionalIntArrayRef shape = std::nullopt) {
  TORCH_CHECK_TYPE(t.defined() && on_gpu(t) && t.scalar_type() == type, name, ": expected ", type,
                   " on the HIP device, got ", t.defined() ? t.scalar_type() : at::ScalarType::Undefined, " on ",
                   t.defined() ? t.device() : c10::Device(c10::kCPU));
  if (beside)
    TORCH_CHECK_VALUE(t.device() == beside->device(), name, ": on ", t.device(), ", the other operands on ",
                      beside->device());
  if (shape) TORCH_CHECK_VALUE(t.sizes().equals(*shape), name, ": expected ", *shape, ", got ", t.sizes());
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
at::ScalarType real_type(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.defined() && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16), name,
                   ": expected float32 or bfloat16 on the HIP device, got ",
                   t.defined() ? t.scalar_type() : at::ScalarType::Undefined);
  return t.scalar_type();
}
struct Rows {
  int64_t rows, cols;
};
Rows rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, ": expected rows of at least one value, got ", t.sizes());
  return {t.numel() / t.size(-1), t.size(-1)};
}
// `shape` with its last dimension replaced
std::vector<int64_t> with_last(IntArrayRef shape, int64_t last) {
  auto v = shape.vec();
  v.back() = last;
  return v;
}
Tensor take_scale(const Tensor& s, const char* name, const Tensor& q) {
  return take(s, name, at::kFloat, &q, with_last(q.sizes(), blocks(q.size(-1))));
}
struct Weight8 {
  Tensor q, s;
};
Weight8 take_weight8(const Tensor& q, const Tensor& s, const char* name, const char* scale_name, int64_t cols,
                     const Tensor& beside) {
  Tensor c = take(q, name, kFp8, &beside);
  TORCH_CHECK_VALUE(c.dim() == 2 && c.size(0) >= 1 && c.size(1) == cols, name, ": expected [rows, ", cols, "], got ",
                    c.sizes());
  return {c, take(s, scale_name, at::kFloat, &beside, IntArrayRef{blocks(c.size(0)), blocks(cols)})};
}

// (straight from the allocator: an at::empty through the dispatcher takes twice as long, and a small call makes three)
Tensor make(const Tensor& like, IntArrayRef shape, at::ScalarType type) {
  if (is_dev(like)) return empty_dev(shape, type);
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
Tensor make_scale(const Tensor& like, IntArrayRef shape) {
  return make(like, with_last(shape, blocks(shape.back())), at::kFloat);
}
void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* rawf(const Tensor& t) { return (float*)raw(t); }

// Where a call runs: t's device, its current stream, and scratch memory of that stream.
struct Site {
  c10::OptionalDeviceGuard guard;
  void* stream;
  Tensor ws;
  explicit Site(const Tensor& t) {
    if (!is_dev(t) && t.device().index() != c10::hip::current_device()) guard.reset_device(t.device());
    stream = cur_stream();
  }
  void* scratch(const Tensor& like, size_t bytes) {
    if (bytes) ws = make(like, {(int64_t)bytes}, at::kByte);
    return raw(ws);
  }
};
void ok(int status, const char* what) {
  if (status == OMT_UNSUPPORTED) TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": ", omt_last_error());
  check(status, what);
}
// A call under the device's lock (library calls on one stream are serialized), with its debug check.
#define FFN_OP(name) \
  OMT_LOCK;          \
  struct AtEnd {     \
    ~AtEnd() noexcept(false) { if (debug_mode() && !std::uncaught_exceptions()) debug_point("omt::" name); } \
  } at_end_

struct NormOperands {
  Tensor x, weight, other;
  Rows r;
};
NormOperands norm_operands(const Tensor& x_, const Tensor& weight_, const OptTensor& other_, const char* xn,
                           const char* on) {
  Tensor x = take(x_, xn, real_type(x_, xn));
  const Rows r = rows_of(x, xn);
  TORCH_CHECK_TYPE(weight_.scalar_type() == x.scalar_type() || weight_.scalar_type() == at::kFloat,
                   "weight: expected ", x.scalar_type(), " or float32, got ", weight_.scalar_type());
  Tensor weight = take(weight_, "weight", weight_.scalar_type(), &x, IntArrayRef{r.cols});
  Tensor other = defined(other_) ? take(*other_, on, x.scalar_type(), &x, x.sizes()) : Tensor();
  return {x, weight, other, r};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm(const Tensor& x_, const Tensor& weight_, const OptTensor& residual,
                                            double eps) {
  FFN_OP("rms_norm");
  const auto o = norm_operands(x_, weight_, residual, "x", "residual");
  Site at(o.x);
  Tensor y = make(o.x, o.x.sizes(), o.x.scalar_type());
  Tensor h = o.other.defined() ? make(o.x, o.x.sizes(), o.x.scalar_type()) : Tensor();
  Tensor rstd = make(o.x, o.x.sizes().slice(0, o.x.dim() - 1), at::kFloat);
  ok(omt_rms_norm_fwd(dtype_of(o.x), dtype_of(o.weight), o.r.rows, o.r.cols, raw(o.x), raw(o.other), raw(o.weight),
                      (float)eps, raw(y), raw(h), rawf(rstd), nullptr, nullptr, at.stream),
     "rms_norm");
  return {y, h, rstd};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8(const Tensor& x_, const Tensor& weight_, const OptTensor& residual,
                                                double eps) {
  FFN_OP("rms_norm_fp8");
  const auto o = norm_operands(x_, weight_, residual, "x", "residual");
  Site at(o.x);
  Tensor q = make(o.x, o.x.sizes(), kFp8), scale = make_scale(o.x, o.x.sizes());
  Tensor h = o.other.defined() ? make(o.x, o.x.sizes(), o.x.scalar_type()) : Tensor();
  ok(omt_rms_norm_fwd(dtype_of(o.x), dtype_of(o.weight), o.r.rows, o.r.cols, raw(o.x), raw(o.other), raw(o.weight),
                      (float)eps, nullptr, raw(h), nullptr, raw(q), rawf(scale), at.stream),
     "rms_norm_fp8");
  return {q, scale, h};
}

std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor& gy_, const Tensor& h_, const Tensor& weight_,
                                             const Tensor& rstd_, const OptTensor& gh, bool weight_grad) {
  FFN_OP("rms_norm_backward");
  const auto o = norm_operands(h_, weight_, gh, "h", "gh");
  Tensor gy = take(gy_, "gy", o.x.scalar_type(), &o.x, o.x.sizes());
  Tensor rstd = take(rstd_, "rstd", at::kFloat, &o.x, o.x.sizes().slice(0, o.x.dim() - 1));
  Site at(o.x);
  Tensor gx = make(o.x, o.x.sizes(), o.x.scalar_type());
  Tensor gw = weight_grad ? make(o.x, {o.r.cols}, o.weight.scalar_type()) : Tensor();
  const size_t need = weight_grad ? omt_rms_norm_bwd_workspace(o.r.rows, o.r.cols) : 0;
  void* ws = at.scratch(o.x, need);
  ok(omt_rms_norm_bwd(dtype_of(o.x), dtype_of(o.weight), o.r.rows, o.r.cols, raw(gy), raw(o.other), raw(o.x),
                      raw(o.weight), rawf(rstd), raw(gx), raw(gw), ws, need, at.stream),
     "rms_norm_backward");
  return {gx, gw};
}

std::tuple<Tensor, Tensor> quantize_fp8(const Tensor& x_, bool pow2) {
  FFN_OP("quantize_fp8");
  Tensor x = take(x_, "x", real_type(x_, "x"));
  const Rows r = rows_of(x, "x");
  Site at(x);
  Tensor q = make(x, x.sizes(), kFp8), scale = make_scale(x, x.sizes());
  ok(omt_quantize_fp8(dtype_of(x), r.rows, r.cols, raw(x), pow2, raw(q), rawf(scale), at.stream), "quantize_fp8");
  return {q, scale};
}

std::tuple<Tensor, Tensor> quantize_fp8_weight(const Tensor& w_) {
  FFN_OP("quantize_fp8_weight");
  Tensor w = take(w_, "w", real_type(w_, "w"));
  TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0, "w: expected a matrix, got ", w.sizes());
  Site at(w);
  Tensor q = make(w, w.sizes(), kFp8), scale = make(w, {blocks(w.size(0)), blocks(w.size(1))}, at::kFloat);
  ok(omt_quantize_fp8_weight(dtype_of(w), w.size(0), w.size(1), raw(w), raw(q), rawf(scale), at.stream),
     "quantize_fp8_weight");
  return {q, scale};
}

Tensor matmul_fp8(const Tensor& a_, const Tensor& a_scale, const Tensor& b_, const Tensor& b_scale,
                  at::ScalarType type) {
  FFN_OP("matmul_fp8");
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16, "dtype: expected bfloat16 or float32, got ", type);
  Tensor a = take(a_, "a", kFp8);
  const Rows r = rows_of(a, "a");
  Tensor sa = take_scale(a_scale, "a's scales", a);
  const Weight8 b = take_weight8(b_, b_scale, "b", "b's scales", r.cols, a);
  const int64_t n = b.q.size(0);
  Site at(a);
  Tensor c = make(a, with_last(a.sizes(), n), type);
  const size_t need = omt_matmul_fp8_workspace(r.rows, n, r.cols, dtype_of(c));
  void* ws = at.scratch(a, need);
  ok(omt_matmul_fp8(r.rows, n, r.cols, raw(a), rawf(sa), raw(b.q), rawf(b.s), dtype_of(c), raw(c), ws, need, at.stream),
     "matmul_fp8");
  return c;
}

struct GluWeights {
  Tensor gate, up;
};
GluWeights glu_weights(const Tensor& gate, const Tensor& up, at::ScalarType type, int64_t k, const Tensor& beside) {
  Tensor g = take(gate, "w_gate", type, &beside);
  TORCH_CHECK_VALUE(g.dim() == 2 && g.size(0) >= 1 && g.size(1) == k, "w_gate: expected [rows, ", k, "], got ", g.sizes());
  return {g, take(up, "w_up", type, &beside, g.sizes())};
}

// (h, x_q, x_scale, g, g_scale, u, u_scale); what `keep` (OMT_KEEP_*) does not ask for is undefined
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> glu(const Tensor& x_, const Tensor& w_gate,
                                                                       const Tensor& w_up, int64_t act, int64_t keep) {
  FFN_OP("glu");
  Tensor x = take(x_, "x", real_type(x_, "x"));
  const Rows r = rows_of(x, "x");
  const GluWeights w = glu_weights(w_gate, w_up, x.scalar_type(), r.cols, x);
  const int64_t f = w.gate.size(0);
  const auto shape = with_last(x.sizes(), f);
  Site at(x);
  Tensor h = make(x, shape, x.scalar_type()), xq, xs, g, gs, u, us;
  if (keep == OMT_KEEP_FP8) {
    xq = make(x, x.sizes(), kFp8), xs = make_scale(x, x.sizes());
    g = make(x, shape, kFp8), gs = make_scale(x, shape);
    u = make(x, shape, kFp8), us = make_scale(x, shape);
  } else if (keep == OMT_KEEP_FULL) {
    g = make(x, shape, x.scalar_type()), u = make(x, shape, x.scalar_type());
  }
  const size_t need = omt_glu_fwd_workspace(dtype_of(x), r.rows, r.cols, f);
  void* ws = at.scratch(x, need);
  ok(omt_glu_fwd(dtype_of(x), r.rows, r.cols, f, (int)act, (int)keep, raw(x), raw(w.gate), raw(w.up), raw(h), raw(xq),
                 rawf(xs), raw(g), rawf(gs), raw(u), rawf(us), ws, need, at.stream),
     "glu");
  return {h, xq, xs, g, gs, u, us};
}

std::tuple<Tensor, Tensor, Tensor> glu_backward(const Tensor& gh_, const Tensor& x_, const OptTensor& x_scale,
                                                const Tensor& g_, const OptTensor& g_scale, const Tensor& u_,
                                                const OptTensor& u_scale, const Tensor& w_gate, const Tensor& w_up,
                                                int64_t act, bool input_grad, bool weight_grad) {
  FFN_OP("glu_backward");
  const at::ScalarType type = real_type(gh_, "gh");
  Tensor gh = take(gh_, "gh", type);
  const Rows r = rows_of(gh, "gh");
  const bool fp8 = defined(x_scale);
  TORCH_CHECK_VALUE(defined(g_scale) == fp8 && defined(u_scale) == fp8, "glu_backward: scales of some values alone");
  const at::ScalarType held = fp8 ? kFp8 : type;
  Tensor x = take(x_, "x", held, &gh), g = take(g_, "g", held, &gh), u = take(u_, "u", held, &gh), xs, gs, us;
  const Rows rx = rows_of(x, "x");
  TORCH_CHECK_VALUE(g.sizes().equals(gh.sizes()) && u.sizes().equals(gh.sizes()) &&
                        with_last(x.sizes(), r.cols) == gh.sizes().vec(),
                    "glu_backward: gh ", gh.sizes(), ", x ", x.sizes(), ", g ", g.sizes(), ", u ", u.sizes(),
                    " do not belong together");
  if (fp8) {
    xs = take_scale(*x_scale, "x's scales", x);
    gs = take_scale(*g_scale, "g's scales", g);
    us = take_scale(*u_scale, "u's scales", u);
  }
  const GluWeights w = glu_weights(w_gate, w_up, type, rx.cols, gh);
  TORCH_CHECK_VALUE(w.gate.size(0) == r.cols, "w_gate: expected ", r.cols, " rows, got ", w.gate.sizes());
  Site at(gh);
  Tensor gx, gwg, gwu;
  if (input_grad) gx = make(gh, x.sizes(), type);
  if (weight_grad) gwg = make(gh, w.gate.sizes(), type), gwu = make(gh, w.up.sizes(), type);
  const size_t need = omt_glu_bwd_workspace(dtype_of(gh), r.rows, rx.cols, r.cols);
  void* ws = at.scratch(gh, need);
  ok(omt_glu_bwd(dtype_of(gh), r.rows, rx.cols, r.cols, (int)act, fp8 ? OMT_KEEP_FP8 : OMT_KEEP_FULL, raw(gh), raw(x),
                 rawf(xs), raw(g), rawf(gs), raw(u), rawf(us), raw(w.gate), raw(w.up), raw(gx), raw(gwg), raw(gwu), ws,
                 need, at.stream),
     "glu_backward");
  return {gx, gwg, gwu};
}

std::tuple<Tensor, Tensor> glu_fp8(const Tensor& x_, const Tensor& x_scale, const Tensor& w_gate,
                                   const Tensor& gate_scale, const Tensor& w_up, const Tensor& up_scale, int64_t act) {
  FFN_OP("glu_fp8");
  Tensor x = take(x_, "x", kFp8);
  const Rows r = rows_of(x, "x");
  Tensor xs = take_scale(x_scale, "x's scales", x);
  const Weight8 g = take_weight8(w_gate, gate_scale, "w_gate", "w_gate's scales", r.cols, x);
  const Weight8 u = take_weight8(w_up, up_scale, "w_up", "w_up's scales", r.cols, x);
  const int64_t f = g.q.size(0);
  TORCH_CHECK_VALUE(u.q.size(0) == f, "w_up: expected ", g.q.sizes(), ", got ", u.q.sizes());
  Site at(x);
  const auto shape = with_last(x.sizes(), f);
  Tensor q = make(x, shape, kFp8), scale = make_scale(x, shape);
  const size_t need = omt_glu_fp8_workspace(r.rows, r.cols, f);
  void* ws = at.scratch(x, need);
  ok(omt_glu_fp8(r.rows, r.cols, f, (int)act, raw(x), rawf(xs), raw(g.q), rawf(g.s), raw(u.q), rawf(u.s), raw(q),
                 rawf(scale), ws, need, at.stream),
     "glu_fp8");
  return {q, scale};
}

}  // namespace

// The same functions for omarchy_mac_torch.hip_ops, without the dispatcher's way (0.6 us of a small call's 6.4)
void bind_ffn(pybind11::module_& m) {
  auto f = m.def_submodule("ffn");
  f.def("rms_norm", torch::wrap_pybind_function(&rms_norm));
  f.def("rms_norm_fp8", torch::wrap_pybind_function(&rms_norm_fp8));
  f.def("rms_norm_backward", torch::wrap_pybind_function(&rms_norm_backward));
  f.def("quantize_fp8", torch::wrap_pybind_function(&quantize_fp8));
  f.def("quantize_fp8_weight", torch::wrap_pybind_function(&quantize_fp8_weight));
  f.def("matmul_fp8", torch::wrap_pybind_function(&matmul_fp8));
  f.def("glu", torch::wrap_pybind_function(&glu));
  f.def("glu_backward", torch::wrap_pybind_function(&glu_backward));
  f.def("glu_fp8", torch::wrap_pybind_function(&glu_fp8));
}

TORCH_LIBRARY_FRAGMENT(omt, m) {
  // (y, h, rstd) / (q, scale, h): h is undefined where there is no residual (it is x)
  m.def("rms_norm(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_fp8(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_backward(Tensor gy, Tensor h, Tensor weight, Tensor rstd, Tensor? gh, bool weight_grad) -> "
        "(Tensor, Tensor)");
  m.def("quantize_fp8(Tensor x, bool pow2) -> (Tensor, Tensor)");
  m.def("quantize_fp8_weight(Tensor w) -> (Tensor, Tensor)");
  m.def("matmul_fp8(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType dtype) -> Tensor");
  m.def("glu(Tensor x, Tensor w_gate, Tensor w_up, int act, int keep) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("glu_backward(Tensor gh, Tensor x, Tensor? x_scale, Tensor g, Tensor? g_scale, Tensor u, Tensor? u_scale, "
        "Tensor w_gate, Tensor w_up, int act, bool input_grad, bool weight_grad) -> (Tensor, Tensor, Tensor)");
  m.def("glu_fp8(Tensor x, Tensor x_scale, Tensor w_gate, Tensor gate_scale, Tensor w_up, Tensor up_scale, int act) -> "
        "(Tensor, Tensor)");
}
// Under every backend, so that an operand elsewhere meets the check above, with its name, rather than the dispatcher's.
TORCH_LIBRARY_IMPL(omt, CompositeExplicitAutograd, m) {
  m.impl("rms_norm", &rms_norm);
  m.impl("rms_norm_fp8", &rms_norm_fp8);
  m.impl("rms_norm_backward", &rms_norm_backward);
  m.impl("quantize_fp8", &quantize_fp8);
  m.impl("quantize_fp8_weight", &quantize_fp8_weight);
  m.impl("matmul_fp8", &matmul_fp8);
  m.impl("glu", &glu);
  m.impl("glu_backward", &glu_backward);
  m.impl("glu_fp8", &glu_fp8);
}

}  // namespace omt
