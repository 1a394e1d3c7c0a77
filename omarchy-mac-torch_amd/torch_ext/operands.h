// Operands of torch.ops.omt's language-model operators, on tensors of the device and on torch.cuda tensors alike: their checks,
// their outputs, and where a call runs. A wrong type or device raises TypeError, a wrong shape or value ValueError, sizes that no
// kernel covers NotImplementedError. Operands that are not contiguous, or not on 16 bytes, are copied first.
#pragma once

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include "omt_torch.h"

namespace omt {

using OptTensor = std::optional<Tensor>;
inline bool on_gpu(const Tensor& t) { return t.device().type() == kDev || t.device().is_cuda(); }
inline int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? OMT_DT_F32 : OMT_DT_BF16; }

// t, contiguous and on 16 bytes, after checking it against a type, and the device and shape of the other operands
inline Tensor take(const Tensor& t, const char* name, at::ScalarType type, const Tensor* beside = nullptr,
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
inline at::ScalarType real_type(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.defined() && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16), name,
                   ": expected float32 or bfloat16 on the HIP device, got ",
                   t.defined() ? t.scalar_type() : at::ScalarType::Undefined);
  return t.scalar_type();
}
struct Rows {
  int64_t rows, cols;
};
inline Rows rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, ": expected rows of at least one value, got ", t.sizes());
  return {t.numel() / t.size(-1), t.size(-1)};
}
// `shape` with its last dimension replaced
inline std::vector<int64_t> with_last(IntArrayRef shape, int64_t last) {
  auto v = shape.vec();
  v.back() = last;
  return v;
}
// (straight from the allocator: an at::empty through the dispatcher takes twice as long, and a small call makes three)
inline Tensor make(const Tensor& like, IntArrayRef shape, at::ScalarType type) {
  if (is_dev(like)) return empty_dev(shape, type);
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
inline void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* rawf(const Tensor& t) { return (float*)raw(t); }

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
inline void ok(int status, const char* what) {
  if (status == OMT_UNSUPPORTED) TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": ", omt_last_error());
  check(status, what);
}
// A call under the device's lock (library calls on one stream are serialized), with its debug check.
#define OMT_OP(name) \
  OMT_LOCK;          \
  struct AtEnd {     \
    ~AtEnd() noexcept(false) { if (debug_mode() && !std::uncaught_exceptions()) debug_point("omt::" name); } \
  } at_end_

}  // namespace omt
