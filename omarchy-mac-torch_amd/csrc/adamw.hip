// AdamW over many tensors in one launch, parameters and gradients in float32 or bfloat16, states in 32 bits or in 8:
//
//     m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//     p -= lr wd p,  p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A bfloat16 parameter may have a master copy in float32, which is what is updated; the parameter is its rounding. Without one
// the parameter itself is, and an update below half its last place is lost.
//
// In 8 bits a state is e4m3 with a float32 scale for each block of 128 consecutive values of the tensor, the largest magnitude /
// 448. The second moment is held as its root: e4m3 spans 2^18 from its smallest value to its largest, so the root's 2^18 are
// 2^36 of the moment, of which a block of weights needs many; and a value over zero is held as e4m3's smallest at least, since
// a second moment rounded to zero beside a first one that is not makes a step as large as m / eps. Both are rounded to
// nearest. This step's update is from the moments before they are rounded.
//
// Bound by memory: 16 bytes a parameter and its scales' 1/8 in float32 with 8-bit states (28 with 32), 10 in bfloat16, 16 with a
// master copy. Sixteen lanes hold a block of 128, eight values each, and find its largest magnitude in their registers.
// Every operation on the moments is rounded by itself (no contraction), so that what is stored in 8 bits does not depend on
// how a compiler pairs them. The loads are on their way while one lane computes the step's scalars.
//
// In 8 bits, 470 million bfloat16 parameters with masters 1390 us (7.58 GB at 5.45 TB/s), without 840; 8.8 million float32 ones, 19 tensors,
// 26 us (0.14 GB at 5.5 TB/s); 0.2 million bfloat16 ones 7 us, a launch and the scalars' latency.
#include "block_fp8.h"

namespace omt {

constexpr int kAdamwSlots = 32;  // tensors to a launch: their table travels in the kernel's arguments
constexpr int kAdamwThreads = 256;
// Elements to a workgroup, eight to a thread: more of them one after another to a thread, with the next ones' loads ahead, cost more
// in uneven ends than they saved in starts (8.8 million parameters float32 28.3 us with 8, 32.9 with 16, 35.2 with 32 and 41.1 with
// 64; 470 million bfloat16 1401, 1407, 1439 and 1471).
constexpr int kAdamwChunk = kAdamwThreads * 8;
constexpr int64_t kAdamwMaxNumel = (int64_t)kAdamwChunk * ((1 << 24) - 1);  // a launch holds fewer than 2^32 threads
constexpr float kFp8Smallest = 0x1p-9f;

struct AdamwSlot {
  void *p, *m, *v;
  const void* g;
  float *master, *m_scale, *v_scale;
  const float* step;
  int64_t n;
};
struct AdamwTable {
  AdamwSlot s[kAdamwSlots];
  int first[kAdamwSlots + 1];  // first chunk of each slot; first[count] = chunks of the launch
  int count;
};
struct AdamwHyper {
  double lr, beta1, beta2, wd;
  float eps;
  const float *lr_dev, *grad_scale, *found_inf;
  int maximize;
};
static_assert(sizeof(AdamwTable) + sizeof(AdamwHyper) < 4096, "the table travels in the kernel's arguments");

// The scale of a block whose largest magnitude has these bits: times 1/448, for which the block's largest value is e4m3's, 448,
// to within 2^-22.
__device__ __forceinline__ float state_scale(uint32_t amax_bits) {
  return __builtin_bit_cast(float, max_u32(amax_bits, __builtin_bit_cast(uint32_t, kFp8Floor))) * (1.f / kFp8Max);
}

// what all elements of a tensor share
struct AdamwScalars {
  float b1, c1, b2, c2;  // beta, 1 - beta
  float rate, root, over_root, decay, eps, grad;  // root: sqrt(1 - b2^t)
};

// beta^t for the step count t, by squaring, each of which doubles the relative error: within about t 2^-53 of itself, so 1 - beta^t is off by
// t beta^t 2^-53 at most (at beta = 0.999, 4e-14)
__device__ __forceinline__ double power(double beta, double t) {
  double p = 1.0;
  for (uint32_t n = (uint32_t)t; n; n >>= 1, beta *= beta)
    if (n & 1) p *= beta;
  return p;
}

template <class P, bool FP8, bool MASTER>
__global__ void __launch_bounds__(kAdamwThreads) adamw_kernel(const AdamwTable t, const AdamwHyper h) {
#pragma clang fp contract(off)
  constexpr bool RECIPROCAL = FP8 && !MASTER;
  if (h.found_inf && *h.found_inf == 1.f) return;
  __shared__ AdamwScalars shared;
  const int chunk = (int)blockIdx.x;
  int si = 0;
  while (si + 1 < t.count && chunk >= t.first[si + 1]) ++si;
  const AdamwSlot& s = t.s[si];
  const int64_t c = (int64_t)(chunk - t.first[si]) * kAdamwChunk + (int)threadIdx.x * 8, block = c / kFp8Block;
  f32x8 p, g = load8<false>((const P*)s.g, c, s.n), m, v, root;  // on their way while the scalars are computed
  float m_scale = 0.f, v_scale = 0.f;
  if constexpr (MASTER) p = load8<false>(s.master, c, s.n);
  else p = load8<false>((const P*)s.p, c, s.n);
  if constexpr (FP8) {
    m = load8<false>((const uint8_t*)s.m, c, s.n), v = load8<false>((const uint8_t*)s.v, c, s.n);
    if (c < s.n) m_scale = s.m_scale[block], v_scale = s.v_scale[block];
  } else {
    m = load8<false>((const float*)s.m, c, s.n), v = load8<false>((const float*)s.v, c, s.n);
  }
  if (threadIdx.x == 0) {
    const double step = (double)*s.step, lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
    const double root = sqrt(1.0 - power(h.beta2, step));
    shared = {(float)h.beta1, (float)(1.0 - h.beta1), (float)h.beta2, (float)(1.0 - h.beta2),
              (float)(lr / (1.0 - power(h.beta1, step))), (float)root, RECIPROCAL ? (float)(1.0 / root) : 0.f, (float)(lr * h.wd), h.eps,
              (h.maximize ? -1.f : 1.f) / (h.grad_scale ? *h.grad_scale : 1.f)};
  }
  __syncthreads();
  const AdamwScalars k = shared;
  if constexpr (FP8) {
    m *= m_scale;
    v *= v_scale;
    v *= v;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float ge = g[e] * k.grad;
    m[e] = k.b1 * m[e] + k.c1 * ge;
    v[e] = k.b2 * v[e] + k.c2 * ge * ge;
    root[e] = sqrtf(v[e]);
    p[e] -= k.decay * p[e];
    // (By the reciprocal instruction, to float32's last place or two, where bytes are so few that a division takes longer: in 8 bits without
    // masters, 155 million bfloat16 parameters 289 us for 350, 8.8 million float32 ones 25.8 for 26.7; in 32 bits, 842 us for 839 of 155
    // million float32 ones, and with masters, 1434 for 1397 of 470 million in 8 bits, it gained nothing.)
    if constexpr (RECIPROCAL) p[e] -= k.rate * m[e] * __builtin_amdgcn_rcpf(root[e] * k.over_root + k.eps);
    else p[e] -= k.rate * m[e] / (root[e] / k.root + k.eps);
  }
  if constexpr (MASTER) store8<false>(s.master, c, s.n, p);
  store8<false>((P*)s.p, c, s.n, p);
  if constexpr (FP8) {
    const float ms = state_scale(row16_max(abs_bits8(m))), vs = state_scale(row16_max(abs_bits8(root)));
    const float inv = 1.f / vs;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = root[e] * inv;
      root[e] = root[e] > 0.f && q < kFp8Smallest ? kFp8Smallest : q;
    }
    store_fp8x8<false>((uint8_t*)s.m, c, s.n, pack_fp8x8(m, 1.f / ms));
    store_fp8x8<false>((uint8_t*)s.v, c, s.n, pack_fp8x8(root, 1.f));
    if ((threadIdx.x & 15) == 0 && c < s.n) s.m_scale[block] = ms, s.v_scale[block] = vs;
  } else {
    store8<false>((float*)s.m, c, s.n, m);
    store8<false>((float*)s.v, c, s.n, v);
  }
}

}  // namespace omt

using namespace omt;

OMT_EXPORT int omt_adamw(int dtype, int state_bits, const omt_adamw_params* hp, const omt_adamw_tensor* ts, int n, void* stream) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "omt_adamw: dtype %d", dtype);
  if (state_bits != 8 && state_bits != 32) return fail(OMT_INVALID, "omt_adamw: states of %d bits", state_bits);
  if (!hp || (n > 0 && !ts) || n < 0) return fail(OMT_INVALID, "omt_adamw: null pointer or negative count");
  int masters = -1;  // of the tensors that are not empty: whether the first has one
  for (int i = 0; i < n; ++i) {
    const omt_adamw_tensor& t = ts[i];
    if (t.numel < 0 || (t.numel > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || !t.step ||
                                        (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))))
      return fail(OMT_INVALID, "omt_adamw: tensor %d: null pointer or negative size", i);
    if (t.numel > kAdamwMaxNumel) return fail(OMT_UNSUPPORTED, "omt_adamw: tensor %d: %lld elements", i, (long long)t.numel);
    if (t.numel == 0) continue;
    if (masters < 0) masters = t.master != nullptr;
    if ((t.master != nullptr) != masters || (t.master && dtype == OMT_DT_F32))
      return fail(OMT_INVALID, "omt_adamw: tensor %d: master copies are for all tensors of a call, of bfloat16, or for none", i);
  }
  const AdamwHyper h{hp->lr, hp->beta1, hp->beta2, hp->weight_decay, (float)hp->eps, hp->lr_dev, hp->grad_scale, hp->found_inf,
                     hp->maximize};
  for (int i = 0; i < n;) {
    AdamwTable t;
    t.count = 0;
    int64_t chunks = 0;
    for (; i < n && t.count < kAdamwSlots; ++i) {
      const omt_adamw_tensor& a = ts[i];
      const int64_t more = cdiv(a.numel, kAdamwChunk);
      if (chunks + more >= 1 << 24) break;
      if (a.numel == 0) continue;
      t.s[t.count] = {a.param, a.exp_avg, a.exp_avg_sq, a.grad, a.master, a.exp_avg_scale, a.exp_avg_sq_scale, a.step, a.numel};
      t.first[t.count++] = (int)chunks;
      chunks += more;
    }
    if (!t.count) break;
    t.first[t.count] = (int)chunks;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(kAdamwThreads), 0, stream_of(stream), t, h);
    };
    if (dtype == OMT_DT_F32) state_bits == 8 ? go(adamw_kernel<float, true, false>) : go(adamw_kernel<float, false, false>);
    else if (masters == 1) state_bits == 8 ? go(adamw_kernel<__bf16, true, true>) : go(adamw_kernel<__bf16, false, true>);
    else state_bits == 8 ? go(adamw_kernel<__bf16, true, false>) : go(adamw_kernel<__bf16, false, false>);
    if (int e = launch_check("adamw_kernel")) return e;
  }
  return OMT_OK;
}
