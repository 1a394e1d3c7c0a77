// Root-mean-square norm of each row, with the residual's addition before it and an output in 8 bits:
//
//     h = x + residual (rounded to x's type, which is what the next layer's residual and the backward read)
//     r = 1 / sqrt(mean(h^2) + eps),  n = h r,  y = n w
//     backward: g = gy w,  gx = gh + r (g - n mean(g n)),  gw = sum over rows of gy n
//
// with gh the gradient that reaches h past the norm; gx is the gradient of x and of the residual. Statistics and sums
// are float32. Bound by memory: a forward reads x and residual and writes h and y (or 1 byte per value and 4 per block
// of 128), the backward reads gy, h and gh and writes gx; each exactly once, a row in registers between the passes (gh of over
// 16384 columns is read after the sum).
//
// A row takes a wave (up to 2048 columns; four rows to a workgroup, no barrier), a workgroup of 256 (up to 8192) or
// one of 1024 threads (up to 32768), eight consecutive columns to a thread and vector, so that 16 lanes hold a block
// of 128 and find its largest magnitude without leaving the row of lanes. The weight gradient sums rows in registers
// over a workgroup's rows, then the workgroups' sums in a fixed order in a second launch: no atomics, the same bits
// each time.
//
// 8192 x 4096 bfloat16 with a residual: forward 47 us (5.7 TB/s), backward 51 and its weights' sums 7; 3001 x 1000 float32: 10.6,
// 10.2 and 2.7; one row: 3.3, a launch. A copy of large tensors reaches 4.7 TB/s on this card: part of these is still in the
// caches.
#include <algorithm>

#include "block_fp8.h"

namespace omt {

constexpr int64_t kNormMaxDim = 32768;

struct NormArgs {
  const void *x, *residual, *weight;
  void *y, *h;
  float* rstd;
  uint8_t* q;
  float* scale;
  int64_t rows, dim;
  float eps;
  int weight_f32;
};

template <bool VEC>
__device__ __forceinline__ f32x8 load_weight(const void* w, int f32, int64_t c, int64_t dim) {
  return f32 ? load8<VEC>((const float*)w, c, dim) : load8<VEC>((const __bf16*)w, c, dim);
}

// Sum over the RT threads of a row, in every one of them; `red` holds a float per wave. All RT threads call it.
template <int RT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (RT > 64) {
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < RT / 64; ++i) v += red[i];
  }
  return v;
}

template <class T, bool VEC, int RT, int NV>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) rms_norm_fwd_kernel(NormArgs a) {
  __shared__ float red[16];
  const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t row = RT == 64 ? group * 4 + (threadIdx.x >> 6) : group;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  if (row >= a.rows) return;  // a whole wave where no barrier follows, or the workgroup
  const int64_t base = row * a.dim;
  f32x8 v[NV];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(i * RT + t) * 8;
    v[i] = load8<VEC>((const T*)a.x + base, c, a.dim);
    if (a.residual) {
      v[i] = rounded8(v[i] + load8<VEC>((const T*)a.residual + base, c, a.dim), (const T*)nullptr);
      store8<VEC>((T*)a.h + base, c, a.dim, v[i]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  }
  const float r = 1.f / sqrtf(row_sum<RT>(ss, red) / (float)a.dim + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = r;
  const int64_t blocks = (a.dim + kFp8Block - 1) / kFp8Block;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(i * RT + t) * 8;
    const f32x8 y = v[i] * r * load_weight<VEC>(a.weight, a.weight_f32, c, a.dim);
    if (a.y) store8<VEC>((T*)a.y + base, c, a.dim, y);
    if (a.q) {
      const float s = block_scale(row16_max(abs_bits8(y)));
      store_fp8x8<VEC>(a.q + base, c, a.dim, pack_fp8x8(y, 1.f / s));
      if ((t & 15) == 0 && c < a.dim) a.scale[row * blocks + c / kFp8Block] = s;
    }
  }
}

struct NormBwdArgs {
  const void *gy, *gh, *h, *weight;
  const float* rstd;
  void* gx;
  float* parts;  // [gridDim.x][dim], or null where no weight gradient is asked for
  int64_t rows, dim;
  int weight_f32;
};

template <class T, bool VEC, int RT, int NV>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) rms_norm_bwd_kernel(NormBwdArgs a) {
  constexpr int ROWS = RT == 64 ? 4 : 1;  // rows of a workgroup at a time
  __shared__ float red[16];
  __shared__ f32x4 sums[ROWS == 4 ? 3 * 64 * NV * 2 : 1];
  int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int sub = RT == 64 ? threadIdx.x >> 6 : 0;
  // Whether a thread's registers hold the weight and its gradient through all rows, and gh through a row's sum. At 32768
  // columns they do not: the gradient is held in LDS, each thread's sums in its own place, and the others are loaded where
  // they are used (2048 x 32768 float32 253 us for 440 with registers spilled to memory, bfloat16 144 for 438).
  constexpr bool kHold = RT * NV <= 2048;
  __shared__ f32x4 held[kHold ? 1 : NV * 2 * RT];
  f32x8 w[kHold ? NV : 1], gw[kHold ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (kHold) w[i] = load_weight<VEC>(a.weight, a.weight_f32, (int64_t)(i * RT + t) * 8, a.dim), gw[i] = f32x8{};
    else held[i * 2 * RT + t] = held[(i * 2 + 1) * RT + t] = f32x4{};
  }
  for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    const int64_t base = row * a.dim;
    const float r = a.rstd[row];
    // (opaque: what follows from it, as whether a column is there, would sit in registers through all rows)
    if constexpr (!kHold) asm volatile("" : "+v"(t));
    f32x8 g[NV], n[NV], gh[kHold ? NV : 1];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (int64_t)(i * RT + t) * 8;
      const f32x8 gy = load8<VEC>((const T*)a.gy + base, c, a.dim);
      n[i] = load8<VEC>((const T*)a.h + base, c, a.dim) * r;
      if constexpr (kHold) gh[i] = a.gh ? load8<VEC>((const T*)a.gh + base, c, a.dim) : f32x8{};  // on its way during the sum
      if constexpr (kHold) {
        gw[i] += gy * n[i];
      } else if (a.parts) {
        const f32x8 p = gy * n[i];
        held[i * 2 * RT + t] += f32x4{p[0], p[1], p[2], p[3]};
        held[(i * 2 + 1) * RT + t] += f32x4{p[4], p[5], p[6], p[7]};
      }
      g[i] = gy * (kHold ? w[kHold ? i : 0] : load_weight<VEC>(a.weight, a.weight_f32, c, a.dim));
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(g[i][e], n[i][e], dot);
    }
    const float mean = row_sum<RT>(dot, red) / (float)a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (int64_t)(i * RT + t) * 8;
      if constexpr (!kHold) gh[0] = a.gh ? load8<VEC>((const T*)a.gh + base, c, a.dim) : f32x8{};
      store8<VEC>((T*)a.gx + base, c, a.dim, (g[i] - n[i] * mean) * r + gh[kHold ? i : 0]);
    }
  }
  if (!a.parts) return;
  if constexpr (ROWS == 4) {  // the four waves' sums, in wave order
    if (sub > 0)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        sums[(((sub - 1) * NV + i) * 2) * 64 + t] = f32x4{gw[i][0], gw[i][1], gw[i][2], gw[i][3]};
        sums[(((sub - 1) * NV + i) * 2 + 1) * 64 + t] = f32x4{gw[i][4], gw[i][5], gw[i][6], gw[i][7]};
      }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      for (int k = 0; k < 3; ++k) {
        const f32x4 lo = sums[((k * NV + i) * 2) * 64 + t], hi = sums[((k * NV + i) * 2 + 1) * 64 + t];
        gw[i] += f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (!kHold) {
      const f32x4 lo = held[i * 2 * RT + t], hi = held[(i * 2 + 1) * RT + t];
      gw[0] = f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
    store8<false>(a.parts + (int64_t)blockIdx.x * a.dim, (int64_t)(i * RT + t) * 8, a.dim, gw[kHold ? i : 0]);
  }
}

// gw[c] = sum over the workgroups' sums: 16 columns to a workgroup, 64 threads a column, each a strided share in order,
// then their sums in order
template <class W>
__global__ void __launch_bounds__(1024) rms_norm_weight_kernel(const float* __restrict__ parts, int count, int64_t dim,
                                                               W* __restrict__ gw) {
  __shared__ float red[64][17];
  const int l = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + l;
  float s = 0.f;
  if (c < dim)
    for (int p = k; p < count; p += 64) s += parts[(int64_t)p * dim + c];
  red[k][l] = s;
  __syncthreads();
  if (k < 8) {
    s = 0.f;
    for (int i = 0; i < 8; ++i) s += red[k * 8 + i][l];
  }
  __syncthreads();
  if (k < 8) red[k][l] = s;
  __syncthreads();
  if (k == 0 && c < dim) {
    for (int i = 1; i < 8; ++i) s += red[i][l];
    gw[c] = (W)s;
  }
}

// Bound by memory: 8192 x 4096 bfloat16 20 us, 5 TB/s
template <bool VEC, class T>
__global__ void __launch_bounds__(256) quantize_fp8_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                           int64_t vecs, int pow2, uint8_t* __restrict__ q,
                                                           float* __restrict__ scale) {
  // 16 lanes to a block of 128, `vecs` (a multiple of 16) vectors of eight to a row
  const int64_t total = rows * vecs, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    const int64_t row = i / vecs, c = (i - row * vecs) * 8;
    const f32x8 v = load8<VEC>(x + row * cols, c, cols);
    const uint32_t m = row16_max(abs_bits8(v));
    const float s = pow2 ? block_scale_pow2(m) : block_scale(m);
    store_fp8x8<VEC>(q + row * cols, c, cols, pack_fp8x8(v, 1.f / s));
    if ((threadIdx.x & 15) == 0) scale[i / 16] = s;
  }
}

// a block of 128 x 128 to a workgroup, in registers (8192 x 4096 bfloat16: 18 us, 5.6 TB/s)
template <bool VEC, class T>
__global__ void __launch_bounds__(256) quantize_fp8_weight_kernel(const T* __restrict__ w, int64_t rows, int64_t cols,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t red[16];
  const int64_t c = (int64_t)blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
  const int64_t r0 = (int64_t)blockIdx.y * kFp8Block + (threadIdx.x >> 4);
  f32x8 v[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = r0 + 16 * i < rows ? load8<VEC>(w + (r0 + 16 * i) * cols, c, cols) : f32x8{};
    m = max_u32(m, abs_bits8(v[i]));
  }
  m = row16_max(m);
  if ((threadIdx.x & 15) == 0) red[threadIdx.x >> 4] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max_u32(m, red[i]);
  const float s = block_scale(m), inv = 1.f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (r0 + 16 * i < rows) store_fp8x8<VEC>(q + (r0 + 16 * i) * cols, c, cols, pack_fp8x8(v[i], inv));
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// ---- host -------------------------------------------------------------------------------------------------------------

static bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}
static int norm_check(const char* fn, int dtype, int wdtype, int64_t rows, int64_t dim) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "%s: dtype %d", fn, dtype);
  if (wdtype != OMT_DT_F32 && wdtype != dtype)
    return fail(OMT_INVALID, "%s: weight dtype %d beside dtype %d", fn, wdtype, dtype);
  if (rows < 0 || dim < 1) return fail(OMT_INVALID, "%s: %lld rows of %lld", fn, (long long)rows, (long long)dim);
  if (dim > kNormMaxDim) return fail(OMT_UNSUPPORTED, "%s: rows of %lld (at most %lld)", fn, (long long)dim,
                                     (long long)kNormMaxDim);
  if (rows > INT32_MAX) return fail(OMT_UNSUPPORTED, "%s: %lld rows", fn, (long long)rows);
  return OMT_OK;
}
// Calls f(RT, NV) as integral constants for rows of `dim`.
template <class F>
static void for_dim(int64_t dim, F f) {
  using std::integral_constant;
  if (dim <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (dim <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (dim <= 2048) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (dim <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (dim <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (dim <= 16384) f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
}
// Workgroups of the backward: four to a CU, each summing the weight gradient of at least four rounds of rows (where there
// are as many as 256 workgroups), so that their sums stay a small part of the traffic.
static int64_t norm_groups(int64_t rows, int64_t dim) {
  const int64_t rounds = cdiv(rows, dim <= 2048 ? 4 : 1);
  return std::max<int64_t>(1, std::min(rounds, std::max<int64_t>(256, std::min<int64_t>(cdiv(rounds, 4), 1024))));
}

}  // namespace omt

using namespace omt;

OMT_EXPORT int omt_rms_norm_fwd(int dtype, int weight_dtype, int64_t rows, int64_t dim, const void* x,
                                const void* residual, const void* weight, float eps, void* y, void* h, float* rstd,
                                void* q, float* scale, void* stream) {
  if (int e = norm_check("omt_rms_norm_fwd", dtype, weight_dtype, rows, dim)) return e;
  if (rows == 0) return OMT_OK;
  if (!x || !weight || (!y && !q) || (q && !scale) || (residual && !h))
    return fail(OMT_INVALID, "omt_rms_norm_fwd: null pointer");
  const bool vec = dim % 8 == 0 && aligned16({x, residual, weight, y, h, q});
  const NormArgs a{x, residual, weight, y, h, rstd, (uint8_t*)q, scale, rows, dim, eps, weight_dtype == OMT_DT_F32};
  for_dim(dim, [&](auto rt, auto nv) {
    constexpr int RT = decltype(rt)::value, NV = decltype(nv)::value;
    // a dimension of the grid holds fewer than 2^32 threads: 2^21 workgroups along it, the rest along the other
    const int64_t groups = RT == 64 ? cdiv(rows, 4) : rows, along = std::min<int64_t>(groups, 1 << 21);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)along, (unsigned)cdiv(groups, along)), dim3(RT == 64 ? 256 : RT), 0,
                         stream_of(stream), a);
    };
    if (dtype == OMT_DT_F32) vec ? go(rms_norm_fwd_kernel<float, true, RT, NV>) : go(rms_norm_fwd_kernel<float, false, RT, NV>);
    else vec ? go(rms_norm_fwd_kernel<__bf16, true, RT, NV>) : go(rms_norm_fwd_kernel<__bf16, false, RT, NV>);
  });
  return launch_check("rms_norm_fwd_kernel");
}

OMT_EXPORT size_t omt_rms_norm_bwd_workspace(int64_t rows, int64_t dim) {
  if (rows < 0 || dim < 1 || dim > kNormMaxDim) return 0;
  return (size_t)(norm_groups(rows, dim) * dim) * sizeof(float);
}

OMT_EXPORT int omt_rms_norm_bwd(int dtype, int weight_dtype, int64_t rows, int64_t dim, const void* gy, const void* gh,
                                const void* h, const void* weight, const float* rstd, void* gx, void* gweight,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = norm_check("omt_rms_norm_bwd", dtype, weight_dtype, rows, dim)) return e;
  if (!weight || (rows > 0 && (!gy || !h || !rstd || !gx))) return fail(OMT_INVALID, "omt_rms_norm_bwd: null pointer");
  if (rows == 0 && !gweight) return OMT_OK;
  if (gweight && (!workspace || workspace_bytes < omt_rms_norm_bwd_workspace(rows, dim)))
    return fail(OMT_INVALID, "omt_rms_norm_bwd: workspace of %zu bytes", workspace_bytes);
  const int64_t groups = norm_groups(rows, dim);
  const bool vec = dim % 8 == 0 && aligned16({gy, gh, h, weight, gx});
  const NormBwdArgs a{gy, gh, h, weight, rstd, gx, gweight ? (float*)workspace : nullptr, rows, dim,
                      weight_dtype == OMT_DT_F32};
  for_dim(dim, [&](auto rt, auto nv) {
    constexpr int RT = decltype(rt)::value, NV = decltype(nv)::value;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(RT == 64 ? 256 : RT), 0, stream_of(stream), a);
    };
    if (dtype == OMT_DT_F32) vec ? go(rms_norm_bwd_kernel<float, true, RT, NV>) : go(rms_norm_bwd_kernel<float, false, RT, NV>);
    else vec ? go(rms_norm_bwd_kernel<__bf16, true, RT, NV>) : go(rms_norm_bwd_kernel<__bf16, false, RT, NV>);
  });
  if (int e = launch_check("rms_norm_bwd_kernel")) return e;
  if (!gweight) return OMT_OK;
  const dim3 grid((unsigned)cdiv(dim, 16));
  if (weight_dtype == OMT_DT_F32)
    hipLaunchKernelGGL(rms_norm_weight_kernel<float>, grid, dim3(1024), 0, stream_of(stream), (const float*)workspace,
                       (int)groups, dim, (float*)gweight);
  else
    hipLaunchKernelGGL(rms_norm_weight_kernel<__bf16>, grid, dim3(1024), 0, stream_of(stream), (const float*)workspace,
                       (int)groups, dim, (__bf16*)gweight);
  return launch_check("rms_norm_weight_kernel");
}

OMT_EXPORT int omt_quantize_fp8(int dtype, int64_t rows, int64_t cols, const void* x, int pow2, void* q, float* scale,
                                void* stream) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "omt_quantize_fp8: dtype %d", dtype);
  if (rows < 0 || cols < 1) return fail(OMT_INVALID, "omt_quantize_fp8: %lld rows of %lld", (long long)rows, (long long)cols);
  if (rows == 0) return OMT_OK;
  if (!x || !q || !scale) return fail(OMT_INVALID, "omt_quantize_fp8: null pointer");
  const bool vec = cols % 8 == 0 && aligned16({x, q});
  const int64_t vecs = cdiv(cols, kFp8Block) * 16;
  const dim3 grid(grid1d(rows * vecs, 256, 1 << 16));
  auto go = [&](auto kernel, auto* p) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream_of(stream), p, rows, cols, vecs, pow2, (uint8_t*)q, scale);
  };
  if (dtype == OMT_DT_F32)
    vec ? go(quantize_fp8_kernel<true, float>, (const float*)x) : go(quantize_fp8_kernel<false, float>, (const float*)x);
  else
    vec ? go(quantize_fp8_kernel<true, __bf16>, (const __bf16*)x) : go(quantize_fp8_kernel<false, __bf16>, (const __bf16*)x);
  return launch_check("quantize_fp8_kernel");
}

OMT_EXPORT int omt_quantize_fp8_weight(int dtype, int64_t rows, int64_t cols, const void* w, void* q, float* scale,
                                       void* stream) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "omt_quantize_fp8_weight: dtype %d", dtype);
  if (rows < 1 || cols < 1)
    return fail(OMT_INVALID, "omt_quantize_fp8_weight: %lld x %lld", (long long)rows, (long long)cols);
  if (cdiv(rows, kFp8Block) > 65535 || cols > INT32_MAX)
    return fail(OMT_UNSUPPORTED, "omt_quantize_fp8_weight: %lld x %lld", (long long)rows, (long long)cols);
  if (!w || !q || !scale) return fail(OMT_INVALID, "omt_quantize_fp8_weight: null pointer");
  const bool vec = cols % 8 == 0 && aligned16({w, q});
  const dim3 grid((unsigned)cdiv(cols, kFp8Block), (unsigned)cdiv(rows, kFp8Block));
  auto go = [&](auto kernel, auto* p) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream_of(stream), p, rows, cols, (uint8_t*)q, scale);
  };
  if (dtype == OMT_DT_F32)
    vec ? go(quantize_fp8_weight_kernel<true, float>, (const float*)w) : go(quantize_fp8_weight_kernel<false, float>, (const float*)w);
  else
    vec ? go(quantize_fp8_weight_kernel<true, __bf16>, (const __bf16*)w) : go(quantize_fp8_weight_kernel<false, __bf16>, (const __bf16*)w);
  return launch_check("quantize_fp8_weight_kernel");
}
