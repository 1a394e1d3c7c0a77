// Losses on a language model's logits x [sequences][length][vocab] with labels, and their gradients. Of each row whose label
// counts (it is not ignore_index): lse = log(sum exp x), lp = x[label] - lse, and d lp / d x = onehot(label) - exp(x - lse).
//
// token_logps: lp and lse of every row, and the gradient from one of lp.
//
// preference: sequences in pairs, the chosen ones in the first half. With L the sum (or mean) of a sequence's lp and R its
//   reference, d = (L - R of the chosen) - (L - R of the rejected):
//     sigmoid  -(1 - s) log sigmoid(beta d) - s log sigmoid(-beta d)
//     hinge    max(0, 1 - beta d)
//     ipo      (d - 1 / (2 beta))^2
//   and the mean over pairs. The gradient of every lp of a sequence is the same.
//
// policy: r = exp(lp - old), loss of a token -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(ref - lp) - (ref - lp) - 1), and the mean
//   over all tokens, or over sequences of each one's mean.
//
// Rows that do not count are not read, so that nothing in them matters, and get a gradient of zeros; so do rows whose lp has a
// gradient of zero. A label outside the vocabulary makes the loss, and its row's gradient, NaN. Exponentials and their sums over a
// row are float32, what is computed of lp (sums over a sequence, ratios next to the clip's borders) is float64. No atomics: every
// sum runs in a fixed order.
//
// Bound by memory. The gradient needs a row's sum, so a row is read twice, or once where a workgroup holds it in registers
// (policy); a pair's coefficient needs all rows of both sequences, so the preference loss reads its rows twice.
#include <algorithm>

#include "block_fp8.h"

namespace omt {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

struct LogitRows {
  const void* x;
  const int64_t* labels;
  int64_t ignore, length, vocab, sequence_stride, row_stride, rows;
  __device__ __forceinline__ int64_t offset(int64_t row) const {
    return row / length * sequence_stride + row % length * row_stride;
  }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// Over the RT threads of a row, in every one of them; `red` holds a float per wave. All RT threads call it.
template <int RT>
__device__ __forceinline__ float row_max(float v, float* red) {
  v = wave_max(v);
  if constexpr (RT > 64) {
    __syncthreads();  // the previous result has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < RT / 64; ++i) v = fmaxf(v, red[i]);
  }
  return v;
}
template <int RT>
__device__ __forceinline__ float row_total(float v, float* red) {
  v = wave_sum(v);
  if constexpr (RT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < RT / 64; ++i) v += red[i];
  }
  return v;
}

// eight logits from column c on, minus infinity behind the row
template <bool VEC, class T>
__device__ __forceinline__ f32x8 load_logits(const T* p, int64_t c, int64_t cols) {
  f32x8 v = load8<VEC>(p, c, cols);
  if (c + 8 > cols)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e >= cols) v[e] = -kInf;
  return v;
}
__device__ __forceinline__ float max8(f32x8 v) {
  return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
// exp(v - m): the difference first, which is exact or nearly so for what counts
__device__ __forceinline__ float exp_from(float v, float m) { return __builtin_amdgcn_exp2f((v - m) * kLog2e); }

// The largest and the sum of exp(x - largest) of a row of memory, in every one of its RT threads.
struct RowStats {
  float top, sum;
};
template <class T, bool VEC, int RT>
__device__ __forceinline__ RowStats row_stats(const T* x, int64_t vocab, float* red) {
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  float m = -kInf, s = 0.f;
  constexpr int U = 4;
  for (int64_t c0 = (int64_t)t * 8; c0 < vocab; c0 += RT * 8 * U) {
    f32x8 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_logits<VEC>(x, c0 + u * RT * 8, vocab);
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, max8(v[u]));
    // (a thread that has met nothing over minus infinity: differences to 0 instead, so that none is NaN)
    const float from = top == -kInf ? 0.f : top;
    s *= exp_from(m, from);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += exp_from(v[u][e], from);
    m = top;
  }
  const float top = row_max<RT>(m, red), from = top == -kInf ? 0.f : top;
  return {top, row_total<RT>(s * exp_from(m, from), red)};
}

__device__ __forceinline__ bool in_vocab(int64_t label, int64_t vocab) { return (uint64_t)label < (uint64_t)vocab; }
// lp of a label, NaN outside the vocabulary; a row of minus infinities has top - top = NaN in it, as the definition has
template <class T>
__device__ __forceinline__ double label_logp(const T* x, int64_t label, int64_t vocab, RowStats st) {
  if (!in_vocab(label, vocab)) return (double)__builtin_nanf("");
  return ((double)(float)x[label] - (double)st.top) - log((double)st.sum);
}

// ---- statistics of rows ---------------------------------------------------------------------------------------------

// Row of this thread, with RT threads to a row; -1 where there is none (a whole wave, or the workgroup)
template <int RT>
__device__ __forceinline__ int64_t this_row(int64_t rows) {
  const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t row = RT == 64 ? group * 4 + (threadIdx.x >> 6) : group;
  return row < rows ? row : -1;
}

template <class T, bool VEC, int RT>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) token_logps_kernel(LogitRows a, float* logps, float* lse) {
  __shared__ float red[16];
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const bool first = (RT == 64 ? threadIdx.x & 63 : threadIdx.x) == 0;
  const int64_t label = a.labels[row];
  if (label == a.ignore) {
    if (first) logps[row] = 0.f, lse[row] = 0.f;
    return;
  }
  const T* x = (const T*)a.x + a.offset(row);
  const RowStats st = row_stats<T, VEC, RT>(x, a.vocab, red);
  if (first) {
    logps[row] = (float)label_logp(x, label, a.vocab, st);
    lse[row] = (float)((double)st.top + log((double)st.sum));
  }
}

// ---- the gradient of rows -------------------------------------------------------------------------------------------

// c (onehot(label) - p) of the eight columns from c0 on, p = exp(x - lse)
__device__ __forceinline__ f32x8 row_gradient(f32x8 p, float c, int64_t c0, int64_t label) {
  f32x8 g = p * -c;
  if ((uint64_t)(label - c0) < 8)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e == label) g[e] += c;
  return g;
}

template <class T, bool VEC, int RT>
__device__ __forceinline__ void write_zeros(T* g, int64_t vocab) {
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  for (int64_t c = (int64_t)t * 8; c < vocab; c += RT * 8) store8<VEC>(g, c, vocab, f32x8{});
}

// per_row: coefs holds one for each row, else one for each sequence
template <class T, bool VEC, int RT>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) logit_grad_kernel(LogitRows a, const float* lse, const float* coefs,
                                                                         int per_row, T* gx) {
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t label = a.labels[row];
  const float coef = coefs[per_row ? row : row / a.length];
  T* g = gx + row * a.vocab;
  if (label == a.ignore || coef == 0.f) return write_zeros<T, VEC, RT>(g, a.vocab);
  const float c = in_vocab(label, a.vocab) ? coef : __builtin_nanf(""), l = lse[row];
  const T* x = (const T*)a.x + a.offset(row);
  constexpr int U = 4;
  for (int64_t c0 = (int64_t)t * 8; c0 < a.vocab; c0 += RT * 8 * U) {
    f32x8 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load8<VEC>(x, c0 + u * RT * 8, a.vocab);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t cu = c0 + u * RT * 8;
      f32x8 p;
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = exp_from(v[u][e], l);
      store8<VEC>(g, cu, a.vocab, row_gradient(p, c, cu, label));
    }
  }
}

// ---- pairs ----------------------------------------------------------------------------------------------------------

__device__ __forceinline__ double block_sum(double v, double* red) {  // 256 threads, in every one of them
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct PairArgs {
  const int64_t* labels;
  const float *logps, *reference;
  int64_t ignore, length, pairs;
  int kind, average;
  double beta, smoothing;
  float *rewards, *coefs;
  double* losses;
};

// log(1 + exp(-z)) without overflow
__device__ __forceinline__ double softplus_neg(double z) { return (z < 0 ? -z : 0.0) + log1p(exp(z < 0 ? z : -z)); }
__device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

__global__ void __launch_bounds__(256) preference_pair_kernel(PairArgs a) {
  __shared__ double red[4];
  const int64_t pair = blockIdx.x;
  double ratio[2], share[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t seq = pair + k * a.pairs, base = seq * a.length;
    double sum = 0.0, count = 0.0;
    for (int64_t i = threadIdx.x; i < a.length; i += 256)
      if (a.labels[base + i] != a.ignore) sum += (double)a.logps[base + i], count += 1.0;
    sum = block_sum(sum, red);
    count = block_sum(count, red);
    share[k] = a.average ? 1.0 / fmax(count, 1.0) : 1.0;
    ratio[k] = sum * share[k] - (double)a.reference[seq];
  }
  if (threadIdx.x) return;
  const double d = ratio[0] - ratio[1], z = a.beta * d;
  double loss, slope;  // of the loss by d
  if (a.kind == OMT_PREFERENCE_SIGMOID) {
    loss = (1.0 - a.smoothing) * softplus_neg(z) + a.smoothing * softplus_neg(-z);
    slope = a.beta * (a.smoothing - sigmoid(-z));
  } else if (a.kind == OMT_PREFERENCE_HINGE) {
    loss = 1.0 - z < 0.0 ? 0.0 : 1.0 - z;  // (NaN stays NaN)
    slope = 1.0 - z < 0.0 || z == 1.0 ? 0.0 : z < 1.0 ? -a.beta : z;
  } else {
    loss = (d - 0.5 / a.beta) * (d - 0.5 / a.beta);
    slope = 2.0 * (d - 0.5 / a.beta);
  }
  a.losses[pair] = loss;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    a.rewards[pair + k * a.pairs] = (float)(a.beta * ratio[k]);
    a.coefs[pair + k * a.pairs] = (float)((k ? -slope : slope) * share[k] / (double)a.pairs);
  }
}

// out = scale * (sum of v), in a fixed order
__global__ void __launch_bounds__(256) mean_kernel(const double* v, int64_t n, double scale, float* out) {
  __shared__ double red[4];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += v[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *out = (float)(s * scale);
}

// ---- policy ---------------------------------------------------------------------------------------------------------

// counts[segment] = the labels of it that count: segments of `span` labels
__global__ void __launch_bounds__(256) count_labels_kernel(const int64_t* labels, int64_t n, int64_t span, int64_t ignore,
                                                           double* counts) {
  __shared__ double red[4];
  const int64_t beg = blockIdx.x * span, end = min(beg + span, n);
  int64_t c = 0;
  for (int64_t i = beg + threadIdx.x; i < end; i += 256) c += labels[i] != ignore;
  const double all = block_sum((double)c, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

struct PolicyArgs {
  const float *old, *reference, *advantages;
  int64_t advantage_sequence, advantage_row;  // strides
  const double* counts;
  int64_t segments;  // counts of the whole batch's parts, or (by_sequence) of each sequence
  int by_sequence;
  double lo, hi, kl;
  float* logps;
  double* terms;  // [rows][2]: the loss's and the KL term's share of the mean
  void* gx;       // null: no gradient
};

// A token's loss and KL term, already times its share of the mean, and the loss's gradient by lp.
struct TokenLoss {
  double loss, kl, slope;
};
__device__ __forceinline__ double token_share(const PolicyArgs& p, const LogitRows& a, int64_t row) {
  if (p.by_sequence) return 1.0 / (p.counts[row / a.length] * (double)(a.rows / a.length));
  double n = 0.0;
  for (int64_t i = 0; i < p.segments; ++i) n += p.counts[i];
  return 1.0 / n;
}
__device__ __forceinline__ TokenLoss token_loss(const PolicyArgs& p, const LogitRows& a, int64_t row, double lp) {
  const double share = token_share(p, a, row);
  const double adv = (double)p.advantages[row / a.length * p.advantage_sequence + row % a.length * p.advantage_row];
  const double r = exp(lp - (double)p.old[row]), ra = r * adv;
  const double bounded = (r < 1.0 - p.lo ? 1.0 - p.lo : r > 1.0 + p.hi ? 1.0 + p.hi : r) * adv;
  TokenLoss t{bounded < ra ? -bounded : -ra, 0.0, bounded < ra ? 0.0 : -ra};
  if (p.reference) {
    const double more = (double)p.reference[row] - lp, e = exp(more);
    t.kl = e - more - 1.0;
    t.loss += p.kl * t.kl;
    t.slope += p.kl * (1.0 - e);
  }
  return {t.loss * share, t.kl * share, t.slope * share};
}

// eight logits of a row as they are in memory, minus infinity behind it
template <bool VEC>
__device__ __forceinline__ f32x8 load_raw(const float* p, int64_t c, int64_t cols) { return load_logits<VEC>(p, c, cols); }
template <bool VEC>
__device__ __forceinline__ bf16x8 load_raw(const __bf16* p, int64_t c, int64_t cols) {
  bf16x8 v;
  if (c + 8 <= cols) {
    if constexpr (VEC) v = *(const bf16x8*)(p + c);
    else __builtin_memcpy(&v, p + c, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = !VEC && c + e < cols ? p[c + e] : (__bf16)-kInf;
  }
  return v;
}
__device__ __forceinline__ f32x8 widen(f32x8 v) { return v; }
__device__ __forceinline__ f32x8 widen(bf16x8 v) { return __builtin_convertvector(v, f32x8); }

// NV vectors of eight logits to a thread hold the row; NV = 0: the row is read again for the gradient
template <class T, bool VEC, int RT, int NV>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) policy_kernel(LogitRows a, PolicyArgs p) {
  __shared__ float red[16];
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t label = a.labels[row];
  T* g = p.gx ? (T*)p.gx + row * a.vocab : nullptr;
  if (label == a.ignore) {
    if (t == 0) p.logps[row] = 0.f, p.terms[row * 2] = p.terms[row * 2 + 1] = 0.0;
    if (g) write_zeros<T, VEC, RT>(g, a.vocab);
    return;
  }
  const T* x = (const T*)a.x + a.offset(row);
  decltype(load_raw<VEC>(x, 0, 0)) held[NV ? NV : 1];
  RowStats st;
  if constexpr (NV > 0) {
    float m = -kInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) held[i] = load_raw<VEC>(x, (int64_t)(i * RT + t) * 8, a.vocab);
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, max8(widen(held[i])));
    st.top = row_max<RT>(m, red);
    const float from = st.top == -kInf ? 0.f : st.top;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const f32x8 v = widen(held[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += exp_from(v[e], from);
    }
    st.sum = row_total<RT>(s, red);
  } else {
    st = row_stats<T, VEC, RT>(x, a.vocab, red);
  }
  const double lp = label_logp(x, label, a.vocab, st);
  const TokenLoss loss = token_loss(p, a, row, lp);
  if (t == 0) {
    p.logps[row] = (float)lp;
    p.terms[row * 2] = loss.loss;
    p.terms[row * 2 + 1] = loss.kl;
  }
  if (!g) return;
  const float c = (float)loss.slope, lse = (float)((double)st.top + log((double)st.sum));
  if (c == 0.f) return write_zeros<T, VEC, RT>(g, a.vocab);
  auto put = [&](f32x8 v, int64_t c0) {
    f32x8 q;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = exp_from(v[e], lse);
    store8<VEC>(g, c0, a.vocab, row_gradient(q, c, c0, label));
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) put(widen(held[i]), (int64_t)(i * RT + t) * 8);
  } else {
    constexpr int U = 4;
    for (int64_t c0 = (int64_t)t * 8; c0 < a.vocab; c0 += RT * 8 * U) {
      f32x8 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load8<VEC>(x, c0 + u * RT * 8, a.vocab);
#pragma unroll
      for (int u = 0; u < U; ++u) put(v[u], c0 + u * RT * 8);
    }
  }
}

// sums[part] = the terms of a part of the rows; with one part, straight to the loss and the KL term
__global__ void __launch_bounds__(256) sum_terms_kernel(const double* terms, int64_t rows, int64_t span, double* sums,
                                                        float* loss, float* kl) {
  __shared__ double red[4];
  const int64_t beg = blockIdx.x * span, end = min(beg + span, rows);
  double l = 0.0, k = 0.0;
  for (int64_t i = beg + threadIdx.x; i < end; i += 256) l += terms[i * 2], k += terms[i * 2 + 1];
  l = block_sum(l, red);
  k = block_sum(k, red);
  if (threadIdx.x) return;
  if (loss) *loss = (float)l, *kl = (float)k;
  else sums[blockIdx.x * 2] = l, sums[blockIdx.x * 2 + 1] = k;
}

// x *= *factor, unless it is 1
template <class T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* x, int64_t n, const float* factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048)
    store8<false>(x, i, n, load8<false>(x, i, n) * f);
}

// ---- launches -------------------------------------------------------------------------------------------------------

constexpr int64_t kLogitMaxRows = 1 << 28, kLogitMaxVocab = 1 << 28;
constexpr int64_t kParts = 64;  // workgroups that count labels, or sum terms, at most

static int logits_check(const char* fn, const omt_logits* q) {
  if (!q) return fail(OMT_INVALID, "%s: null pointer", fn);
  if (q->dtype != OMT_DT_F32 && q->dtype != OMT_DT_BF16) return fail(OMT_INVALID, "%s: dtype %d", fn, q->dtype);
  if (q->sequences < 0 || q->length < 0 || q->vocab < 1)
    return fail(OMT_INVALID, "%s: logits %lld x %lld x %lld", fn, (long long)q->sequences, (long long)q->length, (long long)q->vocab);
  if (q->sequences > kLogitMaxRows || q->length > kLogitMaxRows || q->sequences * q->length > kLogitMaxRows || q->vocab > kLogitMaxVocab)
    return fail(OMT_UNSUPPORTED, "%s: logits %lld x %lld x %lld", fn, (long long)q->sequences, (long long)q->length, (long long)q->vocab);
  if (q->sequences * q->length > 0 && (!q->x || !q->labels)) return fail(OMT_INVALID, "%s: null pointer", fn);
  return OMT_OK;
}
static LogitRows rows_of(const omt_logits* q) {
  return {q->x, q->labels, q->ignore_index, std::max<int64_t>(q->length, 1), q->vocab, q->sequence_stride, q->row_stride,
          q->sequences * q->length};
}
static bool vectors(const omt_logits* q, const void* gx) {
  const int64_t per16 = q->dtype == OMT_DT_F32 ? 4 : 8;
  return q->vocab % 8 == 0 && q->sequence_stride % per16 == 0 && q->row_stride % per16 == 0 && !((uintptr_t)q->x & 15) &&
         !((uintptr_t)gx & 15);
}
// go(T, VEC): the type and whether rows are read by aligned vectors
template <class Go>
static void for_type(const omt_logits* q, const void* gx, Go go) {
  const bool vec = vectors(q, gx);
  if (q->dtype == OMT_DT_F32) vec ? go(0.f, std::true_type()) : go(0.f, std::false_type());
  else vec ? go((__bf16)0.f, std::true_type()) : go((__bf16)0.f, std::false_type());
}
// a workgroup or, at RT = 64, a wave to each row; a dimension of the grid holds fewer than 2^32 threads
template <int RT, class Kernel, class... A>
static void launch_rows(Kernel kernel, int64_t rows, hipStream_t s, A... args) {
  const int64_t groups = RT == 64 ? cdiv(rows, 4) : rows, along = std::min<int64_t>(groups, 1 << 20);
  hipLaunchKernelGGL(kernel, dim3((unsigned)along, (unsigned)cdiv(groups, along)), dim3(RT == 64 ? 256 : RT), 0, s, args...);
}
// go(RT): threads to a row that is read as it is used
template <class Go>
static void for_row_threads(int64_t vocab, Go go) {
  if (vocab <= 2048) go(std::integral_constant<int, 64>());
  else if (vocab <= 32768) go(std::integral_constant<int, 256>());
  else go(std::integral_constant<int, 1024>());
}

static int token_logps(const omt_logits* q, float* logps, float* lse, hipStream_t s) {
  for_type(q, nullptr, [&](auto t, auto vec) {
    typedef decltype(t) T;
    for_row_threads(q->vocab, [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      launch_rows<RT>(token_logps_kernel<T, decltype(vec)::value, RT>, q->sequences * q->length, s, rows_of(q), logps, lse);
    });
  });
  return launch_check("token_logps_kernel");
}
static int logit_grad(const omt_logits* q, const float* lse, const float* coefs, int per_row, void* gx, hipStream_t s) {
  for_type(q, gx, [&](auto t, auto vec) {
    typedef decltype(t) T;
    for_row_threads(q->vocab, [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      launch_rows<RT>(logit_grad_kernel<T, decltype(vec)::value, RT>, q->sequences * q->length, s, rows_of(q), lse, coefs,
                      per_row, (T*)gx);
    });
  });
  return launch_check("logit_grad_kernel");
}

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct PreferencePlan {
  size_t logps, lse, losses, coefs;  // bytes
  size_t total() const { return logps + lse + losses + coefs; }
};
static PreferencePlan preference_plan(int64_t sequences, int64_t length) {
  const size_t rows = up256((size_t)(sequences * length) * 4);
  return {rows, rows, up256((size_t)sequences * 4), up256((size_t)sequences * 4)};
}

struct PolicyPlan {
  int64_t segments, span;  // labels are counted in so many parts of so many
  int64_t parts;           // and the terms summed in so many
  size_t counts, terms, sums;
  size_t total() const { return counts + terms + sums; }
};
static PolicyPlan policy_plan(int64_t sequences, int64_t length, bool by_sequence) {
  const int64_t rows = sequences * length;
  PolicyPlan p;
  p.segments = by_sequence ? sequences : std::min(kParts, std::max<int64_t>(1, cdiv(rows, 4096)));
  p.span = by_sequence ? length : cdiv(rows, p.segments);
  p.parts = std::min(kParts, std::max<int64_t>(1, cdiv(rows, 16384)));
  p.counts = up256((size_t)p.segments * 8), p.terms = up256((size_t)rows * 16), p.sums = up256((size_t)p.parts * 16);
  return p;
}

// go(RT, NV): a row of `vocab` logits of type T in the registers of RT threads, NV vectors each; NV = 0: it does not fit
template <class T, class Go>
static void for_held_row(int64_t vocab, Go go) {
#define HELD(RT, NV) go(std::integral_constant<int, RT>(), std::integral_constant<int, NV>())
  if (vocab <= 512) HELD(64, 1);
  else if (vocab <= 1024) HELD(64, 2);
  else if (vocab <= 2048) HELD(64, 4);
  else if (vocab <= 4096) HELD(256, 2);
  else if (vocab <= 8192) HELD(256, 4);
  else if (vocab <= 16384) HELD(256, 8);
  else if (vocab <= 32768) HELD(1024, 4);
  else if (vocab <= 65536) HELD(1024, 8);
  else if constexpr (sizeof(T) == 2) {
    if (vocab <= 131072) HELD(1024, 16);
    else HELD(1024, 0);
  } else {
    HELD(1024, 0);
  }
#undef HELD
}

}  // namespace omt

using namespace omt;

OMT_EXPORT int omt_token_logps_fwd(const omt_logits* logits, float* logps, float* lse, void* stream) {
  if (int e = logits_check("omt_token_logps_fwd", logits)) return e;
  if (logits->sequences * logits->length == 0) return OMT_OK;
  if (!logps || !lse) return fail(OMT_INVALID, "omt_token_logps_fwd: null pointer");
  return token_logps(logits, logps, lse, stream_of(stream));
}

OMT_EXPORT int omt_token_logps_bwd(const omt_logits* logits, const float* lse, const float* g, void* gx, void* stream) {
  if (int e = logits_check("omt_token_logps_bwd", logits)) return e;
  if (logits->sequences * logits->length == 0) return OMT_OK;
  if (!lse || !g || !gx) return fail(OMT_INVALID, "omt_token_logps_bwd: null pointer");
  return logit_grad(logits, lse, g, 1, gx, stream_of(stream));
}

OMT_EXPORT size_t omt_preference_workspace(int64_t sequences, int64_t length) {
  if (sequences < 0 || length < 0 || sequences > kLogitMaxRows || length > kLogitMaxRows || sequences * length > kLogitMaxRows) return 0;
  return preference_plan(sequences, length).total();
}

OMT_EXPORT int omt_preference_loss(const omt_logits* logits, const float* reference, int kind, double beta, double smoothing,
                                   int average, float* loss, float* rewards, void* gx, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* fn = "omt_preference_loss";
  if (int e = logits_check(fn, logits)) return e;
  const int64_t n = logits->sequences, rows = n * logits->length;
  if (n < 2 || n % 2) return fail(OMT_INVALID, "%s: %lld sequences: pairs are needed", fn, (long long)n);
  if (kind < OMT_PREFERENCE_SIGMOID || kind > OMT_PREFERENCE_IPO) return fail(OMT_INVALID, "%s: kind %d", fn, kind);
  if (!(beta > 0.0) || !(smoothing >= 0.0 && smoothing <= 1.0)) return fail(OMT_INVALID, "%s: beta %g, smoothing %g", fn, beta, smoothing);
  if (n / 2 >= 1 << 24) return fail(OMT_UNSUPPORTED, "%s: %lld sequences", fn, (long long)n);
  if (!reference || !loss || !rewards) return fail(OMT_INVALID, "%s: null pointer", fn);
  const PreferencePlan p = preference_plan(n, logits->length);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.total())
    return fail(OMT_INVALID, "%s: workspace of %zu bytes at %p", fn, workspace_bytes, workspace);
  char* at = (char*)workspace;
  float *logps = (float*)at, *lse = (float*)(at + p.logps);
  double* losses = (double*)(at + p.logps + p.lse);
  float* coefs = (float*)(at + p.logps + p.lse + p.losses);
  hipStream_t s = stream_of(stream);
  if (rows > 0)
    if (int e = token_logps(logits, logps, lse, s)) return e;
  const PairArgs a{logits->labels, logps, reference, logits->ignore_index, logits->length, n / 2, kind, average, beta, smoothing,
                   rewards, coefs, losses};
  hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)(n / 2)), dim3(256), 0, s, a);
  if (int e = launch_check("preference_pair_kernel")) return e;
  hipLaunchKernelGGL(mean_kernel, dim3(1), dim3(256), 0, s, losses, n / 2, 1.0 / (double)(n / 2), loss);
  if (int e = launch_check("mean_kernel")) return e;
  return gx && rows > 0 ? logit_grad(logits, lse, coefs, 0, gx, s) : OMT_OK;
}

OMT_EXPORT size_t omt_policy_workspace(int64_t sequences, int64_t length, int by_sequence) {
  if (sequences < 0 || length < 0 || sequences > kLogitMaxRows || length > kLogitMaxRows || sequences * length > kLogitMaxRows) return 0;
  return policy_plan(sequences, length, by_sequence != 0).total();
}

OMT_EXPORT int omt_policy_loss(const omt_logits* logits, const float* old_logps, const float* reference, const float* advantages,
                               int64_t advantage_sequence_stride, int64_t advantage_row_stride, double clip_low,
                               double clip_high, double kl_weight, int by_sequence, float* loss, float* kl, float* logps,
                               void* gx, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omt_policy_loss";
  if (int e = logits_check(fn, logits)) return e;
  const int64_t rows = logits->sequences * logits->length;
  if (!(clip_low >= 0.0) || !(clip_high >= 0.0)) return fail(OMT_INVALID, "%s: clip %g, %g", fn, clip_low, clip_high);
  if (by_sequence && logits->sequences >= 1 << 24) return fail(OMT_UNSUPPORTED, "%s: %lld sequences", fn, (long long)logits->sequences);
  if (!loss || !kl || (rows > 0 && (!old_logps || !advantages || !logps))) return fail(OMT_INVALID, "%s: null pointer", fn);
  const PolicyPlan p = policy_plan(logits->sequences, logits->length, by_sequence != 0);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.total())
    return fail(OMT_INVALID, "%s: workspace of %zu bytes at %p", fn, workspace_bytes, workspace);
  char* at = (char*)workspace;
  double *counts = (double*)at, *terms = (double*)(at + p.counts), *sums = (double*)(at + p.counts + p.terms);
  hipStream_t s = stream_of(stream);
  if (rows > 0) {
    hipLaunchKernelGGL(count_labels_kernel, dim3((unsigned)p.segments), dim3(256), 0, s, logits->labels, rows, p.span,
                       logits->ignore_index, counts);
    if (int e = launch_check("count_labels_kernel")) return e;
    const PolicyArgs a{old_logps, reference, advantages, advantage_sequence_stride, advantage_row_stride, counts, p.segments,
                       by_sequence, clip_low, clip_high, kl_weight, logps, terms, gx};
    for_type(logits, gx, [&](auto t, auto vec) {
      typedef decltype(t) T;
      for_held_row<T>(logits->vocab, [&](auto rt, auto nv) {
        constexpr int RT = decltype(rt)::value;
        launch_rows<RT>(policy_kernel<T, decltype(vec)::value, RT, decltype(nv)::value>, rows, s, rows_of(logits), a);
      });
    });
    if (int e = launch_check("policy_kernel")) return e;
  }
  const bool two = p.parts > 1;
  hipLaunchKernelGGL(sum_terms_kernel, dim3((unsigned)p.parts), dim3(256), 0, s, terms, rows, cdiv(rows, p.parts), sums,
                     two ? nullptr : loss, two ? nullptr : kl);
  if (int e = launch_check("sum_terms_kernel")) return e;
  if (!two) return OMT_OK;
  hipLaunchKernelGGL(sum_terms_kernel, dim3(1), dim3(256), 0, s, sums, p.parts, p.parts, sums, loss, kl);
  return launch_check("sum_terms_kernel");
}

OMT_EXPORT int omt_scale_by(int dtype, int64_t n, void* x, const float* factor, void* stream) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "omt_scale_by: dtype %d", dtype);
  if (n < 0 || (n > 0 && (!x || !factor))) return fail(OMT_INVALID, "omt_scale_by: null pointer or negative size");
  if (n == 0) return OMT_OK;
  const unsigned grid = grid1d(cdiv(n, 8), 256, 2048);
  hipStream_t s = stream_of(stream);
  if (dtype == OMT_DT_F32) hipLaunchKernelGGL(scale_by_kernel<float>, dim3(grid), dim3(256), 0, s, (float*)x, n, factor);
  else hipLaunchKernelGGL(scale_by_kernel<__bf16>, dim3(grid), dim3(256), 0, s, (__bf16*)x, n, factor);
  return launch_check("scale_by_kernel");
}
