// Losses on a language model's logits x [sequences][length][vocab] with labels, and their gradients. Of each row whose label
// counts (it is not ignore_index): lse = log(sum exp x), lp = x[label] - lse, and d lp / d x = onehot(label) - exp(x - lse).
//
// token_logps: lp and lse of every row, and the gradient from one of lp, by lse in 32 bits or in 64.
//
// preference: sequences in pairs, the chosen ones in the first half. With L the sum (or mean) of a sequence's lp and R its
//   reference, d = (L - R of the chosen) - (L - R of the rejected):
//     sigmoid  -(1 - s) log sigmoid(beta d) - s log sigmoid(-beta d)
//     hinge    max(0, 1 - beta d)
//     ipo      (d - 1 / (2 beta))^2
//   and the mean over pairs. The gradient of every lp of a sequence is the same.
//
// policy: r = exp(lp - old), loss of a token -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(ref - lp) - (ref - lp) - 1), and the mean
//   over all tokens, or over sequences of each one's mean. k of weight 0 takes no part.
//
// Rows that do not count are not read, so that nothing in them matters, and get a gradient of zeros; so do rows whose lp has a
// gradient of zero. A label outside the vocabulary makes the loss, and its row's gradient (its pair's), NaN. Exponentials and their sums over a
// row are float32, what is computed of lp (sums over a sequence, ratios next to the clip's borders, the KL term) is float64. No atomics:
// every sum runs in a fixed order.
//
// Bound by memory. The gradient needs a row's sum, so a row is read twice, or once where a workgroup holds it in registers
// (policy); a pair's coefficient needs all rows of both sequences, so the preference loss reads its rows twice. A row takes a
// wave or a workgroup of 128 to 1024 threads by its bytes, no more than keep several rows in flight on each compute unit, so that
// one's reductions and exponentials pass under another's loads.
//
// 16 x 512 rows in bfloat16 of which 58% count: policy x 131072 685 us (3.40 GB that it cannot do without, 2.15 of them written), x 65536
// 348, x 32768 167; preference x 32768 56 + 6 + 122 us for 0.85 GB; 6 x 301 x 50021 float32, rows on 4 bytes, 140 us for 0.58 GB. A large copy
// reaches 4.74 TB/s on this card: the second pass finds part of its rows in the last cache. Small calls are launches.
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

// A row is a body of vectors of 16 bytes, on 16 bytes, and up to 14 single columns before and behind it, of which a thread has
// one at most: rows of any size, at any alignment, are read by whole vectors.
template <class T> struct Lanes;
template <> struct Lanes<float> {
  typedef f32x4 raw, wide;
  static constexpr int W = 4;
};
template <> struct Lanes<__bf16> {
  typedef bf16x8 raw;
  typedef f32x8 wide;
  static constexpr int W = 8;
};
template <class T>
struct Row {
  typedef typename Lanes<T>::raw Raw;
  typedef typename Lanes<T>::wide Wide;
  static constexpr int W = Lanes<T>::W;
  const T* p;
  int cols, head, body;  // columns, those before the body, and its vectors
  __device__ __forceinline__ Row(const T* at, int64_t n) : p(at), cols((int)n) {
    head = min((int)((0 - (uintptr_t)at) & 15) / (int)sizeof(T), cols);
    body = (cols - head) / W;
  }
  __device__ __forceinline__ Raw load(int j) const {
    Raw v;
    if (j < body) {
      v = *(const Raw*)(p + head + j * W);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = (T)-kInf;
    }
    return v;
  }
  // the single column of thread t; -1 where it has none
  __device__ __forceinline__ int single(int t) const {
    const int c = t < head ? t : body * W + t;
    return c < cols && t < 2 * W ? c : -1;
  }
  __device__ __forceinline__ int column(int j) const { return head + j * W; }
};
__device__ __forceinline__ f32x4 widen(f32x4 v) { return v; }
__device__ __forceinline__ f32x8 widen(bf16x8 v) { return __builtin_convertvector(v, f32x8); }
__device__ __forceinline__ float largest(f32x4 v) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); }
__device__ __forceinline__ float largest(f32x8 v) {
  return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
// exp(v - m): the difference first, which is exact or nearly so for what counts
__device__ __forceinline__ float exp_from(float v, float m) { return __builtin_amdgcn_exp2f((v - m) * kLog2e); }

// The gradient's row: written past the caches, which so keep what is read again, where it lies as the logits' row does (preference
// loss and gradient of 16 x 512 x 32768 bfloat16 241 us with plain stores, 214 with these; unaligned ones stay plain: 187 and 193).
template <class T>
struct GradRow {
  T* g;
  bool aligned;
  __device__ __forceinline__ GradRow(T* at, const Row<T>& r) : g(at), aligned(!((uintptr_t)(at + r.head) & 15)) {}
  __device__ __forceinline__ void store(int c, typename Lanes<T>::wide v) const {
    typename Lanes<T>::raw r = __builtin_convertvector(v, typename Lanes<T>::raw);
    if (aligned) __builtin_nontemporal_store(r, (typename Lanes<T>::raw*)(g + c));
    else __builtin_memcpy(g + c, &r, sizeof(r));
  }
};

// The largest and the sum of exp(x - largest) of a row of memory, in every one of its RT threads.
struct RowStats {
  float top, sum;
};
template <class T, int RT>
__device__ __forceinline__ RowStats row_stats(const Row<T>& x, float* red) {
  constexpr int U = 4, W = Row<T>::W;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int single = x.single(t);
  float m = single >= 0 ? (float)x.p[single] : -kInf, s = single >= 0 && m != -kInf ? 1.f : 0.f;
  if (m != m) s = m;
  typename Row<T>::Raw now[U], next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) now[u] = x.load(t + u * RT);
  for (int j = t;; j += RT * U) {
    const bool more = j - t + RT * U < x.body;  // (the same for the row's threads)
    if (more)
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = x.load(j + (U + u) * RT);
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, largest(widen(now[u])));
    // (a thread that has met nothing over minus infinity: differences to 0 instead, so that none is NaN)
    const float from = top == -kInf ? 0.f : top;
    s *= exp_from(m, from);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const auto v = widen(now[u]);
#pragma unroll
      for (int e = 0; e < W; ++e) s += exp_from(v[e], from);
    }
    m = top;
    if (!more) break;
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
  }
  const float top = row_max<RT>(m, red), from = top == -kInf ? 0.f : top;
  return {top, row_total<RT>(s * exp_from(m, from), red)};
}

__device__ __forceinline__ bool in_vocab(int64_t label, int64_t vocab) { return (uint64_t)label < (uint64_t)vocab; }
// lp of a label, NaN outside the vocabulary; a row of minus infinities has top - top = NaN in it, as the definition has
template <class T>
__device__ __forceinline__ double label_logp(const T* x, int64_t label, int64_t vocab, float top, double log_sum) {
  return in_vocab(label, vocab) ? ((double)(float)x[label] - (double)top) - log_sum : (double)__builtin_nanf("");
}

// ---- statistics of rows ---------------------------------------------------------------------------------------------

// Row of this thread, with RT threads to a row; -1 where there is none (a whole wave, or the workgroup)
template <int RT>
__device__ __forceinline__ int64_t this_row(int64_t rows) {
  const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t row = RT == 64 ? group * 4 + (threadIdx.x >> 6) : group;
  return row < rows ? row : -1;
}

// What is written of each row; null: not asked for. sums: lp in 64 bits, for those that are added up; lse in 32 bits or in 64.
struct RowOut {
  float *logps, *lse;
  double *lse64, *sums;
  RowStats* stats;
};
template <class T, int RT>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) token_logps_kernel(LogitRows a, RowOut out) {
  __shared__ float red[16];
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const bool first = (RT == 64 ? threadIdx.x & 63 : threadIdx.x) == 0;
  const int64_t label = a.labels[row];
  if (label == a.ignore) {
    if (first) {
      if (out.logps) out.logps[row] = 0.f;
      if (out.lse) out.lse[row] = 0.f;
      if (out.lse64) out.lse64[row] = 0.0;
      if (out.sums) out.sums[row] = 0.0;
    }
    return;
  }
  const Row<T> x((const T*)a.x + a.offset(row), a.vocab);
  const RowStats st = row_stats<T, RT>(x, red);
  if (first) {
    const double log_sum = log((double)st.sum), lp = label_logp(x.p, label, a.vocab, st.top, log_sum), lse = (double)st.top + log_sum;
    if (out.logps) out.logps[row] = (float)lp;
    if (out.lse) out.lse[row] = (float)lse;
    if (out.lse64) out.lse64[row] = lse;
    if (out.sums) out.sums[row] = lp;
    if (out.stats) out.stats[row] = st;
  }
}

// ---- pairs ----------------------------------------------------------------------------------------------------------

// two sums over the workgroup's THREADS, in every one of them
template <int THREADS>
__device__ __forceinline__ void block_sums(double& u, double& v, double* red) {
  u = wave_sum(u), v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[(threadIdx.x >> 6) * 2] = u, red[(threadIdx.x >> 6) * 2 + 1] = v;
  __syncthreads();
  u = v = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) u += red[w * 2], v += red[w * 2 + 1];
}

struct PairArgs {
  const int64_t* labels;
  const double* logps;
  const float* reference;
  int64_t ignore, length, pairs;
  int kind, average;
  double beta, smoothing;
  float *rewards, *coefs;
  double* losses;
};

// log(1 + exp(-z)) without overflow
__device__ __forceinline__ double softplus_neg(double z) { return (z < 0 ? -z : 0.0) + log1p(exp(z < 0 ? z : -z)); }
__device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

// The loss of a pair, and of each of its sequences the reward and the gradient of the mean loss by a log-probability
struct PairLoss {
  double loss;
  float rewards[2], coefs[2];
};
__device__ __forceinline__ PairLoss pair_loss(const PairArgs& a, int64_t pair, const double (&sum)[2], const double (&count)[2]) {
  double ratio[2], share[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    share[k] = a.average ? 1.0 / fmax(count[k], 1.0) : 1.0;
    ratio[k] = sum[k] * share[k] - (double)a.reference[pair + k * a.pairs];
  }
  const double d = ratio[0] - ratio[1], z = a.beta * d;
  double loss, slope;  // of the loss by d
  if (a.kind == OMT_PREFERENCE_SIGMOID) {
    // (a term of weight zero is left out: it may be infinite)
    loss = (a.smoothing < 1.0 ? (1.0 - a.smoothing) * softplus_neg(z) : 0.0) + (a.smoothing > 0.0 ? a.smoothing * softplus_neg(-z) : 0.0);
    slope = a.beta * (a.smoothing - sigmoid(-z));
  } else if (a.kind == OMT_PREFERENCE_HINGE) {
    loss = 1.0 - z < 0.0 ? 0.0 : 1.0 - z;  // (NaN stays NaN)
    slope = 1.0 - z < 0.0 || z == 1.0 ? 0.0 : z < 1.0 ? -a.beta : z;
  } else {
    loss = (d - 0.5 / a.beta) * (d - 0.5 / a.beta);
    slope = 2.0 * (d - 0.5 / a.beta);
  }
  PairLoss l;
  l.loss = loss;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    l.rewards[k] = (float)(a.beta * ratio[k]);
    l.coefs[k] = (float)((k ? -slope : slope) * share[k] / (double)a.pairs);
  }
  return l;
}
// log-probabilities of a sequence and how many count, every THREADS-th of them from `first` on (those that do not count are 0)
template <int THREADS>
__device__ __forceinline__ void sequence_share(const PairArgs& a, int64_t seq, int first, double& sum, double& count) {
  const int64_t base = seq * a.length;
  sum = count = 0.0;
#pragma unroll 4
  for (int64_t i = first; i < a.length; i += THREADS) {
    sum += a.logps[base + i];
    count += a.labels[base + i] != a.ignore ? 1.0 : 0.0;
  }
}
__device__ __forceinline__ PairLoss pair_by_wave(const PairArgs& a, int64_t pair) {
  double sum[2], count[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) sequence_share<64>(a, pair + k * a.pairs, threadIdx.x & 63, sum[k], count[k]);
#pragma unroll
  for (int k = 0; k < 2; ++k) sum[k] = wave_sum(sum[k]), count[k] = wave_sum(count[k]);
  return pair_loss(a, pair, sum, count);
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) preference_pair_kernel(PairArgs a) {
  __shared__ double red[THREADS / 32];
  const int64_t pair = blockIdx.x;
  double sum[2], count[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    sequence_share<THREADS>(a, pair + k * a.pairs, threadIdx.x, sum[k], count[k]);
    block_sums<THREADS>(sum[k], count[k], red);
  }
  if (threadIdx.x) return;
  const PairLoss l = pair_loss(a, pair, sum, count);
  a.losses[pair] = l.loss;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    a.rewards[pair + k * a.pairs] = l.rewards[k];
    a.coefs[pair + k * a.pairs] = l.coefs[k];
  }
}

// ---- the gradient of rows -------------------------------------------------------------------------------------------

template <class T, int RT>
__device__ __forceinline__ void write_zeros(const GradRow<T>& g, const Row<T>& x) {
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int single = x.single(t);
  if (single >= 0) g.g[single] = (T)0.f;
  for (int j = t; j < x.body; j += RT) g.store(x.column(j), typename Row<T>::Wide{});
}

// c onehot(label) - scale exp(x - from), scale exp(-from) = c / sum exp x, of the columns from c0 on
struct Slope {
  float c, scale, from;
  int64_t label;
};
template <class Wide>
__device__ __forceinline__ Wide row_gradient(Wide v, const Slope& s, int c0) {
  constexpr int W = sizeof(Wide) / 4;
  Wide g;
#pragma unroll
  for (int e = 0; e < W; ++e) g[e] = exp_from(v[e], s.from) * -s.scale;
  if ((uint64_t)(s.label - c0) < W)
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (c0 + e == s.label) g[e] += s.c;
  return g;
}
// of the thread's single column
template <class T>
__device__ __forceinline__ void single_gradient(const Row<T>& x, T* g, int t, const Slope& s) {
  const int single = x.single(t);
  if (single >= 0) g[single] = (T)(exp_from((float)x.p[single], s.from) * -s.scale + (single == s.label ? s.c : 0.f));
}
// of a row of memory
template <class T, int RT>
__device__ __forceinline__ void write_gradient(const Row<T>& x, const GradRow<T>& g, const Slope& s) {
  constexpr int U = 4;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  single_gradient(x, g.g, t, s);
  for (int j = t; j < x.body; j += RT * U) {
    typename Row<T>::Raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = x.load(j + u * RT);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * RT < x.body) g.store(x.column(j + u * RT), row_gradient(widen(v[u]), s, x.column(j + u * RT)));
  }
}

// Of each row, lse in 32 bits, whose rounding makes exp(x - lse) off by 2^-24 |lse|, or in 64, or its RowStats. per_row: coefs holds one for each row, else one for each sequence.
// backwards: the last rows first, which a pass over all rows has left in the last cache. losses (or null): the mean of so many
// goes to loss, by the first workgroup.
struct GradArgs {
  const float* lse;
  const double* lse64;
  const RowStats* stats;
  const float* coefs;
  int per_row, backwards;
  const double* losses;
  int64_t count;
  float* loss;
};
__device__ __forceinline__ void mean_loss(const double* losses, int64_t count, float* loss) {  // by one wave
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 64) s += losses[i];
  s = wave_sum(s);
  if (threadIdx.x == 0) *loss = (float)(s / (double)count);
}
template <class T, int RT>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) logit_grad_kernel(LogitRows a, GradArgs q, T* gx) {
  if (q.losses && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 64) mean_loss(q.losses, q.count, q.loss);
  int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  if (q.backwards) row = a.rows - 1 - row;
  const int64_t label = a.labels[row];
  const float coef = q.coefs[q.per_row ? row : row / a.length];
  const Row<T> x((const T*)a.x + a.offset(row), a.vocab);
  const GradRow<T> g(gx + row * a.vocab, x);
  if (label == a.ignore || coef == 0.f) return write_zeros<T, RT>(g, x);
  const float c = in_vocab(label, a.vocab) ? coef : __builtin_nanf("");
  RowStats st;
  if (q.stats) {
    st = q.stats[row];
  } else if (q.lse64) {
    const double lse = q.lse64[row];
    st.top = (float)lse;
    st.sum = exp_from((float)(lse - (double)st.top), 0.f);
  } else {
    st = {q.lse[row], 1.f};
  }
  write_gradient<T, RT>(x, g, {c, c / st.sum, st.top, label});
}
// Labels that each row's threads look through for themselves, for a launch less (policy, 8 x 61 x 256 float32: 11.0 us with that
// launch, 9.3 without).
constexpr int64_t kFewLabels = 1024;

// The gradient of few short pairs, whose losses each row's threads compute for themselves, for a launch less (2 pairs x 63 x 256 float32 13.0
// us with that launch, 10.7 without; 4 x 256 x 16384 bfloat16 32.5 and 29.5); the first workgroup adds them up.
constexpr int64_t kFewPairs = 4;
template <class T, int RT>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) few_pairs_grad_kernel(LogitRows a, PairArgs q, const RowStats* stats, float* loss,
                                                                             T* gx) {
  __shared__ double losses[kFewPairs];
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    constexpr int WAVES = (RT == 64 ? 256 : RT) / 64;
    for (int p = threadIdx.x >> 6; p < q.pairs; p += WAVES) {
      const PairLoss l = pair_by_wave(q, p);
      if ((threadIdx.x & 63) == 0) {
        losses[p] = l.loss;
        q.rewards[p] = l.rewards[0], q.rewards[p + q.pairs] = l.rewards[1];
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int p = 0; p < q.pairs; ++p) all += losses[p];
      *loss = (float)(all / (double)q.pairs);
    }
  }
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const int64_t label = a.labels[row], seq = row / a.length;
  const Row<T> x((const T*)a.x + a.offset(row), a.vocab);
  const GradRow<T> g(gx + row * a.vocab, x);
  if (label == a.ignore) return write_zeros<T, RT>(g, x);
  const PairLoss l = pair_by_wave(q, seq % q.pairs);
  const float coef = seq < q.pairs ? l.coefs[0] : l.coefs[1], c = in_vocab(label, a.vocab) ? coef : __builtin_nanf("");
  if (c == 0.f) return write_zeros<T, RT>(g, x);
  const RowStats st = stats[row];
  write_gradient<T, RT>(x, g, {c, c / st.sum, st.top, label});
}

__global__ void __launch_bounds__(64) mean_loss_kernel(const double* losses, int64_t count, float* loss) {
  mean_loss(losses, count, loss);
}

// ---- policy ---------------------------------------------------------------------------------------------------------

// counts[segment] = the labels of it that count: segments of `span` labels
__global__ void __launch_bounds__(1024) count_labels_kernel(const int64_t* labels, int64_t n, int64_t span, int64_t ignore,
                                                           double* counts) {
  __shared__ double red[32];
  const int64_t beg = blockIdx.x * span, end = min(beg + span, n);
  int64_t c = 0;
#pragma unroll 4
  for (int64_t i = beg + threadIdx.x; i < end; i += 1024) c += labels[i] != ignore;
  double all = (double)c, none = 0.0;
  block_sums<1024>(all, none, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

struct PolicyArgs {
  const float *old, *reference, *advantages;
  int64_t advantage_sequence, advantage_row;  // strides
  const double* counts;  // null: each row's threads count for themselves
  int64_t segments;      // counts of the whole batch's parts, 64 at most, or (by_sequence) of each sequence
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
  const double sequences = p.by_sequence ? (double)(a.rows / a.length) : 1.0;
  if (!p.counts) {
    const int64_t beg = p.by_sequence ? row / a.length * a.length : 0, n = p.by_sequence ? a.length : a.rows;
    int c = 0;
    for (int64_t i = threadIdx.x & 63; i < n; i += 64) c += a.labels[beg + i] != a.ignore;
    return 1.0 / (wave_sum((double)c) * sequences);
  }
  if (p.by_sequence) return 1.0 / (p.counts[row / a.length] * sequences);
  return 1.0 / wave_sum((threadIdx.x & 63) < p.segments ? p.counts[threadIdx.x & 63] : 0.0);
}
__device__ __forceinline__ TokenLoss token_loss(const PolicyArgs& p, const LogitRows& a, int64_t row, double lp) {
  const double share = token_share(p, a, row);
  const double adv = (double)p.advantages[row / a.length * p.advantage_sequence + row % a.length * p.advantage_row];
  const double r = exp(lp - (double)p.old[row]), ra = r * adv;
  const double bounded = (r < 1.0 - p.lo ? 1.0 - p.lo : r > 1.0 + p.hi ? 1.0 + p.hi : r) * adv;
  TokenLoss t{bounded < ra ? -bounded : -ra, 0.0, bounded < ra ? 0.0 : -ra};
  if (p.reference) {
    // (exp(more) - 1 as one: beside the reference what is left of it, less than 1's last places, is the term)
    const double more = (double)p.reference[row] - lp, grown = expm1(more);
    t.kl = grown - more;
    if (p.kl != 0.0) {  // (a term of weight zero is left out: it may be infinite)
      t.loss += p.kl * t.kl;
      t.slope -= p.kl * grown;
    }
  }
  return {t.loss * share, t.kl * share, t.slope * share};
}

// NV vectors to a thread hold the row's body; NV = 0: the row is read again for the gradient
template <class T, int RT, int NV>
__global__ void __launch_bounds__(RT == 64 ? 256 : RT) policy_kernel(LogitRows a, PolicyArgs p) {
  __shared__ float red[16];
  const int64_t row = this_row<RT>(a.rows);
  if (row < 0) return;
  const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t label = a.labels[row];
  const Row<T> x((const T*)a.x + a.offset(row), a.vocab);
  const GradRow<T> g((T*)p.gx + row * a.vocab, x);
  if (label == a.ignore) {
    if (t == 0) p.logps[row] = 0.f, p.terms[row * 2] = p.terms[row * 2 + 1] = 0.0;
    if (p.gx) write_zeros<T, RT>(g, x);
    return;
  }
  typename Row<T>::Raw held[NV ? NV : 1];
  RowStats st;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) held[i] = x.load(i * RT + t);
    const int single = x.single(t);
    const float one = single >= 0 ? (float)x.p[single] : -kInf;
    float m = one;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, largest(widen(held[i])));
    st.top = row_max<RT>(m, red);
    const float from = st.top == -kInf ? 0.f : st.top;
    float s = exp_from(one, from);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const auto v = widen(held[i]);
#pragma unroll
      for (int e = 0; e < Row<T>::W; ++e) s += exp_from(v[e], from);
    }
    st.sum = row_total<RT>(s, red);
  } else {
    st = row_stats<T, RT>(x, red);
  }
  const double lp = label_logp(x.p, label, a.vocab, st.top, log((double)st.sum));
  const TokenLoss loss = token_loss(p, a, row, lp);
  if (t == 0) {
    p.logps[row] = (float)lp;
    p.terms[row * 2] = loss.loss;
    p.terms[row * 2 + 1] = loss.kl;
  }
  if (!p.gx) return;
  const float c = (float)loss.slope;
  if (c == 0.f) return write_zeros<T, RT>(g, x);
  const Slope slope{c, c / st.sum, st.top, label};
  if constexpr (NV > 0) {
    single_gradient(x, g.g, t, slope);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * RT + t < x.body) g.store(x.column(i * RT + t), row_gradient(widen(held[i]), slope, x.column(i * RT + t)));
  } else {
    write_gradient<T, RT>(x, g, slope);
  }
}

// sums[part] = the terms of a part of the rows; with one part, straight to the loss and the KL term
__global__ void __launch_bounds__(1024) sum_terms_kernel(const double* terms, int64_t rows, int64_t span, double* sums,
                                                        float* loss, float* kl) {
  __shared__ double red[32];
  const int64_t beg = blockIdx.x * span, end = min(beg + span, rows);
  double l = 0.0, k = 0.0;
#pragma unroll 4
  for (int64_t i = beg + threadIdx.x; i < end; i += 1024) l += terms[i * 2], k += terms[i * 2 + 1];
  block_sums<1024>(l, k, red);
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
constexpr int64_t kFewPairsLength = 256;
constexpr int64_t kParts = 64;  // workgroups that count labels, or sum terms, at most
// Logits of more than this are taken backwards in their second pass (the last cache holds 256 MB; rows that do not count are not in
// it): preference loss and gradient of 16 x 512 x 32768 bfloat16 213 us forwards, 185 backwards, x 131072 834 and 794; of 6 x 301 x
// 50021 float32, all of whose counted rows are still there, 138 and 143.
constexpr int64_t kBackwardsBytes = 384 << 20;

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
// go(T): the logits' type
template <class Go>
static void for_type(const omt_logits* q, Go go) {
  if (q->dtype == OMT_DT_F32) go(0.f);
  else go((__bf16)0.f);
}
static int64_t row_bytes(const omt_logits* q) { return q->vocab * (q->dtype == OMT_DT_F32 ? 4 : 2); }
// a workgroup or, at RT = 64, a wave to each row; a dimension of the grid holds fewer than 2^32 threads
template <int RT, class Kernel, class... A>
static void launch_rows(Kernel kernel, int64_t rows, hipStream_t s, A... args) {
  const int64_t groups = RT == 64 ? cdiv(rows, 4) : rows, along = std::min<int64_t>(groups, 1 << 20);
  hipLaunchKernelGGL(kernel, dim3((unsigned)along, (unsigned)cdiv(groups, along)), dim3(RT == 64 ? 256 : RT), 0, s, args...);
}
// go(RT): threads to a row that is read as it is used. Preference loss and gradient of 16 x 512 rows in bfloat16, us, by 64, 128, 256,
// 512 and 1024 threads: 4 KB 24.1, 25.3, 32.5; 8 KB 35.1, 32.7, 36.9, 52.5; 16 KB 59, 52.8, 51.1, 62; 64 KB -, 202, 186, 181, 186;
// 256 KB -, -, 878, 845, 794.
template <class Go>
static void for_row_threads(int64_t bytes, Go go) {
  if (bytes <= 6144) go(std::integral_constant<int, 64>());
  else if (bytes <= 12288) go(std::integral_constant<int, 128>());
  else if (bytes <= 32768) go(std::integral_constant<int, 256>());
  else if (bytes <= 131072) go(std::integral_constant<int, 512>());
  else go(std::integral_constant<int, 1024>());
}

static int token_logps(const omt_logits* q, const RowOut& out, hipStream_t s) {
  for_type(q, [&](auto t) {
    for_row_threads(row_bytes(q), [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      launch_rows<RT>(token_logps_kernel<decltype(t), RT>, q->sequences * q->length, s, rows_of(q), out);
    });
  });
  return launch_check("token_logps_kernel");
}
static int logit_grad(const omt_logits* q, const GradArgs& a, void* gx, hipStream_t s) {
  for_type(q, [&](auto t) {
    typedef decltype(t) T;
    for_row_threads(row_bytes(q), [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      launch_rows<RT>(logit_grad_kernel<T, RT>, q->sequences * q->length, s, rows_of(q), a, (T*)gx);
    });
  });
  return launch_check("logit_grad_kernel");
}

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct PreferencePlan {
  size_t logps, stats, losses, coefs;  // bytes
  size_t total() const { return logps + stats + losses + coefs; }
};
static PreferencePlan preference_plan(int64_t sequences, int64_t length) {
  const size_t rows = (size_t)(sequences * length);
  return {up256(rows * 8), up256(rows * sizeof(RowStats)), up256((size_t)sequences * 4), up256((size_t)sequences * 4)};
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
  p.segments = by_sequence ? sequences : std::min(kParts, std::max<int64_t>(1, cdiv(rows, 1024)));
  p.span = by_sequence ? length : cdiv(rows, p.segments);
  p.parts = std::min(kParts, std::max<int64_t>(1, cdiv(rows, 65536)));
  p.counts = up256((size_t)p.segments * 8), p.terms = up256((size_t)rows * 16), p.sums = up256((size_t)p.parts * 16);
  return p;
}

// go(RT, NV): a row of so many bytes in the registers of RT threads, NV vectors each; NV = 0: it is read again. Policy loss and gradient
// of 16 x 512 rows in bfloat16, us: 64 KB 180 held by 256 threads, 179 by 512, 218 by 1024, read again 205 to 254; 128 KB held 364, read
// again 381 to 448; 256 KB, which take all registers of a compute unit, 1269 held, 767 read again.
template <class Go>
static void for_held_row(int64_t bytes, Go go) {
#define HELD(RT, NV) if (bytes <= RT * NV * 16) return go(std::integral_constant<int, RT>(), std::integral_constant<int, NV>())
  HELD(64, 1);
  HELD(64, 2);
  HELD(64, 4);
  HELD(64, 8);
  HELD(256, 4);
  HELD(256, 8);
  HELD(256, 16);
  HELD(512, 16);
#undef HELD
  go(std::integral_constant<int, 1024>(), std::integral_constant<int, 0>());
}

}  // namespace omt

using namespace omt;

static int token_logps_fwd(const char* fn, const omt_logits* logits, float* logps, float* lse, double* lse64, void* stream) {
  if (int e = logits_check(fn, logits)) return e;
  if (logits->sequences * logits->length == 0) return OMT_OK;
  if (!logps || (!lse && !lse64)) return fail(OMT_INVALID, "%s: null pointer", fn);
  return token_logps(logits, {logps, lse, lse64, nullptr, nullptr}, stream_of(stream));
}
OMT_EXPORT int omt_token_logps_fwd(const omt_logits* logits, float* logps, float* lse, void* stream) {
  return token_logps_fwd("omt_token_logps_fwd", logits, logps, lse, nullptr, stream);
}
OMT_EXPORT int omt_token_logps_fwd64(const omt_logits* logits, float* logps, double* lse, void* stream) {
  return token_logps_fwd("omt_token_logps_fwd64", logits, logps, nullptr, lse, stream);
}

static int token_logps_bwd(const char* fn, const omt_logits* logits, const float* lse, const double* lse64, const float* g, void* gx,
                           void* stream) {
  if (int e = logits_check(fn, logits)) return e;
  if (logits->sequences * logits->length == 0) return OMT_OK;
  if ((!lse && !lse64) || !g || !gx) return fail(OMT_INVALID, "%s: null pointer", fn);
  return logit_grad(logits, {lse, lse64, nullptr, g, 1, 0, nullptr, 0, nullptr}, gx, stream_of(stream));
}
OMT_EXPORT int omt_token_logps_bwd(const omt_logits* logits, const float* lse, const float* g, void* gx, void* stream) {
  return token_logps_bwd("omt_token_logps_bwd", logits, lse, nullptr, g, gx, stream);
}
OMT_EXPORT int omt_token_logps_bwd64(const omt_logits* logits, const double* lse, const float* g, void* gx, void* stream) {
  return token_logps_bwd("omt_token_logps_bwd64", logits, nullptr, lse, g, gx, stream);
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
  if (kind != OMT_PREFERENCE_SIGMOID && smoothing != 0.0) return fail(OMT_INVALID, "%s: smoothing %g of kind %d", fn, smoothing, kind);
  if (n / 2 >= 1 << 22) return fail(OMT_UNSUPPORTED, "%s: %lld sequences", fn, (long long)n);
  if (!reference || !loss || !rewards) return fail(OMT_INVALID, "%s: null pointer", fn);
  const PreferencePlan p = preference_plan(n, logits->length);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.total())
    return fail(OMT_INVALID, "%s: workspace of %zu bytes at %p", fn, workspace_bytes, workspace);
  char* at = (char*)workspace;
  double* logps = (double*)at;
  RowStats* stats = (RowStats*)(at + p.logps);
  double* losses = (double*)(at + p.logps + p.stats);
  float* coefs = (float*)(at + p.logps + p.stats + p.losses);
  hipStream_t s = stream_of(stream);
  const int64_t pairs = n / 2;
  if (rows > 0)
    if (int e = token_logps(logits, {nullptr, nullptr, nullptr, logps, gx ? stats : nullptr}, s)) return e;
  const PairArgs a{logits->labels, logps, reference, logits->ignore_index, logits->length, pairs, kind, average, beta, smoothing,
                   rewards, coefs, losses};
  if (gx && rows > 0 && pairs <= kFewPairs && logits->length <= kFewPairsLength && row_bytes(logits) <= 32768) {
    for_type(logits, [&](auto t) {
      typedef decltype(t) T;
      for_row_threads(row_bytes(logits), [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        if constexpr (RT <= 256)
          launch_rows<RT>(few_pairs_grad_kernel<T, RT>, rows, s, rows_of(logits), a, (const RowStats*)stats, loss, (T*)gx);
      });
    });
    return launch_check("few_pairs_grad_kernel");
  }
  if (logits->length <= 2048) hipLaunchKernelGGL(preference_pair_kernel<256>, dim3((unsigned)pairs), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(preference_pair_kernel<1024>, dim3((unsigned)pairs), dim3(1024), 0, s, a);
  if (int e = launch_check("preference_pair_kernel")) return e;
  if (gx && rows > 0)
    return logit_grad(logits, {nullptr, nullptr, stats, coefs, 0, rows * row_bytes(logits) > kBackwardsBytes, losses, pairs, loss}, gx, s);
  hipLaunchKernelGGL(mean_loss_kernel, dim3(1), dim3(64), 0, s, losses, pairs, loss);
  return launch_check("mean_loss_kernel");
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
  if (by_sequence && logits->sequences >= 1 << 22) return fail(OMT_UNSUPPORTED, "%s: %lld sequences", fn, (long long)logits->sequences);
  if (!loss || !kl || (rows > 0 && (!old_logps || !advantages || !logps))) return fail(OMT_INVALID, "%s: null pointer", fn);
  const PolicyPlan p = policy_plan(logits->sequences, logits->length, by_sequence != 0);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.total())
    return fail(OMT_INVALID, "%s: workspace of %zu bytes at %p", fn, workspace_bytes, workspace);
  char* at = (char*)workspace;
  double *counts = (double*)at, *terms = (double*)(at + p.counts), *sums = (double*)(at + p.counts + p.terms);
  hipStream_t s = stream_of(stream);
  if (rows > 0) {
    const bool few = (by_sequence ? logits->length : rows) <= kFewLabels;
    if (!few) {
      hipLaunchKernelGGL(count_labels_kernel, dim3((unsigned)p.segments), dim3(1024), 0, s, logits->labels, rows, p.span,
                         logits->ignore_index, counts);
      if (int e = launch_check("count_labels_kernel")) return e;
    }
    const PolicyArgs a{old_logps, reference, advantages, advantage_sequence_stride, advantage_row_stride, few ? nullptr : counts, p.segments,
                       by_sequence, clip_low, clip_high, kl_weight, logps, terms, gx};
    for_type(logits, [&](auto t) {
      for_held_row(row_bytes(logits), [&](auto rt, auto nv) {
        constexpr int RT = decltype(rt)::value;
        launch_rows<RT>(policy_kernel<decltype(t), RT, decltype(nv)::value>, rows, s, rows_of(logits), a);
      });
    });
    if (int e = launch_check("policy_kernel")) return e;
  }
  const bool two = p.parts > 1;
  hipLaunchKernelGGL(sum_terms_kernel, dim3((unsigned)p.parts), dim3(1024), 0, s, terms, rows, cdiv(rows, p.parts), sums,
                     two ? nullptr : loss, two ? nullptr : kl);
  if (int e = launch_check("sum_terms_kernel")) return e;
  if (!two) return OMT_OK;
  hipLaunchKernelGGL(sum_terms_kernel, dim3(1), dim3(1024), 0, s, sums, p.parts, p.parts, sums, loss, kl);
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
