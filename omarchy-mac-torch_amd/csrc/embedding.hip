// Embedding: y[i] = scale * weight[token_i], and its gradient gw[v] = scale * (sum over i with token_i = v of gy[i]), the
// positions of a token in their order, so that the same inputs give the same bits: no atomics on values.
//
// The gradient sorts the positions by token (a stable sort by digits of up to 9 bits: one workgroup in LDS up to 2048
// positions; above, at most 64 workgroups, which count and then scatter each digit), cuts the sorted positions into runs of
// equal length, whatever the tokens' frequencies, and sums each run's rows of gy in float32: what begins and ends within a run
// is rounded and written at once, the sums of a token that reaches over runs are joined by a second launch. Rows that no
// position holds are written as zeros by further workgroups of the sort's launches, which it leaves most of the card to: at a
// vocabulary that is large beside the positions the sort takes no time of its own. Few positions, and a middling number of narrow
// rows, have ways of fewer launches (below). Bound by memory: gy is read once, gw written once.
//
// bfloat16, tokens as text has them: 65536 rows of 2048 from 131072 82 us (0.36 GB at 4.3 TB/s; 0.45 GB pass the caches, since eight of
// them read the frequent rows); the gradient of 32768 positions 148 us (0.67 GB at 4.5 TB/s), of which the sort with its rows of zeros
// 98, the sums 31 and the joins 6. 8191 positions to 256 x 128 float32 20.5 us, three launches.
//
// Tokens outside the vocabulary: a row of NaN (the first row is read in place of theirs, whatever it holds), and no part in the gradient.
#include <algorithm>

#include "block_fp8.h"

namespace omt {

struct TokenArray {
  const void* p;
  int wide;  // int64, else int32
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
};

// ---- forward --------------------------------------------------------------------------------------------------------

struct EmbedArgs {
  TokenArray tokens;
  const void* weight;
  void* y;
  int64_t n, vocab, dim;
  float scale;
};

// LANES threads to a row, eight consecutive columns to a thread at a time
template <class T, bool VEC, int LANES>
__global__ void __launch_bounds__(256) embedding_kernel(EmbedArgs a) {
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  if (row >= a.n) return;
  const int64_t token = a.tokens[row];
  const bool known = (uint64_t)token < (uint64_t)a.vocab;
  const T* w = (const T*)a.weight + (known ? token : 0) * a.dim;
  T* y = (T*)a.y + row * a.dim;
  const float scale = known ? a.scale : __builtin_nanf("");
  constexpr int U = 4;
  for (int64_t c = (int64_t)(threadIdx.x % LANES) * 8; c < a.dim; c += LANES * 8 * U) {
    f32x8 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load8<VEC>(w, c + u * LANES * 8, a.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) store8<VEC>(y, c + u * LANES * 8, a.dim, v[u] * scale);
  }
}

// ---- sorting positions by token -------------------------------------------------------------------------------------

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;  // a thread to each bin
constexpr int kSmallSort = 2048;  // positions that one workgroup sorts in LDS
constexpr int kSortTiles = 64;    // workgroups of a larger sort at most: each adds up the counts of all

// Tokens as keys: those that take part in the gradient, `vocab` for the others, which so come last.
struct KeyOf {
  TokenArray tokens;
  int64_t vocab, padding;
  __device__ __forceinline__ uint32_t operator()(int64_t i) const {
    const int64_t t = tokens[i];
    return (uint64_t)t < (uint64_t)vocab && t != padding ? (uint32_t)t : (uint32_t)vocab;
  }
};

// the wave's lanes, among those that are `on`, with this lane's digit
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool on, int bits) {
  uint64_t m = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const bool one = digit >> b & 1;
    const uint64_t with = __ballot(on && one);
    m &= one ? with : ~with;
  }
  return m;
}
__device__ __forceinline__ uint64_t lanes_below() { return (1ull << (threadIdx.x & 63)) - 1; }

// counts[digit] += the keys of [beg, end) with it, by one wave
template <class Key>
__device__ __forceinline__ void count_digits(uint32_t* counts, int64_t beg, int64_t end, Key key, int shift, int bits) {
  for (int64_t i = beg; i < end; i += 64) {
    const int64_t j = i + (threadIdx.x & 63);
    const bool on = j < end;
    const uint32_t digit = on ? key(j) >> shift & ((1u << bits) - 1) : 0;
    const uint64_t same = same_digit(digit, on, bits);
    if (on && !(same & lanes_below())) atomicAdd(&counts[digit], (uint32_t)__popcll(same));
  }
}
// put(j, place) for the keys of [beg, end) in order, by one wave; at[digit] is the digit's next place
template <class Key, class Put>
__device__ __forceinline__ void place_digits(uint32_t* at, int64_t beg, int64_t end, Key key, int shift, int bits, Put put) {
  for (int64_t i = beg; i < end; i += 64) {
    const int64_t j = i + (threadIdx.x & 63);
    const bool on = j < end;
    const uint32_t digit = on ? key(j) >> shift & ((1u << bits) - 1) : 0;
    const uint64_t same = same_digit(digit, on, bits), below = same & lanes_below();
    uint32_t first = 0;
    if (on && !below) first = atomicAdd(&at[digit], (uint32_t)__popcll(same));
    first = __shfl(first, on ? __ffsll((unsigned long long)same) - 1 : 0);
    if (on) put(j, first + (uint32_t)__popcll(below));
  }
}
// Of kBins values, one to each thread, the sum of those before it.
__device__ __forceinline__ uint32_t exclusive_scan(uint32_t v, uint32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t run = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t up = __shfl_up(run, d);
    if (lane >= d) run += up;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = run;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortWaves; ++i) run += i < wave ? sums[i] : 0;
  return run - v;
}
static_assert(kSortThreads == kBins, "a thread to each bin");

// Rows of the weight's gradient without positions, which workgroups beside a sort's write: those of [first, end), kZeroRows to
// a workgroup.
constexpr int kZeroRows = 64;
struct ZeroRows {
  void* gw;
  int64_t first, end, dim;
  int bytes;  // of an element
  __device__ __forceinline__ int64_t begin(int64_t group) const { return first + group * kZeroRows; }
};
__device__ __forceinline__ void write_zero_rows(const ZeroRows& z, int64_t begin, const uint8_t* holds) {
  const int rows = (int)min((int64_t)kZeroRows, z.end - begin), lane = threadIdx.x & 63;
  const int64_t size = z.dim * z.bytes;
  for (int r = threadIdx.x >> 6; r < rows; r += kSortWaves) {
    if (holds[r]) continue;
    char* row = (char*)z.gw + (begin + r) * size;
    // (rows of any size and alignment: whole vectors on 16 bytes, and the elements before and behind them)
    const int64_t head = min((int64_t)(0 - (uintptr_t)row & 15), size), body = (size - head) / 16, tail = head + body * 16;
    if (lane * z.bytes < head)
      z.bytes == 4 ? *(uint32_t*)(row + lane * 4) = 0 : *(uint16_t*)(row + lane * 2) = 0;
    if (tail + lane * z.bytes < size)
      z.bytes == 4 ? *(uint32_t*)(row + tail + lane * 4) = 0 : *(uint16_t*)(row + tail + lane * 2) = 0;
    for (int64_t i = lane; i < body; i += 64) __builtin_nontemporal_store(omt_u32x4{}, (omt_u32x4*)(row + head) + i);
  }
}

// Up to kSmallSort positions, all digits, in one workgroup.
__global__ void __launch_bounds__(kSortThreads) sort_small_kernel(KeyOf key, int n, int bits, int passes, uint32_t* keys_out,
                                                                  uint32_t* pos_out, ZeroRows zeros) {
  if (blockIdx.x > 0) {  // the positions are few: each workgroup looks through them
    __shared__ uint8_t holds[kZeroRows];
    const int64_t begin = zeros.begin(blockIdx.x - 1);
    if (threadIdx.x < kZeroRows) holds[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSortThreads) {
      const int64_t r = (int64_t)key(i) - begin;
      if ((uint64_t)r < kZeroRows) holds[r] = 1;
    }
    __syncthreads();
    return write_zero_rows(zeros, begin, holds);
  }
  __shared__ uint32_t keys[2][kSmallSort];
  __shared__ uint16_t pos[2][kSmallSort];
  __shared__ uint32_t counts[kSortWaves][kBins];
  __shared__ uint32_t sums[kSortWaves];
  const int wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys[0][i] = key(i), pos[0][i] = (uint16_t)i;
  const int share = (n + kSortThreads - 1) / kSortThreads * 64;  // consecutive positions of a wave
  const int beg = min(wave * share, n), end = min(beg + share, n);
  for (int p = 0; p < passes; ++p) {
    const uint32_t* from = keys[p & 1];
    const uint16_t* from_pos = pos[p & 1];
    uint32_t* to = keys[~p & 1];
    uint16_t* to_pos = pos[~p & 1];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) counts[w][threadIdx.x] = 0;
    __syncthreads();
    auto at = [&](int64_t j) { return from[j]; };
    count_digits(counts[wave], beg, end, at, p * bits, bits);
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) total += counts[w][threadIdx.x];
    uint32_t first = exclusive_scan(total, sums);
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = first;
      first += c;
    }
    __syncthreads();
    place_digits(counts[wave], beg, end, at, p * bits, bits, [&](int64_t j, uint32_t place) {
      to[place] = from[j];
      to_pos[place] = from_pos[j];
    });
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys_out[i] = keys[passes & 1][i], pos_out[i] = pos[passes & 1][i];
}

// The keys and positions that a pass of a larger sort reads: the tokens themselves, or the pass before.
struct SortFrom {
  KeyOf key;
  const uint32_t *keys, *pos;
};
struct SortArgs {
  SortFrom from;
  uint32_t *keys, *pos;  // what it writes
  uint32_t* counts;      // [workgroups][kBins]
  uint32_t* starts;      // [kBins + 1], or null: where each digit begins
  // (or null) of each token that occurs, one of its positions, written by the first launch. The others' entries are whatever the memory
  // held: an entry counts only if the token at that position is the row's, so nothing needs to be cleared first.
  uint32_t* marks;
  int64_t n, tile;  // positions, and how many to a workgroup
  unsigned tiles;   // workgroups that sort; those behind them write zeros
  int shift, bits;
  ZeroRows zeros;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t key_at(const SortFrom& f, int64_t j) {
  return FIRST ? f.key(j) : f.keys[j];
}
__device__ __forceinline__ void write_unmarked_rows(const SortArgs& a) {
  __shared__ uint8_t holds[kZeroRows];
  const int64_t begin = a.zeros.begin(blockIdx.x - a.tiles), row = begin + threadIdx.x;
  if (threadIdx.x < kZeroRows && row < a.zeros.end) {
    const uint32_t at = a.marks[row];
    holds[threadIdx.x] = at < a.n && a.from.key(at) == (uint32_t)row;
  }
  __syncthreads();
  write_zero_rows(a.zeros, begin, holds);
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  if (blockIdx.x >= a.tiles) return write_unmarked_rows(a);
  __shared__ uint32_t counts[kBins];
  counts[threadIdx.x] = 0;
  __syncthreads();
  const int64_t share = a.tile / kSortWaves;
  const int64_t beg = min(blockIdx.x * a.tile + (threadIdx.x >> 6) * share, a.n), end = min(beg + share, a.n);
  count_digits(counts, beg, end, [&](int64_t j) {
    const uint32_t key = key_at<FIRST>(a.from, j);
    if (FIRST && a.marks && key != (uint32_t)a.from.key.vocab) a.marks[key] = (uint32_t)j;
    return key;
  }, a.shift, a.bits);
  __syncthreads();
  a.counts[blockIdx.x * kBins + threadIdx.x] = counts[threadIdx.x];
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs a) {
  if (blockIdx.x >= a.tiles) return write_unmarked_rows(a);
  __shared__ uint32_t counts[kSortWaves][kBins];
  __shared__ uint32_t sums[kSortWaves];
  const int wave = threadIdx.x >> 6;
  uint32_t total = 0, before = 0;  // of this thread's digit, over all workgroups and over those before this one
#pragma unroll 8
  for (unsigned t = 0; t < a.tiles; ++t) {
    const uint32_t c = a.counts[t * kBins + threadIdx.x];
    total += c;
    before += t < blockIdx.x ? c : 0;
  }
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) counts[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t share = a.tile / kSortWaves;
  const int64_t beg = min(blockIdx.x * a.tile + wave * share, a.n), end = min(beg + share, a.n);
  auto key = [&](int64_t j) { return key_at<FIRST>(a.from, j); };
  count_digits(counts[wave], beg, end, key, a.shift, a.bits);
  uint32_t first = exclusive_scan(total, sums);
  if (a.starts && blockIdx.x == 0) {
    a.starts[threadIdx.x] = first;
    if (threadIdx.x == kBins - 1) a.starts[kBins] = first + total;
  }
  first += before;  // (the scan's barriers stand between the counts above and their use below)
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    const uint32_t c = counts[w][threadIdx.x];
    counts[w][threadIdx.x] = first;
    first += c;
  }
  __syncthreads();
  place_digits(counts[wave], beg, end, key, a.shift, a.bits, [&](int64_t j, uint32_t place) {
    a.keys[place] = key(j);
    a.pos[place] = FIRST ? (uint32_t)j : a.from.pos[j];
  });
}

// ---- sums of the sorted rows ----------------------------------------------------------------------------------------

struct SumArgs {
  const void* gy;
  const uint32_t *keys, *pos;  // sorted
  float* parts;                // [runs][2][dim]: what a run holds of a token that began before it, and of one that goes on after
  void* gw;
  int64_t n, vocab, dim;
  int64_t run, runs;  // positions to a run, and how many
  float scale;
};

// LANES threads to a run and 8 LANES columns
template <class T, bool VEC, int LANES>
__global__ void __launch_bounds__(256) embedding_sum_kernel(SumArgs a) {
  const int64_t chunks = (a.dim + LANES * 8 - 1) / (LANES * 8);
  const int64_t unit = blockIdx.x * (int64_t)(256 / LANES) + threadIdx.x / LANES;
  const int64_t run = unit / chunks, c = (unit % chunks * LANES + threadIdx.x % LANES) * 8;
  if (run >= a.runs || c >= a.dim) return;
  const int64_t beg = run * a.run, end = min(beg + a.run, a.n);
  const uint32_t none = (uint32_t)a.vocab;
  uint32_t key = a.keys[beg];
  bool began = beg > 0 && a.keys[beg - 1] == key;  // before this run
  f32x8 sum = {};
  auto put = [&](bool goes_on) {
    if (key == none) return;
    if (began || goes_on) store8<false>(a.parts + (run * 2 + (began ? 0 : 1)) * a.dim, c, a.dim, sum);
    else store8<VEC>((T*)a.gw + key * a.dim, c, a.dim, sum * a.scale);
  };
  constexpr int U = 8;
  uint32_t k[U], at[U];
  auto look = [&](int64_t i) {
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = i + u < end ? a.keys[i + u] : none, at[u] = i + u < end ? a.pos[i + u] : 0;
  };
  look(beg);
  for (int64_t i = beg; i < end; i += U) {
    f32x8 v[U];
    uint32_t now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      now[u] = k[u];
      v[u] = k[u] != none ? load8<VEC>((const T*)a.gy + (int64_t)at[u] * a.dim, c, a.dim) : f32x8{};
    }
    if (i + U < end) look(i + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= end) break;
      if (now[u] != key) {
        put(false);
        key = now[u], began = false, sum = f32x8{};
      }
      sum += v[u];
    }
  }
  put(end < a.n && a.keys[end] == key);
}

// gw of the tokens that began in run blockIdx.x and go on after it: the runs' sums, in order; 8 LANES columns to a workgroup
template <class T, bool VEC, int LANES>
__global__ void __launch_bounds__(256) embedding_join_kernel(SumArgs a) {
  __shared__ f32x8 sums[256];
  const int64_t run = blockIdx.x, beg = run * a.run, end = min(beg + a.run, a.n);
  const uint32_t key = a.keys[end - 1];
  if (key == (uint32_t)a.vocab || end == a.n || a.keys[end] != key) return;  // (the same for the whole workgroup)
  if (beg > 0 && a.keys[beg - 1] == key) return;                            // began before
  // the last run that begins with it: the wave's lanes cut what is left of the runs into 64 at a time
  int64_t last = run, over = a.runs;  // it begins with the key (or holds the token's beginning); it does not
  while (over - last > 1) {
    const int64_t step = (over - last + 63) / 64, at = last + ((threadIdx.x & 63) + 1) * step;
    const int64_t with = __popcll(__ballot(at < over && a.keys[at * a.run] == key));
    over = min(over, last + (with + 1) * step);
    last += with * step;
  }
  constexpr int GROUPS = 256 / LANES;
  const int g = threadIdx.x / LANES;
  const int64_t count = last - run, share = (count + GROUPS - 1) / GROUPS;  // runs after this one, and to a group of threads
  const int64_t from = run + 1 + min(g * share, count), to = min(from + share, last + 1);
  const int64_t c = ((int64_t)blockIdx.y * LANES + threadIdx.x % LANES) * 8;
  f32x8 sum = {};
  if (g == 0) sum = load8<false>(a.parts + (run * 2 + 1) * a.dim, c, a.dim);
#pragma unroll 4
  for (int64_t r = from; r < to; ++r) sum += load8<false>(a.parts + r * 2 * a.dim, c, a.dim);
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (g > 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) sum += sums[i * LANES + threadIdx.x];
  store8<VEC>((T*)a.gw + key * a.dim, c, a.dim, sum * a.scale);
}

// Limits: positions and keys are 32-bit, and a launch holds fewer than 2^24 workgroups of 256 threads along one dimension.
constexpr int64_t kEmbedMaxTokens = 1 << 28, kEmbedMaxVocab = 1 << 28, kEmbedMaxDim = 1 << 16;
constexpr int64_t kEmbedMaxGroups = (1 << 24) - 1;

// ---- few positions ---------------------------------------------------------------------------------------------------

// Few positions in one launch instead of three or more: a workgroup to ROWS rows of the weight and 8 LANES columns looks through all
// tokens, sorts the positions of its rows by row in LDS, and sums them in runs as above, its groups of LANES threads a run each,
// joined in LDS. Rows of zeros are among those of each workgroup.
constexpr int kFewTokens = 2048;
struct FewArgs {
  KeyOf key;
  const void* gy;
  void* gw;
  int n;
  int64_t vocab, dim;
  float scale;
};
// Entries 0..n by row, in LDS: first(j) is entry j's row, or -1, and again(j) the same when it is asked for once more; kept(j) is what
// at[] gets for it. Entries of one row stay in order; starts[r] is where row r begins. All 512 threads call it.
template <int ROWS, class First, class Again, class Kept>
__device__ __forceinline__ void sort_rows(int n, First first, Again again, Kept kept, uint32_t (*counts)[ROWS], uint32_t* starts,
                                          uint16_t* at, uint8_t* of) {
  constexpr int WAVES = 8, BITS = ROWS == 256 ? 8 : ROWS == 64 ? 6 : 3, EACH = ROWS > 64 ? ROWS / 64 : 1;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int share = (n + 511) / 512 * 64, beg = min(wave * share, n), end = min(beg + share, n);
  for (int i = threadIdx.x; i < WAVES * ROWS; i += 512) counts[0][i] = 0;
  __syncthreads();
  for (int i = beg; i < end; i += 256) {
    int r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = i + u * 64 + lane < end ? first(i + u * 64 + lane) : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint64_t same = same_digit((uint32_t)r[u], r[u] >= 0, BITS);
      if (r[u] >= 0 && !(same & lanes_below())) counts[wave][r[u]] += (uint32_t)__popcll(same);
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
  if (wave == 0) {
    uint32_t total = 0;
    if (lane * EACH < ROWS)
      for (int k = 0; k < EACH; ++k)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) total += counts[w][lane * EACH + k];
    uint32_t run = total;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t up = __shfl_up(run, d);
      if (lane >= d) run += up;
    }
    if (lane == 63) starts[ROWS] = run;
    run -= total;
    if (lane * EACH < ROWS)
      for (int k = 0; k < EACH; ++k) {
        starts[lane * EACH + k] = run;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const uint32_t c = counts[w][lane * EACH + k];
          counts[w][lane * EACH + k] = run;
          run += c;
        }
      }
  }
  __syncthreads();
  for (int i = beg; i < end; i += 64) {
    const int j = i + lane, r = j < end ? again(j) : -1;
    const bool on = r >= 0;
    const uint64_t same = same_digit((uint32_t)r, on, BITS), below = same & lanes_below();
    const uint32_t next = on ? counts[wave][r] : 0;
    __builtin_amdgcn_wave_barrier();
    if (on) {
      const uint32_t place = next + (uint32_t)__popcll(below);
      at[place] = kept(j);
      of[place] = (uint8_t)r;
      if (!below) counts[wave][r] = next + (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
}
// put(row, sum) of each of the rows that the m sorted entries hold, by groups of LANES threads; all 512 threads call it
template <class T, bool VEC, int LANES, class Put>
__device__ __forceinline__ void sum_sorted(const uint16_t* at, const uint8_t* of, int m, f32x8 (*parts)[512], const T* gy, int64_t c,
                                           int64_t dim, Put put) {
  constexpr int GROUPS = 512 / LANES;
  const int run = (m + GROUPS - 1) / GROUPS, g = threadIdx.x / LANES;
  const int from = min(g * run, m), to = min(from + run, m);
  bool goes_on = false;
  if (from < to) {
    int row = of[from];
    bool began = from > 0 && of[from - 1] == row;
    f32x8 sum = {};
    constexpr int U = 8;
    for (int i = from; i < to; i += U) {
      f32x8 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = i + u < to ? load8<VEC>(gy + (int64_t)at[i + u] * dim, c, dim) : f32x8{};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= to) break;
        if (of[i + u] != row) {
          if (began) parts[0][threadIdx.x] = sum;
          else put(row, sum);
          row = of[i + u], began = false, sum = f32x8{};
        }
        sum += v[u];
      }
    }
    goes_on = to < m && of[to] == row;
    if (began) parts[0][threadIdx.x] = sum;
    else if (goes_on) parts[1][threadIdx.x] = sum;
    else put(row, sum);
    goes_on = goes_on && !began;
  }
  __syncthreads();
  if (!goes_on) return;
  // a row that began in this run and goes on: the next runs' sums of it, in order
  const int row = of[to - 1];
  f32x8 sum = parts[1][threadIdx.x];
  for (int k = g + 1; k * run < m && of[k * run] == row; ++k) sum += parts[0][k * LANES + threadIdx.x % LANES];
  put(row, sum);
}

template <class T, bool VEC, int LANES, int ROWS>
__global__ void __launch_bounds__(512) embedding_few_kernel(FewArgs a) {
  constexpr int NONE = 255;
  __shared__ uint8_t row_of[kFewTokens];  // of each token: the workgroup's row, or NONE
  __shared__ uint16_t at[kFewTokens];     // positions, by row and then in order
  __shared__ uint8_t of[kFewTokens];      // their rows
  __shared__ uint32_t counts[8][ROWS], starts[ROWS + 1];
  __shared__ f32x8 parts[2][512];  // of a run: what began before it, what goes on after
  const int64_t begin = (int64_t)blockIdx.x * ROWS;
  sort_rows<ROWS>(
      a.n,
      [&](int j) {
        const int64_t row = (int64_t)a.key(j) - begin;
        const int r = (uint64_t)row < ROWS && begin + row < a.vocab ? (int)row : -1;
        row_of[j] = (uint8_t)(r < 0 ? NONE : r);
        return r;
      },
      [&](int j) { return row_of[j] == NONE ? -1 : (int)row_of[j]; }, [&](int j) { return (uint16_t)j; }, counts, starts, at, of);
  const int64_t c = ((int64_t)blockIdx.y * LANES + threadIdx.x % LANES) * 8;
  auto put = [&](int row, f32x8 sum) { store8<VEC>((T*)a.gw + (begin + row) * a.dim, c, a.dim, sum * a.scale); };
  for (int r = threadIdx.x / LANES; r < ROWS && begin + r < a.vocab; r += 512 / LANES)
    if (starts[r] == starts[r + 1]) put(r, f32x8{});
  sum_sorted<T, VEC, LANES>(at, of, (int)starts[ROWS], parts, (const T*)a.gy, c, a.dim, put);
}

// A middling number of positions, which one pass of the sort has cut into bins by their tokens' low bits, so that neighbours among
// the tokens, the frequent ones of a vocabulary, lie in different ones: a workgroup to a bin and 8 LANES columns does as above.
constexpr int kBinTokens = 8192;
struct BinArgs {
  const uint32_t *keys, *pos, *starts;  // by bin; where each begins
  const void* gy;
  void* gw;
  int64_t vocab, dim;
  int bits;  // 2^bits bins
  float scale;
};
template <class T, bool VEC, int LANES, int ROWS>
__global__ void __launch_bounds__(512) embedding_bin_kernel(BinArgs a) {
  __shared__ uint16_t at[kBinTokens];
  __shared__ uint8_t of[kBinTokens];
  __shared__ uint32_t counts[8][ROWS], starts[ROWS + 1];
  __shared__ f32x8 parts[2][512];
  const uint32_t bin = blockIdx.x, base = a.starts[bin], n = a.starts[bin + 1] - base;
  auto row = [&](int j) {
    const uint32_t key = a.keys[base + j];
    return key < a.vocab ? (int)(key >> a.bits) : -1;
  };
  sort_rows<ROWS>((int)n, row, row, [&](int j) { return (uint16_t)a.pos[base + j]; }, counts, starts, at, of);
  const int64_t c = ((int64_t)blockIdx.y * LANES + threadIdx.x % LANES) * 8;
  auto put = [&](int r, f32x8 sum) {
    store8<VEC>((T*)a.gw + (((int64_t)r << a.bits) + bin) * a.dim, c, a.dim, sum * a.scale);
  };
  for (int r = threadIdx.x / LANES; r < ROWS && ((int64_t)r << a.bits) + bin < a.vocab; r += 512 / LANES)
    if (starts[r] == starts[r + 1]) put(r, f32x8{});
  sum_sorted<T, VEC, LANES>(at, of, (int)starts[ROWS], parts, (const T*)a.gy, c, a.dim, put);
}

// How a gradient of few positions is cut, by what it measured: lanes 0 where the sort's launches take less. Skewed tokens, us, with 8
// rows to a workgroup, with 64, and by the sort:
//   300 tokens     256 x 128 bfloat16  5.9,  8.0, 15.7   64 x 4096  6.3,  9.1, 14.6   1000 x 1000 float32  9.6,  7.1, 16.6
//   1024                               8.3, 13.3, 18.0             13.0, 16.4, 16.2                       12.3, 12.2, 19.3
//   2048                              11.9,    -, 21.1             20.9,    -, 23.1                       16.4,    -, 24.4
//   4096                              20.2,    -, 22.7             37.5,    -, 28.6                       26.2,    -, 36.1
// and, of many rows, with 64 rows and 64 lanes to a workgroup at 256, 300, 512 and 1024 tokens, bfloat16: 32768 x 512 13.4, 14.9, 18.2, 28.7
// (in bins 17.6, 18.2, 18.9, 20.4), 131072 x 512 -, 22.3, -, 28.1 (-, 31.1, -, 33.0), 32768 x 4096 53.3, 59.6, 70.3, - (by the sort 61.4, 61.3,
// 61.5). The rule's border of 256 keeps to where the widest of these rows gain; narrower ones would up to 512.
struct FewPlan {
  int lanes, rows;
};
static FewPlan few_plan(int64_t n, int64_t vocab, int64_t dim) {
  const int64_t groups = cdiv(vocab, 8) * cdiv(dim, 128);  // workgroups of 8 rows
  if (n <= 1024) {
    if (groups <= 512) return {16, 8};
    if (cdiv(vocab, 64) * cdiv(dim, 512) < 512) return {16, 64};
    return n <= 256 ? FewPlan{64, 64} : FewPlan{0, 0};
  }
  return n <= kFewTokens && groups <= 2048 ? FewPlan{16, 8} : FewPlan{0, 0};
}

// Threads to a bin's columns, 0 where the sort's launches take less: where the columns are few, since each workgroup's share of them sorts
// the bin again. Skewed tokens, us, in bins and by the sort, at 2049, 4096 and 8192 of them:
//   16 lanes   256 x 128 bfloat16  18.7, 20.9, 24.6 and 22.3, 22.6, 22.7   16384 x 64 18.4, 19.7, 22.1 and 34.4, 35.6, 35.1
//              50021 x 100 float32 23.9, 26.9, 30.1 and 40.5, 42.1, 41.1
//   64 lanes   4096 x 512 bfloat16 18.5, 22.7, 33.4 and 32.3, 33.6, 34.4   131072 x 512 40.0, 46.3, 56.8 and 44.7, 46.0, 48.4
//              300 x 512 19.9, 26.2 and 21.3, 22.0 (tokens of one digit)   16384 x 1024 24.7, 31.3 and 34.5, 37.6
//              32768 x 1024 float32 44.2, 53.0 and 43.8, 45.4              16384 x 2048 50.9, 62.7 and 45.9, 48.1
// (256 rows of 128 at 8192 are 2 us over the sort: one rule for all that is narrow.) Fewer, where one launch is not taken either: 300 and 1024
// to 32768 x 512 18.2, 20.4 and 18.7, 21.7, to 131072 x 512 31.1, 33.0 and 37.2, 38.0, to 16384 x 1024 20.2, 22.3 and 18.7, 21.4; 300 to 131072 x 128
// 18.5 and 25.3.
static int bin_lanes(int64_t n, int64_t vocab, int64_t dim) {
  if (vocab > (int64_t)256 << kDigitBits) return 0;
  if (dim <= 128) return n <= kBinTokens ? 16 : 0;
  if (vocab < kBins || n > kBinTokens / 2 || dim > 1024) return 0;
  return dim <= 512 || vocab * dim <= 1 << 24 ? 64 : 0;
}

// ---- plans ----------------------------------------------------------------------------------------------------------

// Positions to a run: enough runs for the card's threads, no fewer positions than keep the joined sums few.
static int64_t run_length(int64_t n, int64_t dim) {
  const int64_t units = cdiv(dim, 512);
  return std::min<int64_t>(256, std::max<int64_t>(16, cdiv(n * units, 4096)));
}
static int digits_of(int64_t vocab) {
  int bits = 1;
  while ((int64_t)1 << bits <= vocab) ++bits;  // the key `vocab` among them
  return bits;
}
struct EmbedPlan {
  FewPlan few;  // one launch, or
  int bins;     // sorted into bins, with so many lanes, or
  int64_t run, runs;
  size_t starts, counts, marks, sorted, parts;  // bytes: of one array each
  size_t total() const { return few.lanes ? 0 : starts + counts + marks + (bins ? 2 : 4) * sorted + parts; }
};
static EmbedPlan embed_plan(int64_t n, int64_t vocab, int64_t dim) {
  EmbedPlan p{};
  p.few = few_plan(n, vocab, dim);
  p.bins = p.few.lanes ? 0 : bin_lanes(n, vocab, dim);
  p.sorted = (size_t)cdiv(n, 64) * 256;
  p.counts = n > kSmallSort || p.bins ? (size_t)kSortTiles * kBins * 4 : 0;
  if (p.bins) {
    p.starts = (size_t)(kBins + 64) * 4;
    return p;
  }
  p.run = run_length(n, dim);
  p.runs = cdiv(n, p.run);
  p.marks = n > kSmallSort ? (size_t)cdiv(vocab, 64) * 256 : 0;
  p.parts = (size_t)p.runs * 2 * dim * 4;
  return p;
}

static bool on16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}
static int embed_check(const char* fn, int dtype, int token_dtype, int64_t n, int64_t vocab, int64_t dim) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "%s: dtype %d", fn, dtype);
  if (token_dtype != OMT_DT_I64 && token_dtype != OMT_DT_I32) return fail(OMT_INVALID, "%s: tokens of dtype %d", fn, token_dtype);
  if (n < 0 || vocab < 1 || dim < 1)
    return fail(OMT_INVALID, "%s: %lld tokens, weight %lld x %lld", fn, (long long)n, (long long)vocab, (long long)dim);
  return OMT_OK;
}
// go(LANES): threads to a row of `dim`
template <class Go>
static void for_lanes(int64_t dim, Go go) {
  if (dim <= 64) go(std::integral_constant<int, 8>());
  else if (dim <= 128) go(std::integral_constant<int, 16>());
  else if (dim <= 256) go(std::integral_constant<int, 32>());
  else go(std::integral_constant<int, 64>());
}

}  // namespace omt

using namespace omt;

OMT_EXPORT int omt_embedding_fwd(int dtype, int token_dtype, int64_t n, int64_t vocab, int64_t dim, const void* tokens,
                                 const void* weight, float scale, void* y, void* stream) {
  if (int e = embed_check("omt_embedding_fwd", dtype, token_dtype, n, vocab, dim)) return e;
  if (n == 0) return OMT_OK;
  if (!tokens || !weight || !y) return fail(OMT_INVALID, "omt_embedding_fwd: null pointer");
  const bool vec = dim % 8 == 0 && on16({weight, y});
  const EmbedArgs a{{tokens, token_dtype == OMT_DT_I64}, weight, y, n, vocab, dim, scale};
  for_lanes(dim, [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    // a dimension of the grid holds fewer than 2^32 threads: 2^21 workgroups along it, the rest along the other
    const int64_t groups = cdiv(n, 256 / LANES), along = std::min<int64_t>(groups, 1 << 21);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)along, (unsigned)cdiv(groups, along)), dim3(256), 0, stream_of(stream), a);
    };
    if (dtype == OMT_DT_F32) vec ? go(embedding_kernel<float, true, LANES>) : go(embedding_kernel<float, false, LANES>);
    else vec ? go(embedding_kernel<__bf16, true, LANES>) : go(embedding_kernel<__bf16, false, LANES>);
  });
  return launch_check("embedding_kernel");
}

OMT_EXPORT size_t omt_embedding_bwd_workspace(int64_t n, int64_t vocab, int64_t dim) {
  if (n < 0 || n > kEmbedMaxTokens || vocab < 1 || dim < 1) return 0;
  return embed_plan(n, vocab, dim).total();
}

OMT_EXPORT int omt_embedding_bwd(int dtype, int token_dtype, int64_t n, int64_t vocab, int64_t dim, const void* gy,
                                 const void* tokens, int64_t padding_idx, float scale, void* gweight, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  const char* fn = "omt_embedding_bwd";
  if (int e = embed_check(fn, dtype, token_dtype, n, vocab, dim)) return e;
  if (n > kEmbedMaxTokens || vocab > kEmbedMaxVocab || dim > kEmbedMaxDim || cdiv(n, run_length(n, dim)) * cdiv(dim, 64) > kEmbedMaxGroups)
    return fail(OMT_UNSUPPORTED, "%s: %lld tokens, weight %lld x %lld", fn, (long long)n, (long long)vocab, (long long)dim);
  if (!gweight || (n > 0 && (!gy || !tokens))) return fail(OMT_INVALID, "%s: null pointer", fn);
  hipStream_t s = stream_of(stream);
  const KeyOf key{{tokens, token_dtype == OMT_DT_I64}, vocab, padding_idx};
  const bool vec = dim % 8 == 0 && on16({gy, gweight});
  const EmbedPlan p = embed_plan(n, vocab, dim);
  if (const FewPlan few = p.few; few.lanes) {
    const FewArgs a{key, gy, gweight, (int)n, vocab, dim, scale};
    const dim3 grid((unsigned)cdiv(vocab, few.rows), (unsigned)cdiv(dim, few.lanes * 8));
    auto go = [&](auto lanes, auto rows) {
      constexpr int LANES = decltype(lanes)::value, ROWS = decltype(rows)::value;
      auto with = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, s, a); };
      if (dtype == OMT_DT_F32) vec ? with(embedding_few_kernel<float, true, LANES, ROWS>) : with(embedding_few_kernel<float, false, LANES, ROWS>);
      else vec ? with(embedding_few_kernel<__bf16, true, LANES, ROWS>) : with(embedding_few_kernel<__bf16, false, LANES, ROWS>);
    };
    if (few.lanes == 64) go(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
    else if (few.rows == 64) go(std::integral_constant<int, 16>(), std::integral_constant<int, 64>());
    else go(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    return launch_check("embedding_few_kernel");
  }
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.total())
    return fail(OMT_INVALID, "%s: workspace of %zu bytes at %p", fn, workspace_bytes, workspace);
  char* at = (char*)workspace;
  auto array = [&](size_t size) {
    uint32_t* a = (uint32_t*)at;
    at += size;
    return a;
  };
  uint32_t *starts = array(p.starts), *counts = array(p.counts), *marks = array(p.marks), *keys[2], *pos[2];
  for (int i = 0; i < (p.bins ? 1 : 2); ++i) keys[i] = array(p.sorted), pos[i] = array(p.sorted);
  const int64_t tile = cdiv(std::max<int64_t>(1024, cdiv(n, kSortTiles)), kSortThreads) * kSortThreads;
  const unsigned tiles = (unsigned)cdiv(n, tile);
  if (p.bins) {
    const int bits = std::min(kDigitBits, digits_of(vocab));
    const SortArgs q{{key, nullptr, nullptr}, keys[0], pos[0], counts, starts, nullptr, n, tile, tiles, 0, bits, {}};
    hipLaunchKernelGGL(sort_count_kernel<true>, dim3(tiles), dim3(kSortThreads), 0, s, q);
    if (int e = launch_check("sort_count_kernel")) return e;
    hipLaunchKernelGGL(sort_place_kernel<true>, dim3(tiles), dim3(kSortThreads), 0, s, q);
    if (int e = launch_check("sort_place_kernel")) return e;
    const BinArgs a{keys[0], pos[0], starts, gy, gweight, vocab, dim, bits, scale};
    auto go = [&](auto lanes, auto rows) {
      constexpr int LANES = decltype(lanes)::value, ROWS = decltype(rows)::value;
      const dim3 grid(1u << bits, (unsigned)cdiv(dim, LANES * 8));
      auto with = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, s, a); };
      if (dtype == OMT_DT_F32) vec ? with(embedding_bin_kernel<float, true, LANES, ROWS>) : with(embedding_bin_kernel<float, false, LANES, ROWS>);
      else vec ? with(embedding_bin_kernel<__bf16, true, LANES, ROWS>) : with(embedding_bin_kernel<__bf16, false, LANES, ROWS>);
    };
    auto by_rows = [&](auto lanes) {
      if (cdiv(vocab, (int64_t)1 << bits) <= 64) go(lanes, std::integral_constant<int, 64>());
      else go(lanes, std::integral_constant<int, 256>());
    };
    if (p.bins == 16) by_rows(std::integral_constant<int, 16>());
    else by_rows(std::integral_constant<int, 64>());
    return launch_check("embedding_bin_kernel");
  }
  const int all = digits_of(vocab), passes = (all + kDigitBits - 1) / kDigitBits, bits = (all + passes - 1) / passes;
  int last = 0;
  const int64_t zero_groups = cdiv(vocab, kZeroRows);
  const int bytes = dtype == OMT_DT_F32 ? 4 : 2;
  if (n <= kSmallSort) {
    hipLaunchKernelGGL(sort_small_kernel, dim3((unsigned)(1 + zero_groups)), dim3(kSortThreads), 0, s, key, (int)n, bits, passes,
                       keys[0], pos[0], ZeroRows{gweight, 0, vocab, dim, bytes});
    if (int e = launch_check("sort_small_kernel")) return e;
  } else {
    // the rows of zeros, in equal shares beside every launch but the first, which marks the others
    const int64_t share = cdiv(zero_groups, 2 * passes - 1);
    for (int q = 0; q < 2 * passes; ++q) {
      const int64_t done = std::min(zero_groups, std::max(0, q - 1) * share), more = q ? std::min(share, zero_groups - done) : 0;
      const int pass = q / 2;
      const SortArgs a{{key, keys[~pass & 1], pos[~pass & 1]}, keys[pass & 1], pos[pass & 1], counts, nullptr, marks, n, tile, tiles, pass * bits,
                       bits, {gweight, done * kZeroRows, std::min(vocab, (done + more) * kZeroRows), dim, bytes}};
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tiles + (unsigned)more), dim3(kSortThreads), 0, s, a);
      };
      if (q % 2 == 0) pass ? go(sort_count_kernel<false>) : go(sort_count_kernel<true>);
      else pass ? go(sort_place_kernel<false>) : go(sort_place_kernel<true>);
      if (int e = launch_check(q % 2 ? "sort_place_kernel" : "sort_count_kernel")) return e;
      last = pass & 1;
    }
  }
  int status = OMT_OK;
  for_lanes(dim, [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    const int64_t units = p.runs * cdiv(dim, LANES * 8), groups = cdiv(units, 256 / LANES);
    const SumArgs a{gy, keys[last], pos[last], (float*)at, gweight, n, vocab, dim, p.run, p.runs, scale};
    auto go = [&](auto kernel, dim3 grid) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    const dim3 grid((unsigned)groups);
    if (dtype == OMT_DT_F32) vec ? go(embedding_sum_kernel<float, true, LANES>, grid) : go(embedding_sum_kernel<float, false, LANES>, grid);
    else vec ? go(embedding_sum_kernel<__bf16, true, LANES>, grid) : go(embedding_sum_kernel<__bf16, false, LANES>, grid);
    status = launch_check("embedding_sum_kernel");
    if (status || p.runs < 2) return;
    const dim3 joins((unsigned)p.runs, (unsigned)cdiv(dim, LANES * 8));
    if (dtype == OMT_DT_F32) vec ? go(embedding_join_kernel<float, true, LANES>, joins) : go(embedding_join_kernel<float, false, LANES>, joins);
    else vec ? go(embedding_join_kernel<__bf16, true, LANES>, joins) : go(embedding_join_kernel<__bf16, false, LANES>, joins);
    status = launch_check("embedding_join_kernel");
  });
  return status;
}
