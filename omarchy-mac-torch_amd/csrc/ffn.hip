// The feed-forward operators over their matrix products (ffn_gemm.h): which tiles and shares run, operands laid out for
// them, the sums of shares, and the elementwise part of the gated block's backward.
//
//     forward    g = x Wg^T, u = x Wu^T, h = act(g) u
//     backward   dg = gh u act'(g), du = gh act(g)
//                gx = dg Wg + du Wu,  gWg = dg^T x,  gWu = du^T x
//
// The tiles read operands along the reduction, 16 bytes at a time, or, in bfloat16 with rows on 16 bytes, across it, and
// transpose in their LDS reads. There the backward lays out dg and du once, side by side: the product for gx reduces over
// both and takes the weights as they are, one after the other; the one for the weights' gradients takes dg and du, and x,
// across. Otherwise dg and du are laid out twice, by rows and transposed (one below the other), and x and the weights
// transposed: 64 x 64 blocks through LDS, read and written once. At 8192 x 4096 x 8192 bfloat16 the transposing layouts
// take 57 us for dg and du, 72 for the weights and 25 for x; a product across costs 0 to 3% more than one along.
#include <algorithm>

#include "ffn_few.h"

namespace omt {

// ---- operands laid out for the tiles ------------------------------------------------------------------------------------

// Rows copied to a pitch that is a multiple of 16 bytes, zeros past their end; 16 bytes to a thread (8192 x 4095
// bfloat16: 34 us, 4 TB/s; element by element 43).
template <class T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T* __restrict__ src, int64_t rows, int64_t cols,
                                                       int64_t pitch, T* __restrict__ dst) {
  constexpr int N = 16 / sizeof(T);
  const int64_t per = pitch / N, total = rows * per, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    const int64_t r = i / per, c = (i - r * per) * N;
    union {
      T e[N];
      uint4 all;
    } v;
    const T* p = src + r * cols + c;
    if (c + N <= cols) {
      __builtin_memcpy(&v, p, sizeof(v));  // at its type's alignment
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v.e[e] = c + e < cols ? p[e] : T(0);
    }
    *(uint4*)(dst + r * pitch + c) = v.all;
  }
}

// Where lines of an operand go: bfloat16 (kBf16), or float32 as two halves (kSplit). There the 32 elements that a step of
// the tiles reads of a line are scaled by one power of two, so that the largest lies in [2^14, 2^15), and each is held as
// the nearest float16 and the float16 nearest to what is left: 22 bits, or 2^-40 of the largest where that is more. 32
// high halves, then the 32 low ones; the scales lie by step, then line.
// A group that holds an infinity or NaN gives nothing finite, whatever it meets; what counts is where each product is
// infinite, of which sign, and where it is NaN. Its high halves are the signs (0 for zeros, NaN for NaN), its low ones 0 but for the
// infinities, which lie there, and its scale is 1. An infinity then meets the other line's high half once, and not its low one,
// whose sign is its own: inf times v is inf by v's sign, and NaN for 0; two infinities meet each other's sign. So that a high
// half is 0 for zeros alone, smaller values have float16's smallest there, and the low half takes it back.
struct Lines {
  char* p = nullptr;
  int64_t pitch = 0;       // bytes
  float* scale = nullptr;  // kSplit: [pitch / 128][scale_lines]
  int64_t scale_lines = 0;
};
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// 8 elements (at: a multiple of 8) of a line; kSplit: the four threads of a quad call it together for a group of 32
template <int FMT>
__device__ __forceinline__ void write8(const Lines& d, int64_t line, int64_t at, f32x8 v) {
  if constexpr (FMT == kBf16) {
    store8<true>((__bf16*)(d.p + line * d.pitch), at, d.pitch / 2, v);
  } else {
    uint32_t b = abs_bits8(v);
    b = max_u32(b, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
    b = max_u32(b, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
    float scale = 1.f;
    half8 hi, lo = {};
    if (b < 0x7f800000u) {
      const uint32_t e = max_u32(b >> 23, 15u);
      const f32x8 w = v * __builtin_bit_cast(float, (268u - e) << 23);
      scale = __builtin_bit_cast(float, (e - 14u) << 23);
      hi = __builtin_convertvector(w, half8);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (hi[e] == 0 && v[e] != 0.f) hi[e] = (_Float16)copysignf(0x1p-24f, v[e]);
      lo = __builtin_convertvector(w - __builtin_convertvector(hi, f32x8), half8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hi[e] = (_Float16)(v[e] == 0.f || v[e] != v[e] ? v[e] : copysignf(1.f, v[e]));
        if (abs_bits(v[e]) == 0x7f800000u) lo[e] = (_Float16)v[e];
      }
    }
    char* p = d.p + line * d.pitch + (at >> 5) * 128 + (at & 31) * 2;
    *(half8*)p = hi;
    *(half8*)(p + 64) = lo;
    if ((at & 31) == 0) d.scale[(at >> 5) * d.scale_lines + line] = scale;
  }
}

// Blocks of 64 x 64 elements: thread t has eight consecutive ones of rows t / 8 and t / 8 + 32. Columns go through LDS, rows
// of 65 floats: eight lanes of a row and eight rows write 64 banks, and lines read as columns do too.
constexpr int kBlk = 64, kBlkPitch = 65;
__device__ __forceinline__ void to_lds(float* blk, int row, int at, f32x8 v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) blk[row * kBlkPitch + at + e] = v[e];
}
// the block's columns as lines line0.. (below `lines`) of d, elements at.. of each
template <int FMT>
__device__ __forceinline__ void write_columns(const float* blk, const Lines& d, int64_t line0, int64_t lines, int64_t at) {
  const int part = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int line = (threadIdx.x >> 3) + 32 * i;
    if (line0 + line >= lines) break;  // all eight threads of a line
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = blk[(part + e) * kBlkPitch + line];
    write8<FMT>(d, line0 + line, at + part, v);
  }
}

// Up to three matrices of floats with rows of one length as kSplit lines, zeros past their end up to a multiple of 64: one
// launch for all (4096 x 1024 x 4096: 20.0 us, 5 TB/s; three launches took 23.7).
struct SplitArgs {
  const float* src[3];
  int64_t rows[3];
  Lines d[3];
};
template <bool VEC>
__global__ void __launch_bounds__(256) split_rows_kernel(SplitArgs a, int64_t cols) {
  const int z = blockIdx.z;
  const int64_t at = (int64_t)blockIdx.y * kBlk + (threadIdx.x & 7) * 8;
  // one line to a thread, but for those past the 2^32 threads that a dimension of the grid cannot hold
  for (int64_t line = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); line < a.rows[z]; line += (int64_t)gridDim.x * 32)
    write8<kSplit>(a.d[z], line, at, load8<VEC>(a.src[z] + line * cols, at, cols));
}

// The columns of src [rows][cols] as lines of d, zeros from `rows` on up to a multiple of 64, and a second matrix's, where there
// is one, as lines of d2; S float, __bf16, or e4m3 with its scales (one matrix). Bound by memory (two of 8190 x 4100 bfloat16:
// 65 us, 4.1 TB/s).
template <int FMT, bool VEC, class S>
__global__ void __launch_bounds__(256) transpose_kernel(const S* __restrict__ src1, const S* __restrict__ src2,
                                                        const float* __restrict__ scale, int64_t rows, int64_t cols,
                                                        Lines d1, Lines d2) {
  const S* src = blockIdx.z ? src2 : src1;
  const Lines& d = blockIdx.z ? d2 : d1;
  __shared__ float blk[kBlk * kBlkPitch];
  const int64_t r0 = (int64_t)blockIdx.x * kBlk, c0 = (int64_t)blockIdx.y * kBlk;
  const int part = (threadIdx.x & 7) * 8;
  const int64_t blocks = (cols + kFp8Block - 1) / kFp8Block;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i;
    f32x8 v = {};
    if (r0 + r < rows) {
      v = load8<VEC>(src + (r0 + r) * cols, c0 + part, cols);
      if constexpr (sizeof(S) == 1) v *= scale[(r0 + r) * blocks + c0 / kFp8Block];
    }
    to_lds(blk, r, part, v);
  }
  __syncthreads();
  write_columns<FMT>(blk, d, c0, cols, r0);
}

// e4m3 with power-of-two scales as bfloat16, exactly; 16 lanes to a block of 128. Bound by memory (8192 x 4096: 21 us,
// 4.8 TB/s).
__global__ void __launch_bounds__(256) widen_rows_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                         int64_t rows, int64_t cols, __bf16* __restrict__ dst) {
  const int64_t vecs = (cols + kFp8Block - 1) / kFp8Block * 16, total = rows * vecs, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    const int64_t row = i / vecs, c = (i - row * vecs) * 8;
    store8<true>(dst + row * cols, c, cols, load8<true>(q + row * cols, c, cols) * scale[i / 16]);
  }
}

struct GateArgs {
  const void *gh, *g, *u;
  const float *gs, *us;
  int64_t m, f;
  int act, by_rows, by_cols;
  Lines g_rows, u_rows;  // m lines each: dg and du side by side
  Lines g_cols, u_cols;  // f lines each: one below the other
};
// dg and du of a 64 x 64 block of (row, column of f), laid out by rows and by columns. Bound by memory: from gh, g and u each
// once to each layout once. In bfloat16 dg and du are rounded to it, once, as what a matrix instruction of that type takes: the
// gradients then are 2.3e-3 of their size off, 1.7e-3 of it by their own rounding. 8192 x 8192 bfloat16 from 8-bit g and u, by
// rows: 136 us, 4 TB/s; 2049 x 2730 float32, both layouts: 31 us, 4 TB/s, the rows being no multiple of 16 bytes.
template <int FMT, bool VEC, class T, bool FP8>
__global__ void __launch_bounds__(256) glu_gate_kernel(GateArgs a) {
  __shared__ float dg[kBlk * kBlkPitch], du[kBlk * kBlkPitch];
  using Held = std::conditional_t<FP8, uint8_t, T>;
  const int64_t r0 = (int64_t)blockIdx.x * kBlk, c0 = (int64_t)blockIdx.y * kBlk;
  const int part = (threadIdx.x & 7) * 8;
  const int64_t blocks = (a.f + kFp8Block - 1) / kFp8Block;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i;
    f32x8 vg = {}, vu = {};
    if (r0 + r < a.m) {
      const int64_t row = (r0 + r) * a.f;
      const f32x8 gh = load8<VEC>((const T*)a.gh + row, c0 + part, a.f);
      f32x8 g = load8<VEC>((const Held*)a.g + row, c0 + part, a.f);
      f32x8 u = load8<VEC>((const Held*)a.u + row, c0 + part, a.f);
      if constexpr (FP8) {
        const int64_t b = (r0 + r) * blocks + c0 / kFp8Block;
        g *= a.gs[b];
        u *= a.us[b];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const ActAndGrad ag = glu_act_grad(g[e], a.act);
        vg[e] = gh[e] * u[e] * ag.grad;
        vu[e] = gh[e] * ag.act;
      }
      if (!VEC) {  // past the row's end: zeros, whatever the block's scale
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + part + e >= a.f) vg[e] = vu[e] = 0.f;
      }
      if (VEC && c0 + part >= a.f) vg = vu = f32x8{};
      if (a.by_rows) {
        write8<FMT>(a.g_rows, r0 + r, c0 + part, vg);
        write8<FMT>(a.u_rows, r0 + r, c0 + part, vu);
      }
    }
    if (a.by_cols) {
      to_lds(dg, r, part, vg);
      to_lds(du, r, part, vu);
    }
  }
  if (!a.by_cols) return;
  __syncthreads();
  write_columns<FMT>(dg, a.g_cols, c0, a.f, r0);
  write_columns<FMT>(du, a.u_cols, c0, a.f, r0);
}

// ---- tiles whose steps are shared ---------------------------------------------------------------------------------------

// The sum of the shares of eight columns of a row of shared tile j, in the shares' order; four loads in flight. Mostly the time
// of a launch (16 x 4096 x 8192 gated: 4.1 us; 2049 x 1000 float32 from 253 shares: 7.7).
__device__ __forceinline__ f32x8 join8(const GemmArgs& a, int bm, int j, int row, int col) {
  const int64_t from = (int64_t)j * a.steps;
  const int w0 = (int)(from / a.share), w1 = (int)((from + a.steps - 1) / a.share);
  f32x8 sum = {};
  // the first share that begins in an earlier tile holds this one's sum second
  auto at = [&](int w) {
    const int second = (int64_t)w * a.share < from;
    return load8<true>(a.parts + (((int64_t)w * 2 + second) * bm + row) * 256, col, 256);
  };
  int w = w0;
  for (; w + 3 <= w1; w += 4) {
    const f32x8 v0 = at(w), v1 = at(w + 1), v2 = at(w + 2), v3 = at(w + 3);
    sum += v0;
    sum += v1;
    sum += v2;
    sum += v3;
  }
  for (; w <= w1; ++w) sum += at(w);
  return sum;
}

// Shared tiles' results: eight rows of a tile to a workgroup, eight columns to a thread. Rows from `split` on go to out2.
template <bool VEC>
__global__ void __launch_bounds__(256) ffn_join_kernel(GemmArgs a, int bm) {
  const int per = bm / 8, j = blockIdx.x / per, row = blockIdx.x % per * 8 + (threadIdx.x >> 5);
  const TileId id = tile_at(a.whole + j, a.gx, a.gy);
  const int64_t m = (int64_t)id.y * bm + row, c = id.x * 256 + (threadIdx.x & 31) * 8;
  const int64_t to = m < a.split ? m : m - a.split;
  if (m >= a.m || to >= a.limit || c >= a.n) return;
  const f32x8 v = join8(a, bm, j, row, (threadIdx.x & 31) * 8);
  void* out = m < a.split ? a.out : a.out2;
  const int64_t at = to * a.n;
  if (a.out_kind == kOutBf16) store8<VEC>((__bf16*)out + at, c, a.n, v);
  else store8<VEC>((float*)out + at, c, a.n, v);
}

// The gated form's epilogue over them: sixteen rows to a workgroup, 16 lanes to a row's block of 128.
template <bool VEC>
__global__ void __launch_bounds__(256) glu_join_kernel(GemmArgs a, int bm) {
  const int per = bm / 16, j = blockIdx.x / per, row = blockIdx.x % per * 16 + (threadIdx.x >> 4);
  const TileId id = tile_at(a.whole + j, a.gx, a.gy);
  const int64_t m = (int64_t)id.y * bm + row, c = id.x * 128 + (threadIdx.x & 15) * 8;
  if (m >= a.m) return;  // all sixteen lanes of a row
  const f32x8 g = join8(a, bm, j, row, (threadIdx.x & 15) * 8), u = join8(a, bm, j, row, 128 + (threadIdx.x & 15) * 8);
  f32x8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = glu_act(g[e], a.act) * u[e];
  const int64_t at = m * a.n, block = m * ((a.n + kFp8Block - 1) / kFp8Block) + id.x;
  auto in_8 = [&](f32x8 v, void* q, float* scale) {
    const float s = block_scale(row16_max(abs_bits8(v)));
    store_fp8x8<VEC>((uint8_t*)q + at, c, a.n, pack_fp8x8(v, 1.f / s));
    if ((threadIdx.x & 15) == 0) scale[block] = s;
  };
  auto in_type = [&](f32x8 v, void* p) {
    if (a.out_kind == kOutBf16) store8<VEC>((__bf16*)p + at, c, a.n, v);
    else store8<VEC>((float*)p + at, c, a.n, v);
  };
  if (a.out_kind == kOutFp8) in_8(h, a.out, a.out_scale);
  else in_type(h, a.out);
  if (a.keep == kKeepFp8) {
    in_8(g, a.keep_g, a.keep_gs);
    in_8(u, a.keep_u, a.keep_us);
  } else if (a.keep == kKeepFull) {
    in_type(g, a.keep_g);
    in_type(u, a.keep_u);
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------

// The launch of a product of m rows by n (of each weight, if gated) with rows of row_bytes. As many tiles as fill all CUs
// evenly are a workgroup's each; those left over, too few for a round of their own, can be shared, every workgroup taking
// the same number of their steps, and joined by a second launch. Every choice of rows to a tile and of a share is priced, in
// microseconds, and the cheapest taken: rounds of workgroups over the 256 CUs (two at a time to a CU whose LDS holds the
// stages of two: tiles of 16 rows, and of 64 without scales), each its steps and what a tile costs before its first and after
// its last, but no less than the operands' bytes at 5.5 TB/s; sharing adds the second launch and the shares' sums to memory
// and back at 4 TB/s. Steps, and the rest of a tile, in us, measured with all CUs busy (16384 x 4096 x 4096 and x 8192, the
// gated form of kF32 at 5120 x 4096 x 1024 and x 2048; 16 rows at 64 x 4096 x 4096; 64 rows with scales beside 96 in one round of
// 256 workgroups, where both take as long), [mode][rows of a tile]:
constexpr float kStepUs[][kHeights] = {
    // 16    64    96    128    160    192    224   256
    {1.65f, 3.55f, 2.8f, 3.72f, 4.55f, 5.45f, 6.35f, 7.15f},   // kF32
    {1.2f, 1.0f, 0.62f, 0.76f, 0.88f, 1.1f, 1.25f, 1.4f},      // kBf16
    {1.95f, 1.35f, 1.42f, 1.68f, 2.02f, 2.46f, 2.98f, 3.34f},   // kFp8x
    {1.6f, 0.9f, 0.86f, 1.02f, 1.2f, 1.32f, 1.55f, 1.78f},     // kFp8
    {1.1f, 1.25f, 1.16f, 1.4f, 1.68f, 1.95f, 2.3f, 2.7f},      // kSplit
};
constexpr float kJoinUs = 4.f;
constexpr int kCus = 256, kCuLds = 160 * 1024;
template <int MODE, int V>
constexpr int resident_of() {
  return 2 * GemmTile<MODE, kBm[V], gemm_stages<MODE, kBm[V]>()>::LDS <= kCuLds ? 2 : 1;
}
template <int V = 0>
static int resident(int mode, int v) {
  if constexpr (V + 1 < kHeights)
    if (v != V) return resident<V + 1>(mode, v);
  constexpr int of[] = {resident_of<kF32, V>(), resident_of<kBf16, V>(), resident_of<kFp8x, V>(), resident_of<kFp8, V>(),
                        resident_of<kSplit, V>()};
  return of[mode];
}
static float tile_us(int mode, int v) {  // 64 rows: of two workgroups, or of one
  constexpr float us[kHeights] = {1.5f, 8.f, 5.f, 6.5f, 8.f, 8.5f, 10.f, 11.f};
  return kBm[v] == 64 && resident(mode, v) == 1 ? 5.f : us[v];
}
struct GemmPlan {
  int bm, gx, gy, steps, whole, sharers, share;
  float us;
  size_t parts_bytes;
};
// Which operands lie across the reduction (see ffn_gemm_kernel). Such tiles of fewer than 256 rows take a tenth longer.
enum Across { kAlong, kAcrossW, kAcrossBoth };
static GemmPlan plan_gemm(int mode, bool glu, int64_t m, int64_t n, int64_t row_bytes, Across across = kAlong) {
  const int64_t gx = cdiv(n, glu ? 128 : 256), steps = std::max<int64_t>(cdiv(row_bytes & ~15, 128), 1);
  const float bytes_us = (float)(m + n * (glu ? 2 : 1)) * (float)row_bytes / 5.5e6f;
  GemmPlan best{};
  best.us = 1e30f;
  for (int v = 0; v < kHeights; ++v) {
    if (v > 0 && m <= kBm[v - 1] && best.bm) break;
    if (across == kAcrossBoth && kBm[v] != 128 && kBm[v] != 256) continue;
    const float full = kStepUs[mode][v] * (across != kAlong && kBm[v] < 256 ? 1.1f : 1.f);
    const bool two = resident(mode, v) == 2;
    const float tile = tile_us(mode, v);
    const int64_t gy = cdiv(m, kBm[v]), tiles = gx * gy, at_once = two ? 2 * kCus : kCus, left = tiles % at_once;
    // a workgroup alone on its CU takes about half the step that two take, but no less than a load's way, 0.9
    auto step = [&](int64_t groups) {
      return two && groups <= kCus ? std::max(0.9f, 0.6f * full) : full;
    };
    const float rounds_us = (float)(tiles / at_once) * (steps * full + tile);
    auto consider = [&](float us, int64_t whole, int64_t sharers, int64_t share) {
      us = std::max(us, bytes_us);
      if (sharers) {  // a share begins a tile, and each tile's first and last shares may belong to two
        const float sums = (float)(sharers + tiles - whole) * (float)std::min<int64_t>(m, kBm[v]) * 256 * 4;
        us += kJoinUs + 2 * sums / 4e6f;
      }
      if (us < best.us)
        best = {kBm[v], (int)gx, (int)gy, (int)steps, (int)whole, (int)sharers, (int)share, us,
                (size_t)sharers * 2 * kBm[v] * 256 * sizeof(float)};
    };
    consider(rounds_us + (left ? steps * step(left) + tile : 0.f), tiles, 0, 0);
    if (!left || steps < 4) continue;
    for (int64_t k = 1; k <= 32; ++k) {  // a k-th of a tile's steps each, or all CUs' even share
      const int64_t share = k == 1 ? std::max<int64_t>(cdiv(left * steps, at_once), 2) : cdiv(steps, k);
      const int64_t sharers = cdiv(left * steps, share);
      if (share < 2 || share >= steps || sharers > at_once) continue;
      const float begins = steps % share ? 1.5f : 1.f;  // some shares cover the end of one tile and the start of the next
      consider(rounds_us + share * step(sharers) + begins * tile, tiles - left, sharers, share);
    }
  }
  return best;
}
static int run_gemm(int mode, bool glu, const GemmPlan& p, GemmArgs a, void* parts, hipStream_t stream,
                    Across across = kAlong) {
  a.steps = p.steps, a.gx = p.gx, a.gy = p.gy, a.whole = p.whole, a.sharers = p.sharers, a.share = p.share;
  a.parts = (float*)parts;
  int e = across == kAcrossW ? ffn_gemm_bf16_w(a, p.bm, stream)
          : across == kAcrossBoth ? ffn_gemm_bf16_xw(a, p.bm, stream)
          : mode == kF32 ? ffn_gemm_f32(a, p.bm, stream)
          : mode == kSplit ? ffn_gemm_split(a, glu, p.bm, stream)
          : mode == kBf16 ? ffn_gemm_bf16(a, glu, p.bm, stream)
          : mode == kFp8 ? ffn_gemm_fp8(a, p.bm, stream) : ffn_gemm_fp8x(a, glu, p.bm, stream);
  if (e || !p.sharers) return e;
  const bool vec = a.n % 8 == 0;
  const int shared = p.gx * p.gy - p.whole;
  auto go = [&](auto kernel, int rows) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(shared * (p.bm / rows))), dim3(256), 0, stream, a, p.bm);
  };
  if (glu) {
    vec ? go(glu_join_kernel<true>, 16) : go(glu_join_kernel<false>, 16);
    return launch_check("glu_join_kernel");
  }
  vec ? go(ffn_join_kernel<true>, 8) : go(ffn_join_kernel<false>, 8);
  return launch_check("ffn_join_kernel");
}

// A workspace handed out in 256-byte steps; `base` null to count only.
struct Space {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    if (!bytes) return nullptr;
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) & ~(size_t)255;
    return p;
  }
};

static int64_t up(int64_t v, int64_t to) { return cdiv(v, to) * to; }
static int elem_bytes(int mode) { return mode == kF32 || mode == kSplit ? 4 : mode == kBf16 ? 2 : 1; }

// `lines` of n elements (a multiple of 64) in kBf16 or kSplit
static Lines take_lines(Space& sp, int fmt, int64_t lines, int64_t n) {
  Lines d;
  d.pitch = n * elem_bytes(fmt);
  d.p = (char*)sp.take((size_t)(lines * d.pitch));
  if (fmt == kSplit) d.scale = (float*)sp.take((size_t)(n / 32 * lines) * sizeof(float)), d.scale_lines = lines;
  return d;
}
// the same from element `at` (a multiple of 64) and line `line` on
static Lines from(Lines d, int fmt, int64_t line, int64_t at) {
  d.p += line * d.pitch + at * elem_bytes(fmt);
  if (d.scale) d.scale += at / 32 * d.scale_lines + line;
  return d;
}

// An operand's rows as the tiles read them: in place where every row starts on 4 bytes (any float32, an even number of
// bfloat16, a multiple of four e4m3), else copied; kSplit always copied.
static Lines place_rows(Space& sp, int mode, int64_t rows, int64_t cols) {
  if (mode == kSplit) return take_lines(sp, kSplit, rows, up(cols, kBlk));
  Lines d;
  d.pitch = cols * elem_bytes(mode);
  if (d.pitch % 4) {
    d.pitch = up(d.pitch, 16);
    d.p = (char*)sp.take((size_t)(rows * d.pitch));
  }
  return d;
}
static int lay_rows(const Lines& d, int mode, const void* src, int64_t rows, int64_t cols, hipStream_t stream) {
  if (!d.p) return OMT_OK;
  const int64_t pitch = d.pitch / elem_bytes(mode);
  const dim3 grid(grid1d(rows * d.pitch / 16, 256, 1 << 16));
  auto go = [&](auto zero) {
    using T = decltype(zero);
    hipLaunchKernelGGL(pad_rows_kernel<T>, grid, dim3(256), 0, stream, (const T*)src, rows, cols, pitch, (T*)d.p);
  };
  mode == kBf16 ? go(uint16_t(0)) : go(uint8_t(0));
  return launch_check("pad_rows_kernel");
}
// Lays out x [m][k] and the weights [n][k] (w_up may be null) and points a at them.
static int lay_operands(GemmArgs& a, int mode, const Lines& x, const Lines& w, const Lines& w_up, const void* px,
                        const void* pw, const void* pw_up, int64_t m, int64_t n, int64_t k, hipStream_t stream) {
  if (mode == kSplit) {
    const SplitArgs s{{(const float*)px, (const float*)pw, (const float*)pw_up}, {m, n, n}, {x, w, w_up}};
    const dim3 grid(grid1d(std::max(m, n), 32), (unsigned)cdiv(k, kBlk), pw_up ? 3 : 2);
    if (k % 8 == 0) hipLaunchKernelGGL(split_rows_kernel<true>, grid, dim3(256), 0, stream, s, k);
    else hipLaunchKernelGGL(split_rows_kernel<false>, grid, dim3(256), 0, stream, s, k);
    if (int e = launch_check("split_rows_kernel")) return e;
  } else {
    if (int e = lay_rows(x, mode, px, m, k, stream)) return e;
    if (int e = lay_rows(w, mode, pw, n, k, stream)) return e;
    if (pw_up)
      if (int e = lay_rows(w_up, mode, pw_up, n, k, stream)) return e;
  }
  a.x = x.p ? x.p : px, a.w = w.p ? w.p : pw, a.w_up = w_up.p ? w_up.p : pw_up;
  a.xpitch = x.pitch, a.wpitch = w.pitch, a.row_bytes = (int)x.pitch;
  a.m = (int)m, a.n = (int)n, a.split = a.limit = (int)m;
  if (mode == kSplit) {
    a.sx = x.scale, a.sw = w.scale, a.sw_up = w_up.scale;
    a.sx_row = a.sw_row = 1, a.sx_step = (int)x.scale_lines, a.sw_step = (int)w.scale_lines;
  }
  return OMT_OK;
}

static bool on16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}
// Offsets within a tile's rows are 32-bit: 256 rows of at most 4 MiB.
static int product_check(const char* fn, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 1 || k < 1)
    return fail(OMT_INVALID, "%s: %lld x %lld x %lld", fn, (long long)m, (long long)n, (long long)k);
  constexpr int64_t kMost = 1 << 20, kRows = 1 << 30;
  if (k > kMost || m > kRows || n > kMost)
    return fail(OMT_UNSUPPORTED, "%s: %lld x %lld x %lld", fn, (long long)m, (long long)n, (long long)k);
  return OMT_OK;
}
static int need_space(const char* fn, size_t need, const void* ws, size_t bytes) {
  if (need && (!ws || bytes < need)) return fail(OMT_INVALID, "%s: workspace of %zu bytes, %zu needed", fn, bytes, need);
  if (!on16({ws})) return fail(OMT_INVALID, "%s: the workspace is not on 16 bytes", fn);
  return OMT_OK;
}

// The 8-bit matrix instruction adds eight consecutive products at a time, each cut off (towards 0) below 2^-13 of the largest, by
// their factors' powers of two; from there on its sums are float32's. Over Gaussian values that is 1.3e-5 of a block's sum
// (bfloat16's instruction on the same values is 1e-8 off): little beside a bfloat16 result's 2^-8, unless large products cancel,
// when it is up to 7 2^-13 of the largest of each eight. It is a choice of speed (4096 x 4096 x 8192 131 us, widened 243),
// and too much for a float32 result, which widens: float32's sums of exact products.
static int fp8_mode(int out_dtype) { return out_dtype == OMT_DT_BF16 ? kFp8 : kFp8x; }
struct MatmulFp8 {
  int few, mode;
  Lines a, b;
  GemmPlan p{};
  void* parts = nullptr;
  MatmulFp8(Space& sp, int out_dtype, int64_t m, int64_t n, int64_t k)
      : few(few_rows(m, n, k)), mode(fp8_mode(out_dtype)), a(place_rows(sp, mode, m, k)), b(place_rows(sp, mode, n, k)) {
    if (few) return;
    p = plan_gemm(mode, false, m, n, a.pitch);
    parts = sp.take(p.parts_bytes);
  }
};
// float32: on fp32 MFMA as it is, or as halves on float16 MFMA, three products for one. Laying out the halves reads and
// writes the operands once, at 4 TB/s; it is taken where the products win that back.
static int glu_mode(int dtype, int64_t m, int64_t k, int64_t f) {
  if (dtype == OMT_DT_BF16) return kBf16;
  const float lay_us = 8.f * (float)(m + 2 * f) * (float)k / 4e6f + 3.f;
  return plan_gemm(kSplit, true, m, f, up(k, kBlk) * 4).us + lay_us < plan_gemm(kF32, true, m, f, k * 4).us ? kSplit : kF32;
}
struct GluFwd {
  GemmPlan p;
  Lines x, wg, wu;
  void* parts;
  GluFwd(Space& sp, int mode, int64_t m, int64_t k, int64_t f)
      : x(place_rows(sp, mode, m, k)), wg(place_rows(sp, mode, f, k)), wu(place_rows(sp, mode, f, k)) {
    p = plan_gemm(mode, true, m, f, x.pitch);
    parts = sp.take(p.parts_bytes);
  }
};
struct GluBwd {
  bool across;
  int64_t half, mp;  // elements: dg and du of a row padded to `half` each; columns of m padded to mp
  Lines gate_rows, gate_cols, w_cols, x_cols;
  void* x_rows = nullptr;  // across: x in bfloat16
  GemmPlan px, pw;
  void* parts;
  GluBwd(Space& sp, int mode, int64_t m, int64_t k, int64_t f)
      : across(mode == kBf16 && k % 8 == 0 && f % 8 == 0), half(up(f, kBlk)), mp(up(m, kBlk)),
        gate_rows(take_lines(sp, mode, m, 2 * half)) {
    if (across) {
      x_rows = sp.take((size_t)(m * k * 2));
      px = plan_gemm(mode, false, m, k, gate_rows.pitch, kAcrossW);
      pw = plan_gemm(mode, false, 2 * half, k, mp * 2, kAcrossBoth);
    } else {
      gate_cols = take_lines(sp, mode, 2 * f, mp);
      w_cols = take_lines(sp, mode, k, 2 * half);
      x_cols = take_lines(sp, mode, k, mp);
      px = plan_gemm(mode, false, m, k, gate_rows.pitch);
      pw = plan_gemm(mode, false, 2 * f, k, gate_cols.pitch);
    }
    parts = sp.take(std::max(px.parts_bytes, pw.parts_bytes));
  }
};

static int glu_check(const char* fn, int dtype, int64_t m, int64_t k, int64_t f, int act) {
  if (dtype != OMT_DT_F32 && dtype != OMT_DT_BF16) return fail(OMT_INVALID, "%s: dtype %d", fn, dtype);
  if (act != OMT_GLU_SILU && act != OMT_GLU_GELU && act != OMT_GLU_RELU) return fail(OMT_INVALID, "%s: act %d", fn, act);
  return product_check(fn, m, f, k);
}

static int bwd_mode(int dtype) { return dtype == OMT_DT_F32 ? kSplit : kBf16; }

// src2: null, or a second matrix, its lines d2
template <class S>
static int run_transpose(int mode, const S* src, const S* src2, const float* scale, int64_t rows, int64_t cols,
                         const Lines& d, const Lines& d2, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(rows, kBlk), (unsigned)cdiv(cols, kBlk), src2 ? 2 : 1);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, src, src2, scale, rows, cols, d, d2);
  };
  const bool vec = cols % 8 == 0 && on16({src, src2});
  if (mode == kSplit) vec ? go(transpose_kernel<kSplit, true, S>) : go(transpose_kernel<kSplit, false, S>);
  else vec ? go(transpose_kernel<kBf16, true, S>) : go(transpose_kernel<kBf16, false, S>);
  return launch_check("transpose_kernel");
}
// the product of operands laid out as lines: x's lines by w's
static int run_lines(int mode, const GemmPlan& p, GemmArgs a, const Lines& x, const Lines& w, int64_t m, int64_t n,
                     void* parts, hipStream_t stream) {
  a.x = x.p, a.w = w.p, a.xpitch = a.wpitch = x.pitch, a.row_bytes = (int)x.pitch;
  a.m = (int)m, a.n = (int)n;
  a.sx = x.scale, a.sw = w.scale, a.sx_row = a.sw_row = 1;
  a.sx_step = (int)x.scale_lines, a.sw_step = (int)w.scale_lines;
  return run_gemm(mode, false, p, a, parts, stream);
}

}  // namespace omt

using namespace omt;

OMT_EXPORT int omt_ffn_plan(int op, int dtype, int64_t m, int64_t k, int64_t n, int* mode, int* rows,
                            int* sharers) {
  const char* fn = "omt_ffn_plan";
  if (!mode || !rows || !sharers) return fail(OMT_INVALID, "%s: null pointer", fn);
  if (int e = glu_check(fn, dtype, m, k, n, OMT_GLU_SILU)) return e;
  if (m == 0) return fail(OMT_INVALID, "%s: no rows", fn);
  Space sp{nullptr};
  GemmPlan p;
  switch (op) {
    case OMT_FFN_MATMUL_FP8: {
      const MatmulFp8 l(sp, dtype, m, n, k);
      *mode = l.few ? 5 : l.mode, p = l.p;
      if (l.few) p.bm = l.few;
      break;
    }
    case OMT_FFN_GLU: *mode = glu_mode(dtype, m, k, n), p = GluFwd(sp, *mode, m, k, n).p; break;
    case OMT_FFN_GLU_FP8: *mode = kFp8x, p = GluFwd(sp, kFp8x, m, k, n).p; break;
    case OMT_FFN_GLU_GX: *mode = bwd_mode(dtype), p = GluBwd(sp, *mode, m, k, n).px; break;
    case OMT_FFN_GLU_GW: *mode = bwd_mode(dtype), p = GluBwd(sp, *mode, m, k, n).pw; break;
    default: return fail(OMT_INVALID, "%s: op %d", fn, op);
  }
  *rows = p.bm, *sharers = p.sharers;
  return OMT_OK;
}

OMT_EXPORT size_t omt_matmul_fp8_workspace(int64_t m, int64_t n, int64_t k, int out_dtype) {
  if (product_check("omt_matmul_fp8_workspace", m, n, k) || m == 0) return 0;
  Space sp{nullptr};
  MatmulFp8(sp, out_dtype, m, n, k);
  return sp.used;
}

OMT_EXPORT int omt_matmul_fp8(int64_t m, int64_t n, int64_t k, const void* a, const float* a_scale, const void* b,
                              const float* b_scale, int out_dtype, void* c, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const char* fn = "omt_matmul_fp8";
  if (out_dtype != OMT_DT_F32 && out_dtype != OMT_DT_BF16) return fail(OMT_INVALID, "%s: dtype %d", fn, out_dtype);
  if (int e = product_check(fn, m, n, k)) return e;
  if (m == 0) return OMT_OK;
  if (!a || !a_scale || !b || !b_scale || !c) return fail(OMT_INVALID, "%s: null pointer", fn);
  if (!on16({a, b, c})) return fail(OMT_INVALID, "%s: an operand is not on 16 bytes", fn);
  if (int e = need_space(fn, omt_matmul_fp8_workspace(m, n, k, out_dtype), workspace, workspace_bytes)) return e;
  Space sp{(char*)workspace};
  const MatmulFp8 l(sp, out_dtype, m, n, k);
  hipStream_t st = stream_of(stream);
  GemmArgs g{};
  if (int e = lay_operands(g, l.mode, l.a, l.b, {}, a, b, nullptr, m, n, k, st)) return e;
  g.sx = a_scale, g.sw = b_scale;
  g.sx_row = g.sw_row = (int)cdiv(k, kFp8Block), g.sx_step = g.sw_step = 1;
  g.out = c, g.out_kind = out_dtype == OMT_DT_BF16 ? kOutBf16 : kOutF32;
  if (l.few) return matmul_fp8_few({g.x, g.w, g.sx, g.sw, c, g.m, g.n, g.row_bytes, g.out_kind}, st);
  return run_gemm(l.mode, false, l.p, g, l.parts, st);
}

OMT_EXPORT size_t omt_glu_fwd_workspace(int dtype, int64_t m, int64_t k, int64_t f) {
  if (glu_check("omt_glu_fwd_workspace", dtype, m, k, f, OMT_GLU_SILU) || m == 0) return 0;
  Space sp{nullptr};
  GluFwd(sp, glu_mode(dtype, m, k, f), m, k, f);
  return sp.used;
}

OMT_EXPORT int omt_glu_fwd(int dtype, int64_t m, int64_t k, int64_t f, int act, int keep, const void* x,
                           const void* w_gate, const void* w_up, void* h, void* x_q, float* x_scale, void* g,
                           float* g_scale, void* u, float* u_scale, void* workspace, size_t workspace_bytes,
                           void* stream) {
  const char* fn = "omt_glu_fwd";
  if (int e = glu_check(fn, dtype, m, k, f, act)) return e;
  if (keep != OMT_KEEP_NONE && keep != OMT_KEEP_FP8 && keep != OMT_KEEP_FULL) return fail(OMT_INVALID, "%s: keep %d", fn, keep);
  if (m == 0) return OMT_OK;
  if (!x || !w_gate || !w_up || !h || (keep != OMT_KEEP_NONE && (!g || !u)) ||
      (keep == OMT_KEEP_FP8 && (!x_q || !x_scale || !g_scale || !u_scale)))
    return fail(OMT_INVALID, "%s: null pointer", fn);
  if (!on16({x, w_gate, w_up, h, g, u})) return fail(OMT_INVALID, "%s: an operand is not on 16 bytes", fn);
  if (int e = need_space(fn, omt_glu_fwd_workspace(dtype, m, k, f), workspace, workspace_bytes)) return e;
  const int mode = glu_mode(dtype, m, k, f);
  Space sp{(char*)workspace};
  const GluFwd l(sp, mode, m, k, f);
  hipStream_t st = stream_of(stream);
  if (keep == OMT_KEEP_FP8)
    if (int e = omt_quantize_fp8(dtype, m, k, x, 1, x_q, x_scale, stream)) return e;
  GemmArgs a{};
  if (int e = lay_operands(a, mode, l.x, l.wg, l.wu, x, w_gate, w_up, m, f, k, st)) return e;
  a.out = h, a.out_kind = dtype == OMT_DT_BF16 ? kOutBf16 : kOutF32, a.act = act;
  a.keep = keep == OMT_KEEP_FP8 ? kKeepFp8 : keep == OMT_KEEP_FULL ? kKeepFull : kKeepNone;
  a.keep_g = g, a.keep_u = u, a.keep_gs = g_scale, a.keep_us = u_scale;
  return run_gemm(mode, true, l.p, a, l.parts, st);
}

OMT_EXPORT size_t omt_glu_fp8_workspace(int64_t m, int64_t k, int64_t f) {
  if (product_check("omt_glu_fp8_workspace", m, f, k) || m == 0) return 0;
  Space sp{nullptr};
  GluFwd(sp, kFp8x, m, k, f);
  return sp.used;
}

OMT_EXPORT int omt_glu_fp8(int64_t m, int64_t k, int64_t f, int act, const void* x, const float* x_scale,
                           const void* w_gate, const float* gate_scale, const void* w_up, const float* up_scale,
                           void* h_q, float* h_scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omt_glu_fp8";
  if (int e = glu_check(fn, OMT_DT_F32, m, k, f, act)) return e;
  if (m == 0) return OMT_OK;
  if (!x || !x_scale || !w_gate || !gate_scale || !w_up || !up_scale || !h_q || !h_scale)
    return fail(OMT_INVALID, "%s: null pointer", fn);
  if (!on16({x, w_gate, w_up, h_q})) return fail(OMT_INVALID, "%s: an operand is not on 16 bytes", fn);
  if (int e = need_space(fn, omt_glu_fp8_workspace(m, k, f), workspace, workspace_bytes)) return e;
  Space sp{(char*)workspace};
  const GluFwd l(sp, kFp8x, m, k, f);
  hipStream_t st = stream_of(stream);
  GemmArgs a{};
  if (int e = lay_operands(a, kFp8x, l.x, l.wg, l.wu, x, w_gate, w_up, m, f, k, st)) return e;
  a.sx = x_scale, a.sw = gate_scale, a.sw_up = up_scale;
  a.sx_row = a.sw_row = (int)cdiv(k, kFp8Block), a.sx_step = a.sw_step = 1;
  a.out = h_q, a.out_scale = h_scale, a.out_kind = kOutFp8, a.act = act, a.keep = kKeepNone;
  return run_gemm(kFp8x, true, l.p, a, l.parts, st);
}

OMT_EXPORT size_t omt_glu_bwd_workspace(int dtype, int64_t m, int64_t k, int64_t f) {
  if (glu_check("omt_glu_bwd_workspace", dtype, m, k, f, OMT_GLU_SILU)) return 0;
  Space sp{nullptr};
  GluBwd(sp, bwd_mode(dtype), std::max<int64_t>(m, 1), k, f);
  return sp.used;
}

OMT_EXPORT int omt_glu_bwd(int dtype, int64_t m, int64_t k, int64_t f, int act, int keep, const void* gh, const void* x,
                           const float* x_scale, const void* g, const float* g_scale, const void* u,
                           const float* u_scale, const void* w_gate, const void* w_up, void* gx, void* gw_gate,
                           void* gw_up, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omt_glu_bwd";
  if (int e = glu_check(fn, dtype, m, k, f, act)) return e;
  if (keep != OMT_KEEP_FP8 && keep != OMT_KEEP_FULL) return fail(OMT_INVALID, "%s: keep %d", fn, keep);
  if (!gw_gate != !gw_up) return fail(OMT_INVALID, "%s: one of the weights' gradients alone", fn);
  const size_t e = dtype == OMT_DT_F32 ? 4 : 2;
  if (m == 0) {  // no row: no gradient
    if (!gw_gate) return OMT_OK;
    if (int err = omt_memset_zero(gw_gate, (size_t)(f * k) * e, stream)) return err;
    return omt_memset_zero(gw_up, (size_t)(f * k) * e, stream);
  }
  const bool fp8 = keep == OMT_KEEP_FP8;
  if (!gh || !x || !g || !u || !w_gate || !w_up || (fp8 && (!x_scale || !g_scale || !u_scale)))
    return fail(OMT_INVALID, "%s: null pointer", fn);
  if (!on16({x, w_gate, w_up, gx, gw_gate, gw_up})) return fail(OMT_INVALID, "%s: an operand is not on 16 bytes", fn);
  if (m > 1 << 20 || f > 1 << 18)
    return fail(OMT_UNSUPPORTED, "%s: %lld x %lld x %lld", fn, (long long)m, (long long)k, (long long)f);
  if (int err = need_space(fn, omt_glu_bwd_workspace(dtype, m, k, f), workspace, workspace_bytes)) return err;
  if (!gx && !gw_gate) return OMT_OK;
  const int mode = bwd_mode(dtype), out_kind = dtype == OMT_DT_F32 ? kOutF32 : kOutBf16;
  Space sp{(char*)workspace};
  const GluBwd l(sp, mode, m, k, f);
  hipStream_t st = stream_of(stream);

  const GateArgs ga{gh, g, u, g_scale, u_scale, m, f, act, gx || l.across, gw_gate && !l.across,
                    l.gate_rows, from(l.gate_rows, mode, 0, l.half), l.gate_cols,
                    l.across ? Lines{} : from(l.gate_cols, mode, f, 0)};
  const dim3 grid((unsigned)cdiv(m, kBlk), (unsigned)cdiv(f, kBlk));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, ga); };
  auto pick = [&](auto vec) {
    constexpr bool V = decltype(vec)::value;
    if (mode == kSplit) fp8 ? go(glu_gate_kernel<kSplit, V, float, true>) : go(glu_gate_kernel<kSplit, V, float, false>);
    else fp8 ? go(glu_gate_kernel<kBf16, V, __bf16, true>) : go(glu_gate_kernel<kBf16, V, __bf16, false>);
  };
  f % 8 == 0 && on16({gh, g, u}) ? pick(std::true_type{}) : pick(std::false_type{});
  if (int err = launch_check("glu_gate_kernel")) return err;

  auto transpose = [&](const void* src, const void* src2, int64_t rows, int64_t cols, const Lines& d, const Lines& d2) {
    return dtype == OMT_DT_F32
               ? run_transpose(mode, (const float*)src, (const float*)src2, nullptr, rows, cols, d, d2, st)
               : run_transpose(mode, (const __bf16*)src, (const __bf16*)src2, nullptr, rows, cols, d, d2, st);
  };
  if (l.across) {
    GemmArgs a{};
    a.x = l.gate_rows.p, a.xpitch = l.gate_rows.pitch, a.wpitch = k * 2, a.n = (int)k, a.out_kind = out_kind;
    if (gx) {  // [m][dg | du] by Wg, then Wu, across
      a.w = w_gate, a.w_up = w_up, a.t_rows = (int)f, a.up_step = (int)(l.half / 64);
      a.m = a.split = a.limit = (int)m, a.row_bytes = (int)a.xpitch, a.out = gx;
      if (int err = run_gemm(mode, false, l.px, a, l.parts, st, kAcrossW)) return err;
    }
    if (gw_gate) {  // dg and du, and x, across
      a.w = x;
      if (fp8) {
        const dim3 rows(grid1d(m * cdiv(k, kFp8Block) * 16, 256, 1 << 16));
        hipLaunchKernelGGL(widen_rows_kernel, rows, dim3(256), 0, st, (const uint8_t*)x, x_scale, m, k, (__bf16*)l.x_rows);
        if (int err = launch_check("widen_rows_kernel")) return err;
        a.w = l.x_rows;
      }
      a.w_up = nullptr, a.t_rows = (int)m, a.up_step = INT32_MAX;
      a.m = (int)(2 * l.half), a.split = (int)l.half, a.limit = (int)f, a.row_bytes = (int)(l.mp * 2);
      a.out = gw_gate, a.out2 = gw_up;
      if (int err = run_gemm(mode, false, l.pw, a, l.parts, st, kAcrossBoth)) return err;
    }
    return OMT_OK;
  }
  if (gx) {  // [m][dg | du] by [k][Wg^T | Wu^T]
    if (int err = transpose(w_gate, w_up, f, k, l.w_cols, from(l.w_cols, mode, 0, l.half))) return err;
    GemmArgs a{};
    a.out = gx, a.split = a.limit = (int)m, a.out_kind = out_kind;
    if (int err = run_lines(mode, l.px, a, l.gate_rows, l.w_cols, m, k, l.parts, st)) return err;
  }
  if (gw_gate) {  // [dg^T over du^T] by [k][x^T]
    if (int err = fp8 ? run_transpose(mode, (const uint8_t*)x, (const uint8_t*)nullptr, x_scale, m, k, l.x_cols, {}, st)
                      : transpose(x, nullptr, m, k, l.x_cols, {}))
      return err;
    GemmArgs a{};
    a.out = gw_gate, a.out2 = gw_up, a.split = a.limit = (int)f, a.out_kind = out_kind;
    if (int err = run_lines(mode, l.pw, a, l.gate_cols, l.x_cols, 2 * f, k, l.parts, st)) return err;
  }
  return OMT_OK;
}
