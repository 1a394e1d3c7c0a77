// Matrix products of the feed-forward operators: out[m][n] = sum over k of x[m][k] w[n][k], both operands with the
// reduction along their rows, in tiles of BM rows of x by 256 rows of w. The gated form takes 128 rows each of the gate's
// and the up projection's weight, so that a workgroup holds both projections of its outputs, and a block of 128 of them.
//
// Every mode reads its operands the same way, 128 bytes of each row to a step: 32 floats, 64 bfloat16, 128 e4m3.
// They go from memory to LDS without passing registers; within a row, 16-byte chunk c lies at c ^ (row & 7), so that
// the 16 lanes that read one chunk of 16 rows touch every bank. NS stages are in flight, one workgroup barrier a step.
// A lane's two chunks of a row (g and g + 4, g = lane / 16) feed the matrix cores in whatever order of k; the order is
// the same for both operands, and a sum does not mind.
//
// Tiles of 256 rows with all CUs busy, m x n x k (Gaussian values, short runs; long ones are up to a tenth slower, the clock
// giving way to power): bfloat16 8192 x 4096 x 8192 370 us, 1480 TFLOP/s; e4m3 227 us, 2420; halves 1470 us, 375 (1120 of
// the float16 products); e4m3 widened 1210 TFLOP/s (4096 x 4096 x 4096), float32 150. A step of 256 rows takes the LDS as
// long as the matrix cores (192 KB of reads and 64 KB of loads at 128 bytes a clock; 64 products of 16 clocks to each of a
// SIMD's two waves), so the wave's tile is as large as its registers hold, 128 x 64, and the matrix cores are busy for 61% of
// the clocks (gated, bfloat16, 8192 x 4096 x 8192). The scaled modes add vector instructions, which the matrix cores' work
// hides in part: 46% in e4m3 (4096 x 4096 x 8192), 44% in halves (gated, 4096 x 1024 x 4096). A wave tile of 128 x 128 (four
// waves, accumulators in the second half of the register file) reads a third less and took as long (355 to 370 us for 361 to
// 373): a lone wave's other instructions are in its products' way.
#pragma once

#include "block_fp8.h"
#include "lds_dma.h"
#include "tile_map.h"

namespace omt {

// kF32: v_mfma_f32_16x16x4_f32 on the floats themselves. kBf16: v_mfma_f32_16x16x32_bf16. kFp8x: e4m3 values taken to
// bfloat16 (exact) for the same instruction; each step is one block of 128, whose sum is multiplied by the two scales.
// kSplit: floats as two float16 halves of a scaled group of 32 (a step: 32 high halves, 32 low ones; scales by step and
// row), three v_mfma_f32_16x16x32_f16: high by high, high by low, low by high. The product left out is 2^-22 of the
// whole. kFp8: the e4m3 values on v_mfma_f32_16x16x128_f8f6f4.
enum GemmMode { kF32, kBf16, kFp8x, kFp8, kSplit };
enum GluKeep { kKeepNone, kKeepFp8, kKeepFull };
enum OutKind { kOutF32, kOutBf16, kOutFp8 };

// p, the same in every lane, in scalar registers
template <class T>
__device__ __forceinline__ const T* uniform(const T* p) {
  const uint64_t b = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);  // an int: no sign into the upper half
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
  return (const T*)((uint64_t)hi << 32 | lo);
}

// Tiles in groups of eight rows, the rows fastest within a group.
__host__ __device__ __forceinline__ TileId tile_at(int t, int gx, int gy) {
  const int group = t / (8 * gx), y0 = group * 8, rows = gy - y0 < 8 ? gy - y0 : 8, r = t - group * 8 * gx;
  return {r / rows, y0 + r % rows, 0};
}
// The p-th of n workgroups' place among them, so that each XCD (p mod 8) has a run of places.
__device__ __forceinline__ int xcd_place(int p, int n) {
  const int per = n / kXCDs;
  return p < per * kXCDs ? (p % kXCDs) * per + p / kXCDs : p;
}

struct GemmArgs {
  const void *x, *w, *w_up;           // rows of xpitch / wpitch bytes, a multiple of 4; w_up: the gated form's
  const float *sx, *sw, *sw_up;       // 8 bits: x's scales [m][blocks], w's [ceil(n / 128)][blocks]
  int sx_row, sw_row, sx_step, sw_step;  // floats from a row's scale to the next row's, and to its next step's
  int64_t xpitch, wpitch;
  int m, n, row_bytes, steps;         // n: rows of w (and of w_up); row_bytes: the reduction's length
  int gx, gy;                         // tiles, in the order of tile_at
  // The first `whole` of them are a workgroup's each. The others' steps, one tile's after the other's, are cut into shares
  // of `share` steps for `sharers` workgroups, at most two tiles' to a share, whose sums go to parts and are joined after.
  int whole, sharers, share;
  float* parts;                       // [sharers][2][rows of a tile][256]
  void *out, *out2;                   // rows of n; rows of x from split on go to out2
  int split, limit, out_kind;         // rows of out, and of out2, from limit on are no one's
  int t_rows, up_step;                // operands with the reduction along their columns: rows of each, see below
  // the gated form: out gets act(g) * u, in 8 bits with scales out_scale; keep: what the backward pass needs
  int act, keep;
  float* out_scale;
  void *keep_g, *keep_u;
  float *keep_gs, *keep_us;
};

// exp(-g) by the exponential instruction, a few ulp and |g| 2^-24 of it off, and reciprocals to 1 ulp: the sums that they
// meet are no better in float32.
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.442695040888963f * g));
}
// The normal distribution's Phi(g) and, where asked for, its density. The tail Phi(-|g|) is exp(-z^2) times half of
// erfcx(z), z = |g| / sqrt 2, which over t = 1 / (1 + z / 2) is t times a polynomial in t: of degree 8, fitted for the smallest
// relative error (4.4e-8; in float32 with the exponential instruction 4e-7 of g Phi(g) over -1, 3e-6 at -8). The gated form by
// 777 x 1928 x 2504 in 8 bits takes 37.7 us with it, 39.9 with erfcf.
__device__ __forceinline__ float normal_cdf(float g, float* density) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35355339059327373f, fabsf(g), 1.f));
  const float e = __builtin_amdgcn_exp2f(-0.7213475204444817f * g * g);
  float q = -0.0296387915f;
  q = fmaf(q, t, 0.142796934f);
  q = fmaf(q, t, -0.244655848f);
  q = fmaf(q, t, 0.140242666f);
  q = fmaf(q, t, -0.014146396f);
  q = fmaf(q, t, 0.10169632f);
  q = fmaf(q, t, 0.121462673f);
  q = fmaf(q, t, 0.141199917f);
  q = fmaf(q, t, 0.141042516f);
  const float tail = t * q * e;
  if (density) *density = 0.3989422804014327f * e;
  return g < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float glu_act(float g, int act) {
  if (act == OMT_GLU_SILU) return g * sigmoid(g);
  if (act == OMT_GLU_GELU) return g * normal_cdf(g, nullptr);
  return g < 0.f ? 0.f : g;  // NaN stays
}
struct ActAndGrad {
  float act, grad;
};
__device__ __forceinline__ ActAndGrad glu_act_grad(float g, int act) {
  if (act == OMT_GLU_SILU) {
    const float p = sigmoid(g);
    return {g * p, p * (1.f + g * (1.f - p))};
  }
  if (act == OMT_GLU_GELU) {
    float density;
    const float phi = normal_cdf(g, &density);
    return {g * phi, phi + g * density};
  }
  return {g < 0.f ? 0.f : g, g > 0.f ? 1.f : 0.f};
}

// eight consecutive columns c.. of a row of `cols`; vec: see store8
__device__ __forceinline__ void store8_any(void* p, int64_t row, int c, int cols, bool vec, int kind, f32x8 v) {
  if (kind == kOutBf16) {
    __bf16* q = (__bf16*)p + row * cols;
    vec ? store8<true>(q, c, cols, v) : store8<false>(q, c, cols, v);
  } else {
    float* q = (float*)p + row * cols;
    vec ? store8<true>(q, c, cols, v) : store8<false>(q, c, cols, v);
  }
}
__device__ __forceinline__ void store8_fp8(void* p, int64_t row, int c, int cols, bool vec, f32x8 v, float inv) {
  uint8_t* q = (uint8_t*)p + row * cols;
  const uint2 w = pack_fp8x8(v, inv);
  vec ? store_fp8x8<true>(q, c, cols, w) : store_fp8x8<false>(q, c, cols, w);
}
// four; vec: rows of a multiple of four columns
template <class T>
__device__ __forceinline__ void store4(T* p, int c, int cols, bool vec, f32x4 v) {
  if (vec) {
    if (c < cols) {
      if constexpr (sizeof(T) == 4) *(f32x4*)(p + c) = v;
      else *(bf16x4*)(p + c) = __builtin_convertvector(v, bf16x4);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < cols) p[c + e] = (T)v[e];
  }
}
__device__ __forceinline__ void store4_any(void* p, int64_t row, int c, int cols, bool vec, int kind, f32x4 v) {
  if (kind == kOutBf16) store4((__bf16*)p + row * cols, c, cols, vec, v);
  else store4((float*)p + row * cols, c, cols, vec, v);
}
__device__ __forceinline__ f32x8 beside(f32x4 a, f32x4 b) { return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
// eight e4m3 values as bfloat16
__device__ __forceinline__ omt_u32x4 widen_fp8(uint32_t lo, uint32_t hi) {
  return omt_u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
}
__device__ __forceinline__ i32x8 join8(omt_u32x4 a, omt_u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

template <int MODE, int BM, int NS>
struct GemmTile {
  static constexpr int WM = BM >= 96 ? 2 : 1;        // waves along the rows of x; 4 along the rows of w
  static constexpr int NW = WM * 4, THREADS = NW * 64;
  static constexpr int TI = BM / WM / 16, TJ = 4;      // a wave's 16 x 16 tiles
  static constexpr int XI = BM / 8, DI = XI + 32;      // loads of 8 rows a step
  static constexpr int DW = (DI + NW - 1) / NW;        // ... by each wave (some repeated, so that all waves' counts are one)
  static constexpr bool SCALED = MODE != kF32 && MODE != kBf16;
  static constexpr int SROWS = (BM + 63) / 64 * 64;
  static constexpr int SI = SROWS / 64 + 4;            // loads of 64 scales a step
  static constexpr int SW = SCALED ? (SI + NW - 1) / NW : 0;
  static constexpr int LOADS = DW + SW;
  static constexpr int STAGE = (BM + 256) * 128 + (SCALED ? (SROWS + 256) * 4 : 0);
  static constexpr int LDS = NS * STAGE;
};

// XT, WT (kBf16): x, or w, lies with the reduction along its columns, [reduction][m] or [reduction][n], a multiple of 8
// columns and rows on 16 bytes. Its stages are 64 rows of the reduction; the LDS reads that transpose 4 x 16 elements give
// the matrix instructions what they take. A row's 16-byte chunk c lies at c ^ 2 (row & 3): the four rows of such a read
// would share their banks. w may be two matrices one after the other along the reduction, w and from step up_step w_up.
template <int MODE, bool GLU, int BM, int NS, bool XT, bool WT>
__global__ void __launch_bounds__((GemmTile<MODE, BM, NS>::THREADS), (GemmTile<MODE, BM, NS>::NW / 4))
ffn_gemm_kernel(GemmArgs a) {
  using Tl = GemmTile<MODE, BM, NS>;
  static_assert(!(XT || WT) || (MODE == kBf16 && !GLU), "transposed operands: bfloat16, plain");
  static_assert(!XT || BM == 128 || BM == 256, "a row of x's stage: 16 or 32 chunks");
  constexpr int TI = Tl::TI, TJ = Tl::TJ, NT = GLU ? 128 : 256;
  static_assert(Tl::LDS >= 2 * 4 * BM * 4, "the epilogue's maxima lie where the stages were");
  __shared__ __attribute__((aligned(128))) unsigned char lds[Tl::LDS];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;

  // this workgroup's tile, or its share of the steps of one or two
  int tile, s0 = 0, todo = a.steps;
  float* part = nullptr;
  if ((int)blockIdx.x < a.whole) {
    tile = xcd_place(blockIdx.x, a.whole);
  } else {
    const int w = xcd_place(blockIdx.x - a.whole, a.sharers);
    const int64_t begin = (int64_t)w * a.share, all = (int64_t)(a.gx * a.gy - a.whole) * a.steps;
    tile = a.whole + (int)(begin / a.steps);
    s0 = (int)(begin % a.steps);
    todo = (int)(all - begin < a.share ? all - begin : a.share);
    part = a.parts + (int64_t)w * 2 * BM * 256;
  }
  while (todo > 0) {
  // Opaque, so that what follows from it is computed where it is used: taken out of this loop, which mostly runs once, the
  // addresses of the epilogue would sit in 50 registers through the products.
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int r16 = lane & 15, g = lane >> 4;
  const TileId id = tile_at(tile, a.gx, a.gy);
  const int m0 = id.y * BM, n0 = id.x * NT;
  const int s1 = min(a.steps, s0 + todo);

  // where each of this wave's loads reads: a base that advances 128 bytes a step, and the lane's offset from it. Rows
  // past the operand's last read as 0 (an offset out of the range that the load checks).
  const uint32_t chunk16 = ((lane & 7) ^ (lane >> 3)) * 16;
  const unsigned char* dbase[Tl::DW];
  uint32_t doff[Tl::DW], ddst[Tl::DW];
  // The row of w that lies in a row of its stage, both from the tile's first: such that a lane's results of two neighbouring
  // tiles, four rows of each, are eight columns in a row. 4 lanes then store 64 bytes of a bfloat16 row at a time instead of 32
  // (gated, 8192 x 4096 x 8192 bfloat16, 8-bit checkpoints: 884 -> 853 us). float32 results are 64 bytes as they are.
  constexpr int kRun = WT || (!GLU && (MODE == kSplit || MODE == kFp8x)) ? 4 : 8;
  auto w_row = [](int r) {
    return (r & -4 * kRun) + (r >> 2 & 3) * kRun + (r >> 4) % (kRun / 4) * 4 + (r & 3);
  };
#pragma unroll
  for (int t = 0; t < Tl::DW; ++t) {
    const int slot = min(wave + Tl::NW * t, Tl::DI - 1);
    ddst[t] = slot * 1024;
    if ((XT && slot < Tl::XI) || (WT && slot >= Tl::XI)) {
      const bool of_x = slot < Tl::XI;
      const int row_size = of_x ? BM * 2 : 512, at = (of_x ? slot : slot - Tl::XI) * 1024 + lane * 16;
      const int k = at / row_size, c = (at % row_size / 16) ^ ((k & 3) * 2);
      dbase[t] = of_x ? (const unsigned char*)a.x + m0 * 2 : (const unsigned char*)a.w + n0 * 2;
      doff[t] = c * 8 < (of_x ? a.m - m0 : a.n - n0) ? (uint32_t)k * (uint32_t)(of_x ? a.xpitch : a.wpitch) + c * 16 : kOOB;
    } else if (slot < Tl::XI) {
      const int r = slot * 8 + (lane >> 3);
      dbase[t] = (const unsigned char*)a.x + m0 * a.xpitch;
      doff[t] = m0 + r < a.m ? (uint32_t)r * (uint32_t)a.xpitch + chunk16 : kOOB;
    } else {
      const int r8 = (slot - Tl::XI) * 8, r = w_row((GLU ? r8 & 127 : r8) + (lane >> 3));
      dbase[t] = (const unsigned char*)(GLU && r8 >= 128 ? a.w_up : a.w) + n0 * a.wpitch;
      doff[t] = n0 + r < a.n ? (uint32_t)r * (uint32_t)a.wpitch + chunk16 : kOOB;
    }
  }
  const float* sbase[Tl::SW + 1];
  uint32_t soff[Tl::SW + 1], sdst[Tl::SW + 1];
  if constexpr (Tl::SCALED) {
#pragma unroll
    for (int t = 0; t < Tl::SW; ++t) {
      const int slot = min(wave + Tl::NW * t, Tl::SI - 1);
      sdst[t] = (BM + 256) * 128 + slot * 256;
      if (slot < Tl::SROWS / 64) {
        const int r = slot * 64 + lane;
        sbase[t] = a.sx + (int64_t)m0 * a.sx_row;
        soff[t] = m0 + r < a.m && r < BM ? (uint32_t)(r * a.sx_row) * 4 : kOOB;
      } else {
        const int r64 = (slot - Tl::SROWS / 64) * 64, r = w_row((GLU ? r64 & 127 : r64) + lane);
        constexpr int kShift = MODE == kSplit ? 0 : 7;
        sbase[t] = (GLU && r64 >= 128 ? a.sw_up : a.sw) + (int64_t)(n0 >> kShift) * a.sw_row;
        soff[t] = n0 + r < a.n ? (uint32_t)((r >> kShift) * a.sw_row) * 4 : kOOB;
      }
    }
  }
  auto slot_of_x = [&](int t) { return wave + Tl::NW * t < Tl::SROWS / 64; };
  const int whole = a.row_bytes & ~15;  // what the 16-byte loads take of a row
  const uint32_t lds0 = lds_addr((const float*)lds);
  // Step s into stage `buf`. Past the share's last step every lane's offset is out of range: the loads count, and read
  // nothing.
  auto issue = [&](int buf, int s) {
    const uint32_t at = lds0 + buf * Tl::STAGE;
    const uint32_t left = s < s1 && s * 128 < whole ? (uint32_t)(whole - s * 128) : 0u;
    const bool in = chunk16 < left;
#pragma unroll
    for (int t = 0; t < Tl::DW; ++t) {
      if constexpr (XT || WT) {
        const int slot = min(wave + Tl::NW * t, Tl::DI - 1);
        const bool of_x = slot < Tl::XI;
        if (of_x ? XT : WT) {
          const int row_size = of_x ? BM * 2 : 512, k = ((of_x ? slot : slot - Tl::XI) * 1024 + lane * 16) / row_size;
          const bool second = !of_x && s >= a.up_step;
          const int row = (second ? s - a.up_step : s) * 64;
          const unsigned char* p = second ? (const unsigned char*)a.w_up + n0 * 2 : dbase[t];
          const bool there = s < s1 && row + k < a.t_rows;
          lds_load_b128(rsrc_words(uniform(p + row * (of_x ? a.xpitch : a.wpitch)), 0x7fffffffu),
                        __builtin_amdgcn_readfirstlane(at + ddst[t]), there ? doff[t] : kOOB);
          continue;
        }
      }
      lds_load_b128(rsrc_words(uniform(dbase[t] + (int64_t)s * 128), 0x7fffffffu),
                    __builtin_amdgcn_readfirstlane(at + ddst[t]), in ? doff[t] : kOOB);
    }
    if constexpr (Tl::SCALED) {
#pragma unroll
      for (int t = 0; t < Tl::SW; ++t)
        lds_load_b32(rsrc_words(uniform(sbase[t] + (slot_of_x(t) ? s * (int64_t)a.sx_step : s * (int64_t)a.sw_step)), 0x7fffffffu),
                     __builtin_amdgcn_readfirstlane(at + sdst[t]), s < s1 ? soff[t] : kOOB, 0);
    }
  };

  f32x4 acc[TI][TJ] = {};
  const uint32_t frag = r16 * 128 + ((g ^ (r16 & 7)) << 4);  // chunk g of row r16; chunk g + 4 lies at ^ 64
  auto wrow = [&](int j) { return GLU ? (j >> 1) * 128 + wn * 32 + (j & 1) * 16 : wn * 64 + j * 16; };
  const int xrow = wm * TI * 16;

  auto chunk = [](const unsigned char* p) { return *(const omt_u32x4*)p; };
  // every wave's loads up to `landed` stages before the last issued are in LDS, and its reads so far are done
  auto meet = [&](auto left) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(Tl::LOADS * decltype(left)::value) & ~0xF00);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // The last one to three words of rows that are no multiple of 16 bytes, as a step of their own after the others, zeros
  // beside them: laid into stage 0 by hand, with their block's scales. (In the loop they cost it 6%.)
  const bool ragged = MODE != kSplit && !XT && whole != a.row_bytes && s1 == a.steps;
  auto lay_rest = [&]() {
    meet(std::integral_constant<int, 0>{});
    for (int r = wave * 64 + lane; r < BM + 256; r += Tl::THREADS) {
      const bool of_x = r < BM;
      const int w = w_row(GLU ? (r - BM) & 127 : r - BM), part = GLU && r - BM >= 128;
      const bool in = of_x ? m0 + r < a.m : n0 + w < a.n;
      const unsigned char* src = of_x ? (const unsigned char*)a.x + (m0 + r) * a.xpitch
                                      : (const unsigned char*)(part ? a.w_up : a.w) + (n0 + w) * a.wpitch;
      omt_u32x4 rest = {};
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (in && whole + 4 * e < a.row_bytes) rest[e] = *(const uint32_t*)(src + whole + 4 * e);
      omt_u32x4* row = (omt_u32x4*)(lds + r * 128);
#pragma unroll
      for (int c = 0; c < 8; ++c) row[c] = c == (r & 7) ? rest : omt_u32x4{};
      if constexpr (Tl::SCALED) {
        const int64_t block = (a.row_bytes - 1) >> 7;
        float* scales = (float*)(lds + (BM + 256) * 128);
        // (rows between BM and SROWS are no tile's)
        if (of_x) scales[r] = in ? a.sx[(m0 + r) * (int64_t)a.sx_row + block * a.sx_step] : 0.f;
        else scales[Tl::SROWS + r - BM] = in ? (part ? a.sw_up : a.sw)[((n0 + w) >> 7) * (int64_t)a.sw_row + block * a.sw_step] : 0.f;
      }
    }
    __syncthreads();
  };

  // kF32, kBf16: a step in two halves, each of them its products while the next half's chunks come from LDS
  if constexpr (!Tl::SCALED) {
    omt_u32x4 wv[2][TJ], xv[2][TI];
    // Columns from + 16 i.. of a stage with the reduction along its columns: a lane's eight of the reduction (32 kk + 8 g ..)
    // for column r16. In a transposing read of a group of 16 lanes, lane p gives four columns (4 (p & 3) ..) of row p / 4 and
    // gets four rows of column p.
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* LdsQuad;
    const int turn = (r16 >> 2) * 2, quad = ((r16 >> 1) & 1) * 16 + (r16 & 1) * 8;
    auto across = [&](unsigned char* stage, int row_size, int from, int i, int kk) {
      unsigned char* p = stage + (kk * 32 + g * 8 + (r16 >> 2)) * row_size + (from + i / 4 * 64) * 2 +
                         (((i % 4) * 2) ^ turn) * 16 + quad;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad)(p + 4 * row_size));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      return omt_u32x4{l.x, l.y, h.x, h.y};
    };
    auto read = [&](int buf, int kk) {
      const unsigned char* xs = lds + buf * Tl::STAGE + xrow * 128 + (frag ^ (kk * 64));
      const unsigned char* ws = lds + buf * Tl::STAGE + BM * 128 + (frag ^ (kk * 64));
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        if constexpr (WT) wv[kk][j] = across(lds + buf * Tl::STAGE + BM * 128, 512, wn * 64, j, kk);
        else wv[kk][j] = chunk(ws + wrow(j) * 128);
      }
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        if constexpr (XT) xv[kk][i] = across(lds + buf * Tl::STAGE, BM * 2, xrow, i, kk);
        else xv[kk][i] = chunk(xs + i * 2048);
      }
    };
    auto multiply = [&](int kk) {
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          if constexpr (MODE == kBf16) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[kk][j]),
                                                                __builtin_bit_cast(bf16x8, xv[kk][i]), acc[i][j], 0, 0, 0);
          } else {
            const f32x4 wf = __builtin_bit_cast(f32x4, wv[kk][j]), xf = __builtin_bit_cast(f32x4, xv[kk][i]);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], xf[q], acc[i][j], 0, 0, 0);
          }
        }
    };
    // a read, then the products that hide it
    auto blend = [&]() {
      constexpr int kReads = TI * (XT ? 2 : 1) + TJ * (WT ? 2 : 1), kMfma = TI * TJ * (MODE == kF32 ? 4 : 1), kEach = kMfma / kReads;
#pragma unroll
      for (int r = 0; r < kReads; ++r) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kMfma - kReads * kEach, 0);
    };
#pragma unroll
    for (int p = 0; p < NS; ++p) issue(p, s0 + p);
    meet(std::integral_constant<int, NS - 1>{});
    read(0, 0);
    int cur = 0;
    for (int s = s0; s < s1; ++s) {
      const int nxt = cur + 1 == NS ? 0 : cur + 1;
      read(cur, 1);
      multiply(0);
      blend();
      meet(std::integral_constant<int, NS - 2>{});  // step s + 1 is there, and nothing of step s is read any more
      // the loads of a later step before the reads of the next, or after: whichever measured faster (4096 x 4096 x 4096
      // bf16: 256 rows 114 against 120 us, 128 rows 137 against 125)
      if constexpr (BM == 256) issue(cur, s + NS);
      read(nxt, 0);
      if constexpr (BM != 256) issue(cur, s + NS);
      multiply(1);
      blend();
      cur = nxt;
    }
    if (ragged) {
      lay_rest();
      read(0, 0);
      multiply(0);
    }
  } else {
    // a block's sum, then times both scales, onto the sum of the blocks
    constexpr int KQ = MODE == kFp8x ? 4 : 2;
    using Scale = std::conditional_t<MODE == kSplit, f32x4, float>;
    omt_u32x4 wv[TJ][KQ];
    Scale wscale[TJ];
    float xscale[TI];
    auto fragments = [&](omt_u32x4* f, const unsigned char* row) {
      const omt_u32x4 lo = chunk(row + frag), hi = chunk(row + (frag ^ 64));
      if constexpr (MODE == kFp8x) {
        f[0] = widen_fp8(lo[0], lo[1]), f[1] = widen_fp8(lo[2], lo[3]);
        f[2] = widen_fp8(hi[0], hi[1]), f[3] = widen_fp8(hi[2], hi[3]);
      } else {
        f[0] = lo, f[1] = hi;
      }
    };
    auto read_x = [&](omt_u32x4* f, int buf, int i) { fragments(f, lds + buf * Tl::STAGE + (xrow + i * 16) * 128); };
    auto read_w = [&](int buf) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) fragments(wv[j], lds + buf * Tl::STAGE + (BM + wrow(j)) * 128);
    };
    auto read_xscale = [&](int buf, int i) {
      xscale[i] = ((const float*)(lds + buf * Tl::STAGE + (BM + 256) * 128))[xrow + i * 16 + r16];
    };
    auto read_wscales = [&](int buf) {
      const float* sw = (const float*)(lds + buf * Tl::STAGE + (BM + 256) * 128) + Tl::SROWS;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        if constexpr (MODE == kSplit) wscale[j] = *(const f32x4*)(sw + wrow(j) + 4 * g);
        else wscale[j] = sw[wrow(j)];  // one block of 128 rows
      }
    };
    auto products = [&](f32x4* part, const omt_u32x4* xv) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) part[j] = f32x4{};
      if constexpr (MODE == kFp8x) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            part[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[j][q]),
                                                              __builtin_bit_cast(bf16x8, xv[q]), part[j], 0, 0, 0);
      } else if constexpr (MODE == kFp8) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
          part[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join8(wv[j][0], wv[j][1]), join8(xv[0], xv[1]),
                                                                     part[j], 0, 0, 0, 0, 0, 0);
      } else {  // high by low, low by high, high by high
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, wv[j][q == 1]),
                                                             __builtin_bit_cast(f16x8, xv[q == 0]), part[j], 0, 0, 0);
      }
    };
    auto scaled = [&](int i, const f32x4* part) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] += part[j] * (wscale[j] * xscale[i]);
    };
    auto row_by_row = [&](int buf) {
      read_w(buf);
      read_wscales(buf);
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        omt_u32x4 xv[KQ];
        f32x4 part[TJ];
        read_x(xv, buf, i);
        read_xscale(buf, i);
        products(part, xv);
        scaled(i, part);
      }
    };
    // A row of tiles ahead: its products run while the sums of the last are scaled (8192 x 4096 x 16384 at 256 rows: e4m3 550
    // -> 492 us, halves 2955 -> 2850). xv and wv hold the step's first fragments; `meet_here` is called before the last
    // row's products, when all of the step is in registers, `then` after them.
    omt_u32x4 xv[2][KQ];
    auto read_first = [&](int buf) {
      read_w(buf);
      read_x(xv[0], buf, 0);
      if (TI > 1) read_x(xv[1], buf, 1);
    };
    auto rows_ahead = [&](int buf, auto meet_here, auto then) {
      f32x4 part[2][TJ];
      read_wscales(buf);
#pragma unroll
      for (int i = 0; i < TI; ++i) read_xscale(buf, i);
      products(part[0], xv[0]);
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        constexpr int kLast = TI > 1 ? TI - 2 : 0;
        if (i + 2 < TI) read_x(xv[i & 1], buf, i + 2);
        if (i == kLast) meet_here();
        if (i + 1 < TI) products(part[(i + 1) & 1], xv[(i + 1) & 1]);
        if (i == kLast) then();
        scaled(i, part[i & 1]);
      }
    };
    if constexpr (BM == 256 ? MODE != kFp8 : MODE == kFp8x && (BM == 224 || BM == 64)) {
      // 256 rows of halves leave no registers, nor do 224 beside widened fragments, of four times the size: a step's first reads
      // wait for the waves to meet. (64 rows widened are faster so too: 175 us for 187, 4096 x 4096 x 4096.)
#pragma unroll
      for (int p = 0; p < NS - 1; ++p) issue(p, s0 + p);
      int cur = 0, nxt = NS - 1;
      for (int s = s0; s < s1; ++s) {
        meet(std::integral_constant<int, NS - 2>{});
        issue(nxt, s + NS - 1);
        if constexpr (MODE == kFp8x) {
          row_by_row(cur);
        } else {
          read_first(cur);
          rows_ahead(cur, [] {}, [] {});
        }
        cur = cur + 1 == NS ? 0 : cur + 1;
        nxt = nxt + 1 == NS ? 0 : nxt + 1;
      }
    } else {
      // the next step's first reads in the shadow of the last row's products (8192 x 4096 x 8192 at 128 rows: e4m3 312 -> 298
      // us, halves 1675 -> 1567; 4096 x 4096 x 4096 widened 132 -> 117)
#pragma unroll
      for (int p = 0; p < NS; ++p) issue(p, s0 + p);
      meet(std::integral_constant<int, NS - 1>{});
      read_first(0);
      int cur = 0;
      for (int s = s0; s < s1; ++s) {
        const int nxt = cur + 1 == NS ? 0 : cur + 1;
        rows_ahead(cur, [&] { meet(std::integral_constant<int, NS - 2>{}); },
                   [&] {
                     read_first(nxt);
                     issue(cur, s + NS);
                   });
        cur = nxt;
      }
    }
    if (ragged) {
      lay_rest();
      row_by_row(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & ~0xF00);
  asm volatile("" ::: "memory");
  __syncthreads();

  // A lane holds row r16 of each 16 x 16 tile, four columns of it: wcol(j) .. of the workgroup's.
  auto wcol = [&](int j) {
    return kRun == 4 ? wrow(j) + 4 * g : wrow(j & 2) + 8 * g + (j & 1) * 4;
  };
  const bool vec = (a.n & 7) == 0, vec4 = (a.n & 3) == 0;
  if (part) {
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row = xrow + i * 16 + r16;
      if (m0 + row >= a.m) continue;
#pragma unroll
      for (int j = 0; j < TJ; ++j) *(f32x4*)(part + row * 256 + wcol(j)) = acc[i][j];
    }
    todo -= s1 - s0;
    s0 = 0;
    ++tile;
    part += BM * 256;
    continue;
  }
  todo = 0;
  if constexpr (!GLU) {
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int m = m0 + xrow + i * 16 + r16;
      const int row = m < a.split ? m : m - a.split;
      if (m >= a.m || row >= a.limit) continue;
      void* out = m < a.split ? a.out : a.out2;
      if constexpr (kRun == 4) {
#pragma unroll
        for (int j = 0; j < TJ; ++j) store4_any(out, row, n0 + wcol(j), a.n, vec4, a.out_kind, acc[i][j]);
      } else {
#pragma unroll
        for (int j = 0; j < TJ; j += 2)
          store8_any(out, row, n0 + wcol(j), a.n, vec, a.out_kind, beside(acc[i][j], acc[i][j + 1]));
      }
    }
  } else {
    uint32_t* top = (uint32_t*)lds;  // [g, u or h][wave][row]: each wave's largest magnitudes of 32 columns
    constexpr bool out8 = MODE == kFp8x;  // 8-bit operands give an 8-bit result and keep nothing
    const bool keep8 = !out8 && a.keep == kKeepFp8;
    auto note = [&](int z, int i, f32x8 v) {
      uint32_t b = abs_bits8(v);
      b = max_u32(b, (uint32_t)__shfl_xor((int)b, 16));
      b = max_u32(b, (uint32_t)__shfl_xor((int)b, 32));
      if (g == 0) top[(z * 4 + wn) * BM + xrow + i * 16 + r16] = b;
    };
    // the block's scale and its reciprocal, as the other kernels have them
    auto scale_of = [&](int z, int lr, float* inv) {
      const uint32_t* p = top + z * 4 * BM + lr;
      const float s = block_scale(max_u32(max_u32(p[0], p[BM]), max_u32(p[2 * BM], p[3 * BM])));
      *inv = 1.f / s;
      return s;
    };
    const int blocks = (a.n + kFp8Block - 1) / kFp8Block, c = n0 + wcol(0);
    const bool first = wn == 0 && g == 0;
    auto gates = [&](int i) { return beside(acc[i][0], acc[i][1]); };
    auto ups = [&](int i) { return beside(acc[i][2], acc[i][3]); };
    auto finish = [&](auto act) {
      auto h8 = [&](int i) {
        const f32x8 gv = gates(i), uv = ups(i);
        f32x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = glu_act(gv[e], decltype(act)::value) * uv[e];
        return h;
      };
      if constexpr (out8) {  // h in the place of g
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          const f32x8 h = h8(i);
          note(0, i, h);
          acc[i][0] = f32x4{h[0], h[1], h[2], h[3]};
          acc[i][1] = f32x4{h[4], h[5], h[6], h[7]};
        }
        __syncthreads();
      } else if (keep8) {
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          note(0, i, gates(i));
          note(1, i, ups(i));
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int lr = xrow + i * 16 + r16, m = m0 + lr;
        if (m >= a.m) continue;
        const int64_t at = (int64_t)m * blocks + (n0 >> 7);
        float inv;
        if constexpr (out8) {
          const float s = scale_of(0, lr, &inv);
          if (first) a.out_scale[at] = s;
          store8_fp8(a.out, m, c, a.n, vec, gates(i), inv);
        } else {
          store8_any(a.out, m, c, a.n, vec, a.out_kind, h8(i));
          if (keep8) {
            float s = scale_of(0, lr, &inv);
            if (first) a.keep_gs[at] = s;
            store8_fp8(a.keep_g, m, c, a.n, vec, gates(i), inv);
            s = scale_of(1, lr, &inv);
            if (first) a.keep_us[at] = s;
            store8_fp8(a.keep_u, m, c, a.n, vec, ups(i), inv);
          } else if (a.keep == kKeepFull) {
            store8_any(a.keep_g, m, c, a.n, vec, a.out_kind, gates(i));
            store8_any(a.keep_u, m, c, a.n, vec, a.out_kind, ups(i));
          }
        }
      }
    };
    if (a.act == OMT_GLU_SILU) finish(std::integral_constant<int, OMT_GLU_SILU>{});
    else if (a.act == OMT_GLU_GELU) finish(std::integral_constant<int, OMT_GLU_GELU>{});
    else finish(std::integral_constant<int, OMT_GLU_RELU>{});
  }
  }
}

template <int MODE, bool GLU, int BM, int NS, bool XT = false, bool WT = false>
int launch_gemm(const GemmArgs& a, hipStream_t stream) {
  constexpr int kThreads = GemmTile<MODE, BM, NS>::THREADS;
  const int64_t tiles = (int64_t)a.gx * a.gy, groups = (int64_t)a.whole + a.sharers;
  if ((tiles > groups ? tiles : groups) * kThreads > UINT32_MAX)  // what a launch holds; one of more runs a part of it and says nothing
    return fail(OMT_UNSUPPORTED, "ffn_gemm_kernel: %lld tiles", (long long)tiles);
  hipLaunchKernelGGL((ffn_gemm_kernel<MODE, GLU, BM, NS, XT, WT>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
  return launch_check("ffn_gemm_kernel");
}

// Two stages, or three where they fit the CU's 160 KB. Two workgroups of 16 rows fit it together, and two of 64 without
// scales, and hide each other's waits better than a third stage does (64 rows bf16, 4096 x 4096 x 4096: 144 us with two, 226
// with three and one workgroup). Of 64 rows with scales one fits, and gains nothing from a third (16384 x 4096 x 8192 e4m3 964 us
// with two, 960 with three; widened 1388 and 1539; halves, x 2048, 1159 and 1161); 128 rows gain 1-3%.
template <int MODE, int BM>
constexpr int gemm_stages() {
  return BM > 64 && 3 * GemmTile<MODE, BM, 1>::STAGE <= 160 * 1024 ? 3 : 2;
}
// bm rows of x to a tile (a.gx, a.gy in those units). The heights between 64 and 256 are there for the rows that a whole
// number of tiles leaves over, and the CUs: 777 rows by 20 columns of tiles are 140 workgroups of 128 rows, 180 of 96.
constexpr int kHeights = 8, kBm[kHeights] = {16, 64, 96, 128, 160, 192, 224, 256};
template <int MODE, bool GLU, bool WT = false, int V = 0>
int launch_gemm_of(const GemmArgs& a, int bm, hipStream_t stream) {
  if constexpr (V + 1 < kHeights)
    if (bm != kBm[V]) return launch_gemm_of<MODE, GLU, WT, V + 1>(a, bm, stream);
  return launch_gemm<MODE, GLU, kBm[V], gemm_stages<MODE, kBm[V]>(), false, WT>(a, stream);
}
// kBf16, plain, with w, or both operands, along their columns (the latter: 128 or 256 rows)
int ffn_gemm_bf16_w(const GemmArgs& a, int bm, hipStream_t stream);
int ffn_gemm_bf16_xw(const GemmArgs& a, int bm, hipStream_t stream);
// kF32 in the gated form only, kFp8 in the plain one only
int ffn_gemm_f32(const GemmArgs& a, int bm, hipStream_t stream);
int ffn_gemm_bf16(const GemmArgs& a, bool glu, int bm, hipStream_t stream);
int ffn_gemm_split(const GemmArgs& a, bool glu, int bm, hipStream_t stream);
int ffn_gemm_fp8x(const GemmArgs& a, bool glu, int bm, hipStream_t stream);
int ffn_gemm_fp8(const GemmArgs& a, int bm, hipStream_t stream);

}  // namespace omt
