// The 8-bit product for few rows, out = x[m][k] w[n][k]^T with m of a token or of a batch's next tokens: bound by reading
// w once, and where w is small, by a launch. A workgroup has 16 or 32 rows of w over the whole reduction, so nothing is left
// to join between workgroups; its waves take the blocks of 128 in turn, 16 bytes of a row to a lane, from memory to
// registers: w's values are used once, and the way through LDS would only add waits. The waves' sums meet in LDS, in the
// waves' order. The matrix instruction is bfloat16's (e4m3 is exact in it, and its sums nearly so), whatever the result.
//
// Against the tiles of 16 rows with their shares joined by a second launch, us (m x n x k, weights from memory):
// 1 x 4096 x 8192 9.2 for 14.7 (33.5 MB: 7.1 at a copy's rate), 1 x 4096 x 4096 5.8 for 11.0, 1 x 512 x 512 3.2 for 5.8,
// 16 x 4096 x 4096 7.4 for 12.7, 32 x 4096 x 4096 9.5 for 12.5, 64 x 2048 x 2048 8.7 for 10.3.
// One block in flight to a wave and 16 waves to a CU read as fast as deeper rings of 8 or 4 waves (1 x 4096 x 8192: 9.5 to
// 13.4), which also hold what they never use where a wave has two blocks in all.
#include "ffn_few.h"

namespace omt {

template <int WAVES, int MT, int NT>
__global__ void __launch_bounds__(WAVES * 64) matmul_fp8_few_kernel(FewArgs a) {
  __shared__ f32x4 sums[WAVES][MT][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NT), blocks = (a.k + kFp8Block - 1) / kFp8Block, whole = a.k / kFp8Block;
  const auto w = make_rsrc((const char*)a.w + (int64_t)n0 * a.k, 0x7fffffffu), x = make_rsrc(a.x, 0x7fffffffu),
             sx = make_rsrc(a.sx, 0x7fffffffu);
  const float* sw = a.sw + (int64_t)(n0 / kFp8Block) * blocks;
  // the lane's row of each tile, as an offset; rows past an operand's last read as 0 (out of the range that the load checks)
  uint32_t wrow[NT], xrow[MT], srow[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) wrow[t] = n0 + t * 16 + r16 < a.n ? (uint32_t)(t * 16 + r16) * (uint32_t)a.k : kOOB;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    xrow[t] = t * 16 + r16 < a.m ? (uint32_t)(t * 16 + r16) * (uint32_t)a.k : kOOB;
    srow[t] = t * 16 + r16 < a.m ? (uint32_t)((t * 16 + r16) * blocks) * 4 : kOOB;
  }
  struct Frag {
    omt_u32x4 c[2];  // bytes 16 g.. and 64 + 16 g.. of a block of a row
  };
  auto load = [&](Frag& f, auto r, uint32_t row, int b) {
    const uint32_t at = (uint32_t)b * kFp8Block + g * 16;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      f.c[c] = __builtin_bit_cast(omt_u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(row + at + c * 64), 0, 0));
  };
  auto load_rest = [&](Frag& f, auto r, uint32_t row, int b) {  // up to the row's end, word by word
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = b * kFp8Block + g * 16 + (e >> 2) * 64 + (e & 3) * 4;
      f.c[e >> 2][e & 3] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)(at < a.k ? row + (uint32_t)at : kOOB), 0, 0);
    }
  };
  f32x4 acc[MT][NT] = {};
  auto block = [&](int b, auto load) {
    Frag wf[NT], xf[MT];
    float xs[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) load(wf[t], w, wrow[t], b);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      load(xf[t], x, xrow[t], b);
      xs[t] = bload(sx, srow[t] + b * 4, 0);
    }
    const float ws = sw[b];
    omt_u32x4 wv[NT][4];
    auto widen = [](omt_u32x4* to, const Frag& f) {
#pragma unroll
      for (int q = 0; q < 4; ++q) to[q] = widen_fp8(f.c[q >> 1][(q & 1) * 2], f.c[q >> 1][(q & 1) * 2 + 1]);
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) widen(wv[t], wf[t]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      omt_u32x4 xv[4];
      widen(xv, xf[i]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 part = {};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[t][q]),
                                                         __builtin_bit_cast(bf16x8, xv[q]), part, 0, 0, 0);
        acc[i][t] += part * (xs[i] * ws);
      }
    }
  };
#pragma unroll 1
  for (int b = wave; b < whole; b += WAVES) block(b, load);
  if (whole < blocks && wave == whole % WAVES) block(whole, load_rest);

#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][i][t][lane] = acc[i][t];  // columns 16 t + 4 g.. of row 16 i + r16
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NT * 256; o += WAVES * 64) {
    const int row = o / (NT * 16), c = o % (NT * 16);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) sum += sums[v][row >> 4][c >> 4][((c & 15) >> 2) * 16 + (row & 15)][c & 3];
    if (row < a.m && n0 + c < a.n) {
      const int64_t at = (int64_t)row * a.n + n0 + c;
      if (a.out_kind == kOutBf16) ((__bf16*)a.out)[at] = (__bf16)sum;
      else ((float*)a.out)[at] = sum;
    }
  }
}

template <int WAVES, int MT, int NT>
static int launch_few(const FewArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(a.n, 16 * NT));
  hipLaunchKernelGGL((matmul_fp8_few_kernel<WAVES, MT, NT>), grid, dim3(WAVES * 64), 0, stream, a);
  return launch_check("matmul_fp8_few_kernel");
}

// 16 rows of w to a workgroup of 16 waves; 32 to one of 8 where there are workgroups enough (n = 16384, k = 1024, 16 rows:
// 6.0 us for 8.3; n = 32768, k = 4096: 31.4 for 39.3: the rows of x are read half as often). For more rows of x 8 waves, whose
// registers leave room for two workgroups (32 x 2048 x 2048: 5.9 for 6.1).
int matmul_fp8_few(const FewArgs& a, hipStream_t stream) {
  if (a.m <= 16) return a.n < 8192 ? launch_few<16, 1, 1>(a, stream) : launch_few<8, 1, 2>(a, stream);
  return a.m <= 32 ? launch_few<8, 2, 1>(a, stream) : launch_few<8, 4, 1>(a, stream);
}

}  // namespace omt
