// The 8-bit product for few rows (ffn_few.hip).
#pragma once

#include "ffn_gemm.h"

namespace omt {

struct FewArgs {
  const void *x, *w;     // rows of k e4m3, k a multiple of 4
  const float *sx, *sw;  // [m][blocks], [ceil(n / 128)][blocks]
  void* out;
  int m, n, k, out_kind;
};

// The rows of x that it takes in one piece, 0 for the tiles: a workgroup reads all of x, so its time goes with rows times k
// (16 x 1024 x 16384: 20.4 us for the tiles' 16.4; 64 x 4096 x 4096: 15.5 for 15.2), and for over 16 rows, where it has 16 rows of
// w, with n (32 x 16384 x 4096: 31 for 24). The limits are where 16, 32 and 64 rows meet the tiles, and hold for fewer rows too,
// although one row is the faster here past them (1 x 4096 x 16384: 17.7 for 21.5).
inline int few_rows(int64_t m, int64_t n, int64_t k) {
  const int rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
  return m <= rows && rows * k <= 16 * 8192 && (m <= 16 || n <= 4096) ? rows : 0;
}
// m at most few_rows of them
int matmul_fp8_few(const FewArgs& a, hipStream_t stream);

}  // namespace omt
