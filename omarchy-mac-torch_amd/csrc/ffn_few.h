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

// The rows of x that it takes in one piece, 0 where the tiles are the faster: a workgroup reads all of x, so its time goes
// with rows times k (1024 x 16384, 16 rows: 20.4 us for the tiles' 16.4; 4096 x 4096, 64 rows: 15.5 for 15.2), and for over
// 16 rows with n (32 x 16384 x 4096: 31 for 24).
inline int few_rows(int64_t m, int64_t n, int64_t k) {
  const int rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
  return m <= rows && rows * k <= 16 * 8192 && (m <= 16 || n <= 4096) ? rows : 0;
}
// m at most few_rows of them
int matmul_fp8_few(const FewArgs& a, hipStream_t stream);

}  // namespace omt
