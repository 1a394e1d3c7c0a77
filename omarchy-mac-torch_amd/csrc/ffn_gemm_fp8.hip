#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_fp8(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  if (bm == 16) return glu ? launch_gemm<kFp8x, true, 16, 2>(a, stream) : launch_gemm<kFp8x, false, 16, 2>(a, stream);
  return glu ? launch_gemm<kFp8x, true, 64, 2>(a, stream) : launch_gemm<kFp8x, false, 64, 2>(a, stream);
}

}  // namespace omt
