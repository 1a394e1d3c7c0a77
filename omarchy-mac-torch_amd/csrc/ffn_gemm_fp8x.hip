#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_fp8x(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return glu ? launch_gemm_of<kFp8x, true>(a, bm, stream) : launch_gemm_of<kFp8x, false>(a, bm, stream);
}

}  // namespace omt
