#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_fp8(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return launch_gemm_of<kFp8x>(a, glu, bm, stream);
}

}  // namespace omt
