#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_bf16(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return launch_gemm_of<kBf16>(a, glu, bm, stream);
}

}  // namespace omt
