#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_bf16(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return glu ? launch_gemm_of<kBf16, true>(a, bm, stream) : launch_gemm_of<kBf16, false>(a, bm, stream);
}

}  // namespace omt
