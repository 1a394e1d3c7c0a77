#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_bf16(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  if (bm == 16) return glu ? launch_gemm<kBf16, true, 16, 2>(a, stream) : launch_gemm<kBf16, false, 16, 2>(a, stream);
  return glu ? launch_gemm<kBf16, true, 64, 2>(a, stream) : launch_gemm<kBf16, false, 64, 2>(a, stream);
}

}  // namespace omt
