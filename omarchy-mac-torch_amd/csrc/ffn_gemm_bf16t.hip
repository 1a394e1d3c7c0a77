#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_bf16_w(const GemmArgs& a, int bm, hipStream_t stream) {
  return launch_gemm_of<kBf16, false, true>(a, bm, stream);
}
int ffn_gemm_bf16_xw(const GemmArgs& a, int bm, hipStream_t stream) {
  return bm == 256 ? launch_gemm<kBf16, false, 256, gemm_stages<kBf16, 256>(), true, true>(a, stream)
                   : launch_gemm<kBf16, false, 128, gemm_stages<kBf16, 128>(), true, true>(a, stream);
}

}  // namespace omt
