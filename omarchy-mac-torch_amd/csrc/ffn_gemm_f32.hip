#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_f32(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  if (bm == 16) return glu ? launch_gemm<kF32, true, 16, 2>(a, stream) : launch_gemm<kF32, false, 16, 2>(a, stream);
  return glu ? launch_gemm<kF32, true, 64, 2>(a, stream) : launch_gemm<kF32, false, 64, 2>(a, stream);
}

}  // namespace omt
