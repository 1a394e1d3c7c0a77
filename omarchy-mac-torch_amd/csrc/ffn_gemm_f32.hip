#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_f32(const GemmArgs& a, int bm, hipStream_t stream) {
  return launch_gemm_of<kF32, true>(a, bm, stream);
}

}  // namespace omt
