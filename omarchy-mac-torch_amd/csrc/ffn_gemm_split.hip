#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_split(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return launch_gemm_of<kSplit>(a, glu, bm, stream);
}

}  // namespace omt
