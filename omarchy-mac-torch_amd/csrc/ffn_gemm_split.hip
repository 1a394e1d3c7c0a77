#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_split(const GemmArgs& a, bool glu, int bm, hipStream_t stream) {
  return glu ? launch_gemm_of<kSplit, true>(a, bm, stream) : launch_gemm_of<kSplit, false>(a, bm, stream);
}

}  // namespace omt
