#include "ffn_gemm.h"

namespace omt {

int ffn_gemm_fp8(const GemmArgs& a, int bm, hipStream_t stream) { return launch_gemm_of<kFp8, false>(a, bm, stream); }

}  // namespace omt
