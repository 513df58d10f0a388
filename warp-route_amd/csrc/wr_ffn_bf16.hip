// Products of the dense FFN in bf16 (wr_ffn_gemm.h).
#include "wr_ffn_gemm.h"

namespace wr {
namespace ffn {

hipError_t launch_bf16(const GemmArgs& g, int shape, int form, hipStream_t s) {
  return launch_float<bf16>(g, shape, form, s);
}

}  // namespace ffn
}  // namespace wr
