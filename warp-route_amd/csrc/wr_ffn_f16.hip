// Products of the dense FFN in f16 (wr_ffn_gemm.h).
#include "wr_ffn_gemm.h"

namespace wr {
namespace ffn {

hipError_t launch_f16(const GemmArgs& g, int shape, int form, hipStream_t s) {
  return launch_float<f16>(g, shape, form, s);
}

}  // namespace ffn
}  // namespace wr
