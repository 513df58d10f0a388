// Products of the dense FFN in f32 (wr_ffn_gemm.h).
#include "wr_ffn_gemm.h"

namespace wr {
namespace ffn {

hipError_t launch_f32(const GemmArgs& g, int shape, int form, hipStream_t s) {
  return launch_float<float>(g, shape, form, s);
}

}  // namespace ffn
}  // namespace wr
