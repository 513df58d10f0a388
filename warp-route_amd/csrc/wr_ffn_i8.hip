// Products of int8 codes (wr_ffn_gemm.h): int32 sums, which are exact, scaled per
// row and column in the epilogue.
#include "wr_ffn_gemm.h"

namespace wr {
namespace ffn {

hipError_t launch_i8(const GemmArgs& g, int shape, int form, hipStream_t s) {
  if (form == kFormGatedMax)
    return launch_shape<int8_t, false, false, kGatedMax>(g, shape, s);
  return launch_shape<int8_t, false, false, kScale>(g, shape, s);
}

}  // namespace ffn
}  // namespace wr
