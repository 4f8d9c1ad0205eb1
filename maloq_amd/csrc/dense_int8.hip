// x W^T of int8 operands (dense_gemm.h).
#include "dense_gemm.h"

namespace maloq {
namespace dense {

void launch_nt_int8(int out, const GemmArgs& a, int tile, void* stream) {
  if (out == F32) launch_gemm<I8, F32, false, false>(a, tile, stream);
  if (out == BF16) launch_gemm<I8, BF16, false, false>(a, tile, stream);
  if (out == F16) launch_gemm<I8, F16, false, false>(a, tile, stream);
}

}  // namespace dense
}  // namespace maloq
