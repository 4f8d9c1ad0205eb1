// x W^T of 16-bit and fp32 operands (dense_gemm.h).
#include "dense_gemm.h"

namespace maloq {
namespace dense {

void launch_nt(int in, const GemmArgs& a, int tile, void* stream) {
  if (in == F32) launch_gemm<F32, F32, false, false>(a, tile, stream);
  if (in == BF16) launch_gemm<BF16, BF16, false, false>(a, tile, stream);
  if (in == F16) launch_gemm<F16, F16, false, false>(a, tile, stream);
}

}  // namespace dense
}  // namespace maloq
