// x W^T of e4m3 operands (dense_gemm.h).
#include "dense_gemm.h"

namespace maloq {
namespace dense {

void launch_nt8(int out, const GemmArgs& a, int tile, void* stream) {
  if (out == F32) launch_gemm<E4M3, F32, false, false>(a, tile, stream);
  if (out == BF16) launch_gemm<E4M3, BF16, false, false>(a, tile, stream);
  if (out == F16) launch_gemm<E4M3, F16, false, false>(a, tile, stream);
}

}  // namespace dense
}  // namespace maloq
