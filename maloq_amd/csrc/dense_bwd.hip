// The products of a dense layer's gradients (dense_gemm.h): dz W, the weights read across their
// rows, and dz^T x, both operands read across theirs.
#include "dense_gemm.h"

namespace maloq {
namespace dense {

void launch_nn(int in, const GemmArgs& a, int tile, void* stream) {
  if (in == F32) launch_gemm<F32, F32, false, true>(a, tile, stream);
  if (in == BF16) launch_gemm<BF16, BF16, false, true>(a, tile, stream);
  if (in == F16) launch_gemm<F16, F16, false, true>(a, tile, stream);
}

void launch_tn(int in, const GemmArgs& a, int tile, void* stream) {
  if (in == F32) launch_gemm<F32, F32, true, true>(a, tile, stream);
  if (in == BF16) launch_gemm<BF16, BF16, true, true>(a, tile, stream);
  if (in == F16) launch_gemm<F16, F16, true, true>(a, tile, stream);
}

}  // namespace dense
}  // namespace maloq
