// x W^T whose activation's argument is kept in 8 bits (dense_gemm.h, pack8.h).  8192 x 4096 x 16384 bf16 with silu 822 to 833 us, where
// the argument stored in 16 bits takes 799 to 803 and none 780 to 783 (without an activation 765 to 771; ten launches in a row, all in
// one run): 134 MB less to write, more of the vector units' work, which a tile of 256 x 256, alone on its CU, hides behind nothing.
#include "pack8.h"

namespace maloq {
namespace dense {

void launch_nt_packed(int in, const GemmArgs& a, int tile, void* stream) {
  if (in == F32) launch_gemm<F32, F32, false, false, true>(a, tile, stream);
  if (in == BF16) launch_gemm<BF16, BF16, false, false, true>(a, tile, stream);
  if (in == F16) launch_gemm<F16, F16, false, false, true>(a, tile, stream);
}

}  // namespace dense
}  // namespace maloq
