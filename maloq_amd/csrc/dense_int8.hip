// x W^T of int8 operands (dense_gemm.h).  Sums are exact: int32, also between the parts of a contraction.  A half of a tile's K step,
// 64 bytes of a row, is one MFMA of 16 x 16 x 64, so that the loops are those of 16 bits.  8192 x 4096 x 16384 of normal numbers' rows
// with bias 446 to 452 us (2.4 POP/s), with silu 468 to 471, of zeros 401 (power, then starts and epilogues: eight tiles a CU); the
// library's product, without an epilogue, 469 to 490, e4m3 operands 429 to 439.  fp32 results 502 (twice the bytes;
// 12 registers spill, where e4m3's 473 spill none).
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
