// x W^T of a few rows (tokens in decoding): the weights are read once and everything else hides
// under that.
//
// A wave has 16 columns, straight from memory into the fragments of 16 x 16 MFMAs: a lane has 16
// bytes of one weight row (lane % 16) and of one row of x, the same elements of both, which is all
// that a product asks of their order.  The next piece is loaded before this one is multiplied.  No
// alignment is asked for: loads of 16 bytes may start anywhere.
//
// In 8 bits an instruction's own sums are short of fp32 as those of the tiles are (dense_gemm.h).
//
// The sixteen waves of a workgroup take every sixteenth 128 bytes of the contraction each, and their
// sums meet in LDS, in their order.  With many rows x is read as often as W this way, through the
// same L1: beyond FEW_ROWS the tiles of dense_gemm.h are faster (4096 -> 16384 bf16, weights from memory: one
// row 23.2 us, 5.8 TB/s, and 31.0 with tiles; 16 rows 33.6 and 33.1, in 8 bits 19.5 and 23.8).  Waves and pieces
// in flight, one row, 16 and 8 bits: 16 waves of one piece 23.2 and 14.8 us, of two 26.6 and 16.0; eight of one 25.7 and
// 16.8, of two 26.0 and 17.7; four of four 27.7 and 16.1.
#include "dense_gemm.h"

namespace maloq {
namespace dense {

constexpr int WAVES = 16;

// 16 bytes of a row
__device__ __forceinline__ i32x4 load16(const char* p) { return __builtin_bit_cast(i32x4, load_loose(p)); }
// .. of which `have` bytes exist, the others zero
template <int ES>
__device__ __forceinline__ i32x4 load_part(const char* p, int have) {
  union {
    i32x4 v;
    uint16_t h[8];
    uint8_t b[16];
  } u;
  u.v = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16 / ES; ++i) {
    if constexpr (ES == 2) {
      if (i * 2 < have) u.h[i] = *reinterpret_cast<const uint16_t*>(p + 2 * i);
    } else {
      if (i < have) u.b[i] = *reinterpret_cast<const uint8_t*>(p + i);
    }
  }
  return u.v;
}

template <int IN>
__device__ __forceinline__ f32x4 product16(const i32x4& a, const i32x4& b, f32x4 c) {
  if constexpr (IN == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  if constexpr (IN == F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  if constexpr (IN == E4M3) {
    typedef long i64x2 __attribute__((ext_vector_type(2)));
    const i64x2 x = __builtin_bit_cast(i64x2, a), y = __builtin_bit_cast(i64x2, b);
    c = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(x[0], y[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(x[1], y[1], c, 0, 0, 0);
  }
}

template <int IN, int OUT>
__device__ __forceinline__ void finish1(const GemmArgs& a, int m, int n, float v) {
  if constexpr (IN == E4M3) v = v * a.e.sa[m] * a.e.sb[n];
  if (a.e.bias) v += load1<OUT>(a.e.bias, n);
  if (a.e.z) store1<OUT>(a.e.z, static_cast<int64_t>(m) * a.N + n, v);
  with_act(a.e.act, [&](auto act) { v = act_fwd<OUT == F32, decltype(act)::value>(v); });
  if (a.e.res) v += load1<OUT>(a.e.res, m * a.e.ldr + n);
  store1<OUT>(a.e.out, m * a.e.ldo + n, v);
}

template <int IN, int OUT>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(GemmArgs a) {
  constexpr int ES = IN == E4M3 ? 1 : 2;
  __shared__ float sums[WAVES][256];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int n0 = blockIdx.x * 16;
  const int kbytes = a.K * ES, at = (lane >> 4) * 16;
  const int pieces = kbytes / 128, n = n0 + (lane & 15), m = lane & 15;
  const char* w = a.b + (n < a.N ? n : a.N - 1) * a.ldb + at;
  const char* x = a.a + (m < a.M ? m : a.M - 1) * a.lda + at;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};

  constexpr int U = 1;  // 128-byte pieces at a time, as many again on the way
  struct Some {
    i32x4 w[U][2], x[U][2];
  };
  auto load = [&](Some& s, int piece) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = (piece + u * WAVES < pieces ? piece + u * WAVES : pieces - 1) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) s.w[u][h] = load16(w + p + 64 * h), s.x[u][h] = load16(x + p + 64 * h);
    }
  };
  auto multiply = [&](const Some& s, int piece) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (piece + u * WAVES >= pieces) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) acc = product16<IN>(s.w[u][h], s.x[u][h], acc);
    }
  };
  if (wave < pieces) {
    Some s0, s1;
    load(s0, wave);
    for (int piece = wave;;) {
      const int next = piece + U * WAVES, last = next + U * WAVES;
      if (next < pieces) load(s1, next);
      multiply(s0, piece);
      if (next >= pieces) break;
      if (last < pieces) load(s0, last);
      multiply(s1, next);
      if (last >= pieces) break;
      piece = last;
    }
  }
  if (wave == pieces % WAVES && pieces * 128 < kbytes) {  // the wave whose turn it is: the rest
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int left = kbytes - pieces * 128 - 64 * h - at;
      acc = product16<IN>(load_part<ES>(w + pieces * 128 + 64 * h, left), load_part<ES>(x + pieces * 128 + 64 * h, left), acc);
    }
  }
  // a lane has columns 4 (lane / 16) .. + 3 of row lane % 16
  *reinterpret_cast<f32x4*>(&sums[wave][(lane & 15) * 16 + 4 * (lane >> 4)]) = acc;
  __syncthreads();
  const int row = tid / 16, c = n0 + tid % 16;
  if (row >= a.M || c >= a.N) return;
  float v = 0.f;
#pragma unroll
  for (int s = 0; s < WAVES; ++s) v += sums[s][tid];
  finish1<IN, OUT>(a, row, c, v);
}

template <int IN, int OUT>
static void launch(const GemmArgs& a, hipStream_t st) {
  few_rows_kernel<IN, OUT><<<(a.N + 15) / 16, 64 * WAVES, 0, st>>>(a);
}

void launch_few(int in, int out, const GemmArgs& a, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (in == BF16) launch<BF16, BF16>(a, st);
  if (in == F16) launch<F16, F16>(a, st);
  if (in == E4M3 && out == F32) launch<E4M3, F32>(a, st);
  if (in == E4M3 && out == BF16) launch<E4M3, BF16>(a, st);
  if (in == E4M3 && out == F16) launch<E4M3, F16>(a, st);
}

}  // namespace dense
}  // namespace maloq
