#pragma once
// Rows of values in 8 bits for a backward pass: blocks of 32 consecutive values of a row (the last one perhaps shorter),
// each with one byte e, value = q 2^(e - 133).  e is the exponent field of the block's largest finite magnitude, one more
// where its mantissa is at least 126.5 / 64, so that q = nearest(value / step) is within -126 .. 126; 127 and -127 stand
// for the infinities and -128 for NaN.  A step is a power of two: the division is exact, and what x is kept as does not
// hang on how a quotient was rounded.  What comes back is off by half a step, 2^-6 to 2^-7 of half the largest, has seven
// bits, and so is exact in bf16 and fp16 (but for the largest of a type, which would round to twice a power: clamped).
#include "dense_gemm.h"

namespace maloq {
namespace dense {

constexpr int PACK = 32;  // values of a block, four lanes of eight
__host__ __device__ constexpr int64_t pack_blocks(int64_t n) { return (n + PACK - 1) / PACK; }

struct __attribute__((packed, aligned(1))) Eight {
  uint32_t w[2];
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// Eight values of a lane, of which the four lanes that share a block give the exponent (all four must be active).
// SIGN: a positive value stays positive.
template <bool SIGN>
__device__ __forceinline__ Eight pack_values(const float (&v)[8], int& e) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t b = finite_bits(v[k]);
    m = m > b ? m : b;
  }
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const uint32_t u = __shfl_xor(m, o);
    m = m > u ? m : u;
  }
  e = static_cast<int>((m + 0x30000u) >> 23);
  Eight r = {{0, 0}};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    int q = static_cast<int>(rintf(ldexpf(v[k], 133 - e)));
    if (SIGN && q == 0 && v[k] > 0.f) q = 1;
    if (__builtin_isinf(v[k])) q = v[k] > 0.f ? 127 : -127;
    if (v[k] != v[k]) q = -128;
    r.w[k / 4] |= static_cast<uint32_t>(q & 255) << (8 * (k % 4));
  }
  return r;
}
// TYPE: what the values must fit
template <int TYPE>
__device__ __forceinline__ void unpack_values(const Eight& p, int e, float (&v)[8]) {
  constexpr float most = TYPE == F16 ? 65504.f : (TYPE == BF16 ? 0x1.fep127f : 0x1.fffffep127f);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int q = static_cast<int>(p.w[k / 4] << (24 - 8 * (k % 4))) >> 24;
    float x = within(ldexpf(static_cast<float>(q), e - 133), most);
    if (q == 127) x = __builtin_inff();
    if (q == -127) x = -__builtin_inff();
    if (q == -128) x = __builtin_nanf("");
    v[k] = x;
  }
}
__device__ __forceinline__ Eight load_eight(const uint8_t* p, int have) {
  if (have >= 8) return *reinterpret_cast<const Eight*>(p);
  Eight r = {{0, 0}};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < have) r.w[k / 4] |= static_cast<uint32_t>(p[k]) << (8 * (k % 4));
  return r;
}
__device__ __forceinline__ void store_eight(uint8_t* p, const Eight& v, int have) {
  if (have >= 8) {
    *reinterpret_cast<Eight*>(p) = v;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < have) p[k] = static_cast<uint8_t>(v.w[k / 4] >> (8 * (k % 4)));
  }
}

// What an activation is given, from a product's epilogue: eight columns from n on (a multiple of 8) of row m.  The four
// lanes of a block call it together; those past the last column too.
__device__ __forceinline__ void pack_argument(const Epilogue& e, int64_t m, int n, int N, const float (&z)[8]) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = n + k < N ? z[k] : 0.f;
  int x;
  const Eight q = e.act == ACT_RELU ? pack_values<true>(v, x) : pack_values<false>(v, x);
  if (n >= N) return;
  store_eight(e.z8 + m * N + n, q, N - n);
  if (n % PACK == 0) e.ze[m * pack_blocks(N) + n / PACK] = static_cast<uint8_t>(x);
}

}  // namespace dense
}  // namespace maloq
