#pragma once
// Rows of values in 8 bits for a backward pass: blocks of 32 consecutive values of a row (the last one perhaps shorter),
// each with one byte e, value = q 2^(e - 133).  e is the exponent field of the block's largest finite magnitude, one more
// where its mantissa is at least 126.5 / 64, and at least 7 (steps of 2^-126), so that q = nearest(value / step) is within
// -126 .. 126; 127 and -127 stand for the infinities and -128 for NaN.  A step is a power of two: the division is exact, and
// what x is kept as does not hang on how a quotient was rounded.  What comes back is off by half a step, 2^-7 to 2^-6 of
// half the largest, has seven bits, and so is exact in bf16 and fp16 (but for the largest of a type, which would round to
// twice a power: clamped, in fp32 to bf16's, which is as near, so that all are bf16 numbers).
//
// These run in the epilogue of products that leave nothing else for the vector units to hide behind: a value takes four
// instructions to pack (its magnitude's maximum, a multiplication and addition that rounds it to an integer in the low bits,
// three byte selections for four) and three to unpack.  What is not finite takes a branch of its own.
#include "dense_gemm.h"

namespace maloq {
namespace dense {

constexpr int PACK = 32;  // values of a block, four lanes of eight
__host__ __device__ constexpr int64_t pack_blocks(int64_t n) { return (n + PACK - 1) / PACK; }

struct __attribute__((packed, aligned(1))) Eight {
  uint32_t w[2];
};

__device__ __forceinline__ uint32_t max_of_four_lanes(uint32_t m) {
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const uint32_t u = __shfl_xor(m, o);
    m = m > u ? m : u;
  }
  return m;
}
__device__ __forceinline__ int pack_exponent(uint32_t m) {
  const int e = static_cast<int>((m + 0x30000u) >> 23);
  return e > 7 ? e : 7;
}
// Eight values of a lane, of which the four lanes that share a block give the exponent (all four must be active).
// SIGN: a positive value stays positive.
template <bool SIGN>
__device__ __forceinline__ Eight pack_values(const float (&v)[8], int& e) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t b = __float_as_uint(v[k]) & 0x7fffffffu;
    m = m > b ? m : b;
  }
  m = max_of_four_lanes(m);
  uint32_t q[8];
  if (__builtin_expect(m < 0x7f800000u, 1)) {
    e = pack_exponent(m);
    const float scale = __uint_as_float(static_cast<uint32_t>(260 - e) << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      constexpr float whole = 0x1.8p23f;  // the sum's last bit is 1: it is rounded to an integer, ties to the even one
      const float t = fmaf(v[k], scale, whole);
      q[k] = __float_as_uint(t);
      if (SIGN && t == whole && v[k] > 0.f) q[k] += 1;
    }
  } else {  // (the block's four lanes together)
    m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = __float_as_uint(v[k]) & 0x7fffffffu;
      m = b < 0x7f800000u && b > m ? b : m;
    }
    e = pack_exponent(max_of_four_lanes(m));
    const float scale = __uint_as_float(static_cast<uint32_t>(260 - e) << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      int n = __builtin_isfinite(v[k]) ? static_cast<int>(rintf(v[k] * scale)) : v[k] != v[k] ? -128 : v[k] > 0.f ? 127 : -127;
      if (SIGN && n == 0 && v[k] > 0.f) n = 1;
      q[k] = static_cast<uint32_t>(n);
    }
  }
  Eight r;
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // (the low bytes of four)
    const uint32_t lo = __builtin_amdgcn_perm(q[4 * k + 1], q[4 * k], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[4 * k + 3], q[4 * k + 2], 0x0c0c0400u);
    r.w[k] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return r;
}
// TYPE: what the values must fit (fp32: bf16)
template <int TYPE>
__device__ __forceinline__ void unpack_values(const Eight& p, int e, float (&v)[8]) {
  constexpr float most = TYPE == F16 ? 65504.f : 0x1.fep127f;
  const float step = __uint_as_float(static_cast<uint32_t>(e > 7 ? e - 6 : 1) << 23), low = -128.f * step;
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {  // bytes from -128 on as such from 0 on
    v[k] = fmaf(static_cast<float>(((p.w[k / 4] ^ 0x80808080u) >> (8 * (k % 4))) & 255u), step, low);
    top = fmaxf(top, fabsf(v[k]));
  }
  const float finite = 126.5f * step < most ? 126.5f * step : most;
  if (__builtin_expect(!(top <= finite), 0)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int q = static_cast<int>(p.w[k / 4] << (24 - 8 * (k % 4))) >> 24;
      v[k] = within(static_cast<float>(q) * step, most);
      if (q == 127) v[k] = __builtin_inff();
      if (q == -127) v[k] = -__builtin_inff();
      if (q == -128) v[k] = __builtin_nanf("");
    }
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
// lanes of a block call it together; those past the last column too.  WHOLE: all eight exist.
template <bool WHOLE>
__device__ __forceinline__ void pack_argument(const Epilogue& e, bool relu, int64_t m, int n, int N, const float (&z)[8]) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = WHOLE || n + k < N ? z[k] : 0.f;
  int x;
  const Eight q = relu ? pack_values<true>(v, x) : pack_values<false>(v, x);
  if (!WHOLE && n >= N) return;
  store_eight(e.z8 + m * N + n, q, WHOLE ? 8 : N - n);
  if (n % PACK == 0) e.ze[m * pack_blocks(N) + n / PACK] = static_cast<uint8_t>(x);
}

}  // namespace dense
}  // namespace maloq
