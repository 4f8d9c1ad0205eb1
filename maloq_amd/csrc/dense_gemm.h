#pragma once
// Tiled matrix products of the dense layers (dense.hip): C[m][n] = sum_k A(m, k) B(n, k), with the
// epilogue y = act(C [sa_m sb_n] + bias_n) + residual_mn.
//
// A workgroup of four waves owns a TM x TN tile of C (256 x 256, 128 x 128; 64 or 32 x 128 where rows
// are few), a wave a quarter of it in MFMA tiles of 16 x 16 (256 x 256) or 32 x 32.  Both operands are
// copied global -> LDS by DMA, 128 bytes of the contraction a K step (whole cache lines: with 64
// the requests to L2 were twice as many and its channels three quarters busy, 8192^3 bf16 886 us, 803 so)
// for an operand whose rows run along it (N), 64 rows of it (fp32: 32) for one whose rows run across it
// (TR: the weights of an input gradient, both operands of a weight gradient), which is read back
// transposed (ds_read_b64_tr_b16; fp32: single values, whose rows lie in different banks).  256 x 256: an
// operand's step is 32 KB, five of which are all of the LDS: A of three steps and B of two, in turn.
//
// Software pipeline: a step is two halves.  The MFMAs of each take registers that were read during the
// half before; between them, in an order that is pinned, stand the LDS reads of the next half
// and the copies of step s + 2: A's in the first half (its place held A of step s - 1), B's in the
// second (B of step s).  One barrier a step, before the second half: all waves have read step
// s, and step s + 1 has come.
//
// What bounds it: large products of 16 and 8 bits the power that the card may draw: 8192^3 bf16 of normal
// numbers runs at 1.9 GHz with the matrix units busy 0.77 of the time, a launch 763 to 827 us of twenty in a row (1.33 to
// 1.44 PFLOP/s) and 728 of a hundred, e4m3 405 (2.7) and 367; the library's products, without an epilogue, 780 and 400 of
// twenty; of zeros 605 and 288.  A tile's start takes 2.8 us and
// its epilogue 6.4 (silu 9, gelu 15: the vector units; residual 12) of 80 at k = 4096.  (One workgroup a
// CU that stays, with the next tile's first copies on their way during an epilogue in two free slots,
// was no faster: bf16 840 -> 850 us, e4m3 480 -> 515.)  fp32: splitting the fragments, 44 vector
// instructions to six MFMAs, on one or two waves a SIMD: 8192^3 200 TFLOP/s, the library's fp32 units 154.
//
// Sums are fp32, but for the e4m3 products inside an instruction: the matrix unit adds eight consecutive ones of the
// contraction as whole multiples of 2^-13 of the power of two below the largest, what is smaller cut off
// towards zero, and the eights in fp32 (measured: 256 256 + 2 2 gives 65536 within an eight, 65540 across two).  That is taken:
// sums of 4096 products of normal numbers' e4m3 rows are off by 1.5e-5 in norm, where the operands were rounded by up
// to 2^-4 and a bf16 result is by 1.7e-3, and products without it are the 16-bit ones at half the rate.
//
// What the operands must fulfil (the host sees to it): bases and row strides multiples of 16 bytes,
// the contiguous extent a multiple of 16 bytes.  Rows past the last are the last again (what they
// give is not stored); what lies past the contraction's end comes from a page of zeros.
#include "common.h"
#include "split_bf16.h"

#include <type_traits>

namespace maloq {
namespace dense {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Types of operands and of results.  fp32 products are six bf16 products of floats split in three
// (split_bf16.h); the split is of the fragments, between the products of the tile before.
enum { F32 = 0, BF16 = 1, F16 = 2, E4M3 = 3 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

constexpr int64_t MAX_THREADS = (int64_t(1) << 32) - 1;  // of a launch

__host__ __device__ constexpr int size_of(int type) { return type == F32 ? 4 : (type == E4M3 ? 1 : 2); }

// ------------------------------------------------------------- activations
// fp32 results need more than the hardware's exponential and reciprocal (1 ulp each, the
// exponential's argument rounded too) give; for 16 bits these are four digits more than enough.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (EXACT) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
// 1 - Phi(a), a >= 0, and exp(-a^2 / 2): erfc's scaled form is smooth in t = 1 / (1 + 0.3 a), and a
// polynomial without a constant (fitted here for the relative error: these coefficients are off by at most 2^-21.9
// on 0 .. 14) times the exponential keeps most of the tail's relative accuracy.  In fp32 the product is off by
// 2^-20.8 up to a = 2, 2^-18.5 at 7 and 2^-17 at 13 (the exponential's argument is rounded), by 2^-22 of 1 at most, and
// zero from 13.2 on, below the normal numbers: for results of 16 bits.  Half the instructions of erff, whose two
// ranges a wave takes both.
__device__ __forceinline__ float normal_tail(float a, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.3f, 1.f));
  float p = 0.03556318f;
  p = fmaf(p, t, -0.15676896f);
  p = fmaf(p, t, 0.20566134f);
  p = fmaf(p, t, -0.0530985f);
  p = fmaf(p, t, 0.12827862f);
  p = fmaf(p, t, 0.09999177f);
  p = fmaf(p, t, 0.12074249f);
  p = fmaf(p, t, 0.11962998f);
  e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);
  return p * t * e;
}
template <bool EXACT, int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;  // (NaN stays)
  if constexpr (ACT == ACT_SILU) return z * sigmoid<EXACT>(z);
  if constexpr (ACT == ACT_GELU) {
    if constexpr (EXACT) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    float e;
    const float a = fabsf(z) > 32.f ? 32.f : fabsf(z);  // (beyond, the tail is 0: no infinity times 0; NaN stays)
    return fmaf(-a, normal_tail(a, e), z < 0.f ? 0.f : z);
  }
  return z;
}
// z within +-most; NaN stays
__device__ __forceinline__ float within(float z, float most) { return z > most ? most : (z < -most ? -most : z); }
// Far out the slopes are 0 and 1 to every bit long before the ends to which arguments are brought here: an infinite
// one, which a finite product below or above fp16's range is stored as, makes no 0 times infinity.
template <bool EXACT, int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == ACT_SILU) {
    const float c = within(z, 128.f), p = sigmoid<EXACT>(c);
    return p * (1.f + c * (1.f - p));
  }
  if constexpr (ACT == ACT_GELU) {
    const float c = within(z, 32.f);
    if constexpr (EXACT) return 0.5f * (1.f + erff(c * 0.70710678118654752f)) + c * expf(-0.5f * c * c) * 0.39894228040143268f;
    float e;
    const float tail = normal_tail(fabsf(c), e);
    return fmaf(c * e, 0.39894228040143268f, z < 0.f ? tail : 1.f - tail);
  }
  return 1.f;
}

// ----------------------------------------------------- elements of a type
template <int TYPE>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (TYPE == F32) return static_cast<const float*>(p)[i];
  if constexpr (TYPE == BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (TYPE == F32) static_cast<float*>(p)[i] = v;
  if constexpr (TYPE == BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  if constexpr (TYPE == F16) static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}
// Eight at once, anywhere in memory (16 bytes at any address are one access): as they lie there, and
// as floats.
struct __attribute__((packed, aligned(1))) Loose {
  uint32_t w[4];
};
__device__ __forceinline__ uint4 load_loose(const void* p) {
  const Loose v = *static_cast<const Loose*>(p);
  return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
__device__ __forceinline__ void store_loose(void* p, uint4 v) { *static_cast<Loose*>(p) = {{v.x, v.y, v.z, v.w}}; }

template <int TYPE>
struct Raw8 {
  uint4 q[TYPE == F32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> load_raw8(const void* p, int64_t i) {
  Raw8<TYPE> r;
  const char* q = static_cast<const char*>(p) + i * size_of(TYPE);
  r.q[0] = load_loose(q);
  if constexpr (TYPE == F32) r.q[1] = load_loose(q + 16);
  return r;
}
template <int TYPE>
__device__ __forceinline__ void unpack8(const Raw8<TYPE>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
  if constexpr (TYPE == F32) {
    const uint32_t u[4] = {r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]), v[4 + k] = __uint_as_float(u[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (TYPE == BF16) {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        v[2 * k] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k])));
        v[2 * k + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k] >> 16)));
      }
    }
  }
}
template <int TYPE>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  unpack8<TYPE>(load_raw8<TYPE>(p, i), v);
}
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> pack8(const float (&v)[8]) {
  Raw8<TYPE> r;
  if constexpr (TYPE == F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      r.q[h] = make_uint4(__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (TYPE == BF16) {
        w[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
      } else {
        w[k] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * k])) |
               static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * k + 1]))) << 16;
      }
    }
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
  const Raw8<TYPE> r = pack8<TYPE>(v);
  char* q = static_cast<char*>(p) + i * size_of(TYPE);
  store_loose(q, r.q[0]);
  if constexpr (TYPE == F32) store_loose(q + 16, r.q[1]);
}
// The first `have` of eight (the others read as zeros).
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> load_part8(const void* p, int64_t i, int have) {
  if (have >= 8) return load_raw8<TYPE>(p, i);
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < have ? load1<TYPE>(p, i + k) : 0.f;
  return pack8<TYPE>(v);
}
template <int TYPE>
__device__ __forceinline__ void store_part8(void* p, int64_t i, const float (&v)[8], int have) {
  if (have >= 8) {
    store8<TYPE>(p, i, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < have) store1<TYPE>(p, i + k, v[k]);
  }
}

// --------------------------------------------------------------- epilogue
struct Epilogue {
  const float *sa, *sb;   // scales of A's and B's rows (both or neither)
  const void* bias;       // [N] or null
  const void* res;        // [M][ldr] or null
  int64_t ldr;
  void* out;              // [M][ldo]
  int64_t ldo;
  void* z;                // [M][N]: what the activation is given, or null
  int act;
};

// f(0), .., f(N - 1), as constants (a loop whose body holds others is not unrolled at any size)
template <int N, class F>
__device__ __forceinline__ void each(const F& f) {
  if constexpr (N > 1) each<N - 1>(f);
  f(std::integral_constant<int, N - 1>{});
}
// f(activation as a constant)
template <class F>
__device__ __forceinline__ void with_act(int act, const F& f) {
  if (act == ACT_NONE) f(std::integral_constant<int, ACT_NONE>{});
  if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
  if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>{});
}

// Eight columns from n on of row m, of which `have` exist: v sb + bias, of the lane's columns (ones and
// zeros where there are none), activation, residual.
template <int OUT, int ACT>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t m, int n, int N, int have, float (&v)[8],
                                        const float (&bias)[8], const float (&sb)[8], const Raw8<OUT>& res) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = fmaf(v[k], sb[k], bias[k]);
  if (e.z) store_part8<OUT>(e.z, m * N + n, v, have);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = act_fwd<OUT == F32, ACT>(v[k]);
  if (e.res) {
    float r[8];
    unpack8<OUT>(res, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += r[k];
  }
  store_part8<OUT>(e.out, m * e.ldo + n, v, have);
}
// The same at the edge of the result.
template <int OUT>
__device__ __forceinline__ void finish_edge(const Epilogue& e, int64_t m, int n, int N, float (&v)[8], const float (&bias)[8],
                                            const float (&sb)[8]) {
  Raw8<OUT> res{};
  if (e.res) res = load_part8<OUT>(e.res, m * e.ldr + n, N - n);
  with_act(e.act, [&](auto act) { finish8<OUT, decltype(act)::value>(e, m, n, N, N - n, v, bias, sb, res); });
}
// (loads without a branch each, so that they are in flight together)
template <int OUT, bool SCALED>
__device__ __forceinline__ void columns8(const Epilogue& e, int n, int N, float (&bias)[8], float (&sb)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) bias[k] = 0.f, sb[k] = 1.f;
  if (e.bias) {
#pragma unroll
    for (int k = 0; k < 8; ++k) bias[k] = load1<OUT>(e.bias, n + k < N ? n + k : N - 1);
  }
  if constexpr (SCALED) {
#pragma unroll
    for (int k = 0; k < 8; ++k) sb[k] = e.sb[n + k < N ? n + k : N - 1];
  }
}
// ----------------------------------------------------------------- kernel
struct GemmArgs {
  const char *a, *b;
  int64_t lda, ldb;     // bytes from one row to the next
  int M, N, K;          // K: elements
  int full, tail;       // tiles with the whole contraction to one workgroup; tiles after them, split
  int splits;           // parts of a split tile's contraction
  int steps;            // K steps of a part
  float* part;          // [splits][tail][TM][TN]
  Epilogue e;
};

static __device__ __constant__ uint4 zero_page[4] = {};

// T rows (columns) of an operand, dealt to W waves
template <int T, int W>
struct Geo {
  static constexpr int SLOT = T * 128;       // bytes of a step
  static constexpr int P = SLOT / 1024 / 4;  // 1 KB pieces that a wave copies
  static constexpr int OWN = T / W;          // of a wave
};
// A tile and its waves
template <int TM, int TN>
struct Tile {
  static constexpr int WN = TM >= 128 ? 2 : 4, WM = 4 / WN;
  using A = Geo<TM, WM>;
  using B = Geo<TN, WN>;
  static constexpr int LDS = 3 * A::SLOT + 2 * B::SLOT;
  static constexpr int PITCH = B::OWN * 4 + 16;  // bytes of a row of the epilogue's strip
  static constexpr int GROUPS = LDS > 80 * 1024 ? 1 : (LDS > 53 * 1024 ? 2 : 3);  // a CU
};

// Accumulators of an MI x MI tile
template <int MI>
struct Acc {
  typedef float type __attribute__((ext_vector_type(MI * MI / 64)));
};
// 16 x 16 products of 64 bytes of each row (8 bits: 128).  In asm, which ties the result to the
// accumulator: left to the compiler, which does not see how to place 64 of them, a hundred copies a
// K step.  It does not see either that a product's reader and a value's product have to wait: within
// a loop of them those are the same products a step later, and settle() stands before and behind it.
template <int IN, class C, class F>
__device__ __forceinline__ void mfma_in_place(C& c, const F& a, const F& b) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (IN == BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  if constexpr (IN == F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  if constexpr (IN == E4M3) asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
#endif
}
// Eight accumulators are where they are, for products to come and for readers of those before.
__device__ __forceinline__ void settle(f32x4 (&c)[8]) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
               : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]));
#endif
}
template <class C>
__device__ __forceinline__ void settle(C&) {}
template <int IN>
__device__ __forceinline__ f32x4 mfma16(const s16x8& a, const s16x8& b, const f32x4& c) {
  if constexpr (IN == F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int IN>
__device__ __forceinline__ f32x16 mfma16(const s16x8& a, const s16x8& b, const f32x16& c) {
  if constexpr (IN == F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight floats in three planes.  FIX: an infinity as (+-1, 0, +-inf), which gives infinity with the
// other operand's leading plane; without, it gives NaN.
struct Planes {
  s16x8 p[3];
};
template <bool FIX>
__device__ __forceinline__ Planes planes(const i32x4& lo, const i32x4& hi) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = __int_as_float(lo[k]), v[4 + k] = __int_as_float(hi[k]);
  uint4 pl[3];
  split8(v, pl);
  if constexpr (FIX) {
    uint32_t* w = reinterpret_cast<uint32_t*>(pl);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int sh = 16 * (k & 1);
      const uint32_t sign = v[k] < 0.f ? 0x8000u : 0u, keep = ~(0xffffu << sh);
      if (__builtin_isinf(v[k])) {
        w[k >> 1] = (w[k >> 1] & keep) | (sign | 0x3f80u) << sh;
        w[4 + (k >> 1)] &= keep;
        w[8 + (k >> 1)] = (w[8 + (k >> 1)] & keep) | (sign | 0x7f80u) << sh;
      }
    }
  }
  Planes r;
#pragma unroll
  for (int i = 0; i < 3; ++i) r.p[i] = __builtin_bit_cast(s16x8, pl[i]);
  return r;
}

typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)((__attribute__((address_space(3))) const char*)p));
}

template <class P>
__device__ __forceinline__ P* uniform(P* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<P*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// One operand: how this lane copies it into a slot and reads it back.
// MI: rows of an MFMA tile.
template <int IN, int T, int W, bool TR, int MI>
struct Operand {
  using G = Geo<T, W>;
  static constexpr int TI = G::OWN / MI;
  static constexpr int ES = size_of(IN), KE = 128 / ES;
  static_assert(!TR || ES > 1, "8-bit operands run along the contraction");
  const char* base;     // the tile's first row (TR: column) at the contraction's start
  int64_t kstep;
  unsigned off[G::P];   // of a piece's 16 bytes from base + the step's offset
  int kel[2];           // element of the step's contraction that they start at: of even and of odd pieces; TR: of the first
  int rd[TR && TI > 4 ? TI : 4];  // where a lane's fragments lie in a slot: TR: of MFMA tile t; else of part ks of the step

  // rows: the operand's extent across the contraction; r0: the tile's first
  __device__ __forceinline__ void init(const char* p, int64_t ld, int rows, int r0, int wave, int lane, int own) {
    if constexpr (!TR) {
      // a row's eight 16-byte chunks lie XORed with (row / 2) % 8: the reads of any 16 consecutive
      // rows then hit all banks once
      base = uniform(p + static_cast<int64_t>(r0) * ld);
      kstep = 128;
#pragma unroll
      for (int j = 0; j < G::P; ++j) {
        int r = (wave * G::P + j) * 8 + (lane >> 3);
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        if (j < 2) kel[j] = c * (16 / ES);
        r = r0 + r < rows ? r : rows - 1 - r0;
        off[j] = static_cast<unsigned>(r * ld + c * 16);
      }
#pragma unroll
      for (int ks = 0; ks < MI / 8; ++ks)
        rd[ks] = (own * G::OWN + lane % MI) * 128 + (((64 / MI * ks + lane / MI) ^ ((lane >> 1) & 7)) << 4);
    } else {
      // 16 bits: chunk c of contraction row r lies at c ^ 4 (r % 4): the four rows that a transposed
      // read of 16 lanes takes lie in different banks.  (16-row tiles: those of the next 16 lanes, eight rows
      // on, in the same.  With the halves of 64 bytes swapped there none do, and each tile of an operand
      // needs an address of its own: 4 to 7 % slower.)
      constexpr int CH = T * ES / 16;  // chunks of a row
      base = uniform(p + static_cast<int64_t>(r0) * ES);
      kstep = KE * ld;
      const int last = ((rows - r0) * ES + 15) / 16 - 1;  // of the row's chunks
#pragma unroll
      for (int j = 0; j < G::P; ++j) {
        const int at = (wave * G::P + j) * 64 + lane, r = at / CH;
        int c = ES == 2 ? (at % CH) ^ ((r & 3) << 2) : at % CH;
        c = c < last ? c : last;
        if (j == 0) kel[0] = kel[1] = r;
        off[j] = static_cast<unsigned>(r * ld + c * 16);
      }
      const int g = lane >> 4, aa = lane & 3, kk = (lane >> 2) & 3;
#pragma unroll
      for (int t = 0; t < TI; ++t) {
        if constexpr (ES == 4)
          rd[t] = (4 * (lane >> 5) * T + own * G::OWN + 32 * t + (lane & 31)) * 4;
        else if constexpr (MI == 32)
          rd[t] = (8 * (g >> 1) + kk) * (T * ES) + (2 * (g & 1) + (aa >> 1)) * 16 + (aa & 1) * 8 + 64 * ((own * TI + t) ^ kk);
        else
          rd[t] = (8 * g + kk) * (T * ES) + (2 * (t & 1) + (aa >> 1)) * 16 + (aa & 1) * 8 + 64 * (((own * TI + t) >> 1) ^ kk);
      }
    }
  }
  __device__ __forceinline__ int element(int j) const { return TR ? kel[0] + j * (64 * 16 / (T * ES)) : kel[j & 1]; }
  // where K step `step` starts
  __device__ __forceinline__ const char* source(int step) const { return base + step * kstep; }
  // Piece j of a K step to the slot at LDS address `lds`.  WHOLE: none of it
  // lies past the contraction's end; else left: its elements from the step's first on.  (s_nop: a
  // wait state between the scalar write of m0 and its use.  The compiler keeps nothing in m0, and warns.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  template <bool WHOLE>
  __device__ __forceinline__ void copy(int j, unsigned lds, int wave, const char* p, int left) const {
    const unsigned at = __builtin_amdgcn_readfirstlane(lds + (wave * G::P + j) * 1024);
    if constexpr (WHOLE) {
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[j]), "s"(p), "s"(at) : "memory", "m0");
    } else {
      const char* q = element(j) < left ? p + off[j] : reinterpret_cast<const char*>(&zero_page[0]);
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(q), "s"(at) : "memory", "m0");
    }
  }
#pragma clang diagnostic pop
  // 16 bytes of a lane's fragment of MFMA tile t.  16-bit: of elements 512 / MI ks .. of the step, the
  // (lane / MI)-th eight; 8-bit and fp32: chunk 2 ks + lane / 32 of it (the same elements of both
  // operands, in the same order)
  __device__ __forceinline__ i32x4 read(const char* slot, int t, int ks) const {
    if constexpr (TR && ES == 4) {  // (the elements that a row's chunk 2 ks + lane / 32 holds)
      const int* p = reinterpret_cast<const int*>(slot + rd[t]) + 8 * ks * T;
      return i32x4{p[0], p[T], p[2 * T], p[3 * T]};
    } else if constexpr (TR) {
      const char* p = slot + rd[t] + (512 / MI * ks) * (T * ES);
      const s16x4 a = read_tr(p), b = read_tr(p + 4 * (T * ES));
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const i32x4*>(slot + rd[ks] + t * (MI * 128));
    }
  }
};

// Item `at` of `count` in an order in which the workgroups that run at the same time on one XCD
// (they are dealt out over the eight in turn) have consecutive ones; at least `count` for none.
__device__ __forceinline__ unsigned dealt(unsigned at, unsigned count) { return (at & 7) * ((count + 7) >> 3) + (at >> 3); }
// First row and column of tile `id`: runs of 8 tiles down, then across, so that consecutive ones share rows and columns.
template <int TM, int TN>
__device__ __forceinline__ void tile_at(unsigned id, int mt, int nt, int& m0, int& n0) {
  constexpr unsigned GM = 8;
  const unsigned group = id / (GM * nt), first = group * GM;
  const unsigned high = mt - first < GM ? mt - first : GM;
  const unsigned in_group = id - group * (GM * nt);
  m0 = (first + in_group % high) * TM;
  n0 = in_group / high * TN;
}

// EVEN: the contraction is whole steps; else every copy of a 256 x 256 tile selects its source (8192 x 4096 x 16384
// bf16 778 us, 8192 x 4088 x 16384 900; the smaller tiles' loops do so in the last steps alone)
template <int IN, int OUT, int TM, int TN, bool TRA, bool TRB, bool EVEN>
__global__ __launch_bounds__(256, (Tile<TM, TN>::GROUPS)) void gemm_kernel(GemmArgs a) {
  using G = Tile<TM, TN>;
  using GA = typename G::A;
  using GB = typename G::B;
  // 256 x 256: MFMAs of 16 x 16 x 32 (8 bits: x 128).  They are as fast as those of 32 x 32 x 16 (64) and take and
  // give back half the accumulators, and what bounds these products is power: 8192^3 bf16 of
  // normal numbers 805 us -> 760, of zeros, at full clock, 600 -> 605.
  constexpr int MI = IN != F32 && TM == 256 ? 16 : 32;
  using A = Operand<IN, TM, G::WM, TRA, MI>;
  using B = Operand<IN, TN, G::WN, TRB, MI>;
  constexpr int KE = A::KE, TI = A::TI, TJ = B::TI, KS = MI / 16;  // KS: parts of half a step
  __shared__ alignas(1024) char smem[G::LDS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;

  const int mt = (a.M + TM - 1) / TM, nt = (a.N + TN - 1) / TN;
  const unsigned full8 = (a.full + 7) & ~7;
  const bool split = blockIdx.x >= full8;
  const unsigned parts = a.tail * a.splits;
  const unsigned item = split ? dealt(blockIdx.x - full8, parts) : dealt(blockIdx.x, a.full);
  if (item >= (split ? parts : a.full)) return;  // whole workgroup, before any barrier
  const unsigned part = split ? item / a.tail : 0, of_tail = split ? item - part * a.tail : 0;
  int m0, n0;
  tile_at<TM, TN>(split ? a.full + of_tail : item, mt, nt, m0, n0);
  m0 = __builtin_amdgcn_readfirstlane(m0), n0 = __builtin_amdgcn_readfirstlane(n0);

  const int ksteps = (a.K + KE - 1) / KE;
  const int kb = __builtin_amdgcn_readfirstlane(split ? part * a.steps : 0);
  const int most = split ? a.steps : ksteps;
  const int kn = kb + most < ksteps ? most : (ksteps > kb ? ksteps - kb : 0);
  const int nsteps = __builtin_amdgcn_readfirstlane(kn);
  // of these, the first ones that end within the contraction
  const int whole = __builtin_amdgcn_readfirstlane(kb + kn < ksteps || a.K % KE == 0 ? kn : kn - 1);

  const int wm = wave / G::WN, wn = wave % G::WN;
  A oa;
  B ob;
  oa.init(a.a, a.lda, a.M, m0, wave, lane, wm);
  ob.init(a.b, a.ldb, a.N, n0, wave, lane, wn);
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) char*)smem));

  typename Acc<MI>::type acc[TI][TJ];
  const std::false_type any{};
  const std::true_type inside{};

  // What the epilogue needs of the lane's columns and rows.  Fetched before the products; in 8 bits
  // and of fp32 results, where registers are short, after them.
  constexpr bool EARLY = IN != E4M3 && OUT != F32 && MI == 32;
  constexpr int LPR = GB::OWN / 8;  // lanes of a row of a strip
  constexpr int RS = 64 / LPR, ROWS = 32 / RS;  // rows of a strip at a time, and how often
  // (a tile that lies inside: without a test a row; else rows past the last load that one's again)
  const bool inner = m0 + TM <= a.M && n0 + TN <= a.N;
  const int nw = n0 + wn * GB::OWN, past = nw + (lane % LPR) * 8 + 8 - a.N;
  // (columns that end within a lane's eight: the last eight, some of them the lane's before it too)
  const int cl = (lane % LPR) * 8 - (!split && past > 0 && past < 8 && a.N >= nw + 8 ? past : 0), n = nw + cl;
  float bias[8], sb[8], sa[TI];
  Raw8<OUT> res[ROWS];
  auto fetch_residual = [&](auto all, int i) __attribute__((always_inline)) {
    constexpr bool ALL = decltype(all)::value;
    const int64_t m = m0 + wm * GA::OWN + 32 * i + lane / LPR;
    if (!ALL && n + 8 > a.N) return;
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int64_t r = m + u * RS;
      res[u] = load_raw8<OUT>(a.e.res, (ALL || r < a.M ? r : a.M - 1) * a.e.ldr + n);
    }
  };
  auto fetch = [&] {
    if (!split) columns8<OUT, IN == E4M3>(a.e, n, a.N, bias, sb);
    if constexpr (IN == E4M3) {
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int m = m0 + wm * GA::OWN + MI * i + lane % MI;
        sa[i] = a.e.sa[m < a.M ? m : a.M - 1];
      }
    }
    if (!split && a.e.res) {
      if (inner)
        fetch_residual(inside, 0);
      else
        fetch_residual(any, 0);
    }
  };
  if (EARLY) fetch();

  struct Frags {
    i32x4 a[KS][TI], b[KS][TJ];
  };
  constexpr int READS = KS * (TI + TJ), PRODUCTS = (IN == E4M3 || IN == F32 ? 1 : KS) * TI * TJ;  // of half a step
  struct Source {
    const char* p;
    int left;
  };
  // (past the end: the last again, not read)
  auto source_a = [&](int s) -> Source {
    const int k = kb + (s < nsteps ? s : nsteps - 1);
    return {oa.source(k), a.K - k * KE};
  };
  auto source_b = [&](int s) -> Source {
    const int k = kb + (s < nsteps ? s : nsteps - 1);
    return {ob.source(k), a.K - k * KE};
  };
  // unit u of half h of the step in the slots
  auto read = [&](Frags& f, const char* slot_a, const char* slot_b, int h, int u) {
    const int ks = u / (TI + TJ), t = u % (TI + TJ);
    if (t < TJ)
      f.b[ks][t] = ob.read(slot_b, t, KS * h + ks);
    else
      f.a[ks][t - TJ] = oa.read(slot_a, t - TJ, KS * h + ks);
  };
  // (B's tile is the MFMA's first operand: a lane then holds four consecutive columns of a row of C)
  auto product = [&](const Frags& f, int q) {
    if constexpr (IN == E4M3 && MI == 32) {
      const int i = q / TJ, j = i % 2 ? TJ - 1 - q % TJ : q % TJ;
      const i32x8 x = __builtin_shufflevector(f.b[0][j], f.b[1][j], 0, 1, 2, 3, 4, 5, 6, 7);
      const i32x8 y = __builtin_shufflevector(f.a[0][i], f.a[1][i], 0, 1, 2, 3, 4, 5, 6, 7);
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, acc[i][j], 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);  // (unit block scales)
    } else if constexpr (IN != F32 && IN != E4M3) {
      const int ks = q / (TI * TJ), i = q / TJ % TI, j = i % 2 ? TJ - 1 - q % TJ : q % TJ;
      if constexpr (MI == 16)
        mfma_in_place<IN>(acc[i][j], f.b[ks][j], f.a[ks][i]);
      else
        acc[i][j] = mfma16<IN>(__builtin_bit_cast(s16x8, f.b[ks][j]), __builtin_bit_cast(s16x8, f.a[ks][i]), acc[i][j]);
    }
  };
  // Products of `now`, reads of half h of the step in slots ra, rb into `next` (the first three quarters
  // of the time, so that the last has come when the next half asks for it), copies by `copy`.
  auto half = [&](auto pieces, const Frags& now, Frags& next, int ra, int rb, int h, auto&& copy) {
    constexpr int P = decltype(pieces)::value;
    constexpr int QR = PRODUCTS >= 4 ? PRODUCTS * 3 / 4 : 1;
    each<PRODUCTS>([&](auto at) __attribute__((always_inline)) {
      constexpr int q = decltype(at)::value;
      if constexpr (q < QR) {
#pragma unroll
        for (int u = q * READS / QR; u < (q + 1) * READS / QR; ++u) read(next, smem + ra, smem + rb, h, u);
      }
#pragma unroll
      for (int j = q * P / PRODUCTS; j < (q + 1) * P / PRODUCTS; ++j) copy(j);
      product(now, q);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  Frags f0, f1;
  constexpr int B0 = 3 * GA::SLOT;  // B's slots stand behind A's
  int xa = 0, xb = B0;              // slots of the step's A and B
  auto step = [&](auto is_whole, int s) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    // the next step's, and of A after that
    const int ya = xa == 2 * GA::SLOT ? 0 : xa + GA::SLOT, yb = 2 * B0 + GB::SLOT - xb, za = ya == 2 * GA::SLOT ? 0 : ya + GA::SLOT;
    const Source ca = source_a(s + 2), cb = source_b(s + 2);
    half(std::integral_constant<int, GA::P>{}, f0, f1, xa, xb, 1, [&](int j) {
      oa.template copy<WHOLE>(j, lds0 + za, wave, ca.p, ca.left);
    });
    // this wave's reads of step s and its copies of step s + 1 done (A of s + 2 in flight); then all waves'
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(GA::P) : "memory");
    half(std::integral_constant<int, GB::P>{}, f1, f0, ya, yb, 0, [&](int j) {
      ob.template copy<WHOLE>(j, lds0 + xb, wave, cb.p, cb.left);
    });
    xa = ya, xb = yb;
  };

  // 8 bits of 16 x 16 x 128: a product takes the step's whole 128 bytes, so that the halves are A's rows,
  // the lower and the upper half of the wave's tiles.  A tile of B is read for the next step as soon as its
  // last product of this one is under way, and A's lower half during the second.
  struct Frags8 {
    i32x8 a[TI], b[TJ];
  };
  auto read_b8 = [&](Frags8& f, int slot, int t) __attribute__((always_inline)) {
    f.b[t] = __builtin_shufflevector(ob.read(smem + slot, t, 0), ob.read(smem + slot, t, 1), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read_a8 = [&](Frags8& f, int slot, int t) __attribute__((always_inline)) {
    f.a[t] = __builtin_shufflevector(oa.read(smem + slot, t, 0), oa.read(smem + slot, t, 1), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto step8 = [&](auto is_whole, Frags8& f, int s) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    constexpr int H = TI / 2, N = H * TJ;
    const int ya = xa == 2 * GA::SLOT ? 0 : xa + GA::SLOT, yb = 2 * B0 + GB::SLOT - xb, za = ya == 2 * GA::SLOT ? 0 : ya + GA::SLOT;
    const Source ca = source_a(s + 2), cb = source_b(s + 2);
    each<2 * N>([&](auto at) __attribute__((always_inline)) {
      constexpr int h = decltype(at)::value / N, q = decltype(at)::value % N, j = q / H, i = H * h + (j % 2 ? H - 1 - q % H : q % H);
      if constexpr (h == 1 && q == 0)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(GA::P) : "memory");
#pragma unroll
      for (int c = q * GA::P / N; c < (q + 1) * GA::P / N; ++c) {
        if (h == 0)
          oa.template copy<WHOLE>(c, lds0 + za, wave, ca.p, ca.left);
        else
          ob.template copy<WHOLE>(c, lds0 + xb, wave, cb.p, cb.left);
      }
      mfma_in_place<E4M3>(acc[i][j], f.b[j], f.a[i]);
      if constexpr (h == 0 && q % H == 1 && q / H < H) read_a8(f, xa, H + q / H);
      if constexpr (h == 1 && q % H == 1 && q / H < H) read_a8(f, ya, q / H);
      if constexpr (h == 1 && q % H == H - 1) read_b8(f, yb, j);
      __builtin_amdgcn_sched_barrier(0);
    });
    xa = ya, xb = yb;
  };

  // fp32: the products of a half take planes that were split during the half before, from registers
  // that were read during the one before that; the barrier stands before the first half.
  struct Split {
    Planes a[TI], b[TJ];
  };
  auto split_all = [&](auto fix, const Frags& f, Split& p) __attribute__((always_inline)) {
    constexpr bool FIX = decltype(fix)::value;
#pragma unroll
    for (int j = 0; j < TJ; ++j) p.b[j] = planes<FIX>(f.b[0][j], f.b[1][j]);
#pragma unroll
    for (int i = 0; i < TI; ++i) p.a[i] = planes<FIX>(f.a[0][i], f.a[1][i]);
  };
  auto half32 = [&](auto fix, const Split& now, Split& next, const Frags& split_these) __attribute__((always_inline)) {
    split_all(fix, split_these, next);
    each<SPLIT_PRODUCTS * TI * TJ>([&](auto at) {
      constexpr int q = decltype(at)::value, p = q / (TI * TJ), i = q / TJ % TI, j = q % TJ;
      acc[i][j] = mfma16<BF16>(now.b[j].p[split_b(p)], now.a[i].p[split_a(p)], acc[i][j]);
    });
    constexpr int N = SPLIT_PRODUCTS * TI * TJ, V = (44 * (TI + TJ) + N - 1) / N;  // vector instructions to one product
#pragma unroll
    for (int q = 0; q < N; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    }
  };
  Split p0, p1;
  auto step32 = [&](auto is_whole, auto fix, int s) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    const int ya = xa == 2 * GA::SLOT ? 0 : xa + GA::SLOT, yb = 2 * B0 + GB::SLOT - xb;
    const Source ca = source_a(s + 3), cb = source_b(s + 2);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(GA::P) : "memory");
#pragma unroll
    for (int u = 0; u < READS; ++u) read(f0, smem + ya, smem + yb, 0, u);
#pragma unroll
    for (int j = 0; j < GB::P; ++j) ob.template copy<WHOLE>(j, lds0 + xb, wave, cb.p, cb.left);
    half32(fix, p0, p1, f1);
#pragma unroll
    for (int u = 0; u < READS; ++u) read(f1, smem + ya, smem + yb, 1, u);
#pragma unroll
    for (int j = 0; j < GA::P; ++j) oa.template copy<WHOLE>(j, lds0 + xa, wave, ca.p, ca.left);
    half32(fix, p1, p0, f0);
    xa = ya, xb = yb;
  };

  auto contract = [&](auto fix) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int r = 0; r < MI * MI / 64; ++r) acc[i][j][r] = 0.f;
    if (nsteps <= 0) return;
    xa = 0, xb = B0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Source ca = source_a(s), cb = source_b(s);
#pragma unroll
      for (int j = 0; j < GA::P; ++j) oa.template copy<false>(j, lds0 + s * GA::SLOT, wave, ca.p, ca.left);
#pragma unroll
      for (int j = 0; j < GB::P; ++j) ob.template copy<false>(j, lds0 + B0 + s * GB::SLOT, wave, cb.p, cb.left);
    }
    int s = 0;
    if constexpr (IN == F32) {
      const Source ca = source_a(2);
#pragma unroll
      for (int j = 0; j < GA::P; ++j) oa.template copy<false>(j, lds0 + 2 * GA::SLOT, wave, ca.p, ca.left);
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * GA::P + GB::P) : "memory");
#pragma unroll
      for (int u = 0; u < READS; ++u) read(f0, smem, smem + B0, 0, u);
#pragma unroll
      for (int u = 0; u < READS; ++u) read(f1, smem, smem + B0, 1, u);
      split_all(fix, f0, p0);
      for (; s + 3 < whole; ++s) step32(inside, fix, s);
      for (; s < nsteps; ++s) step32(any, fix, s);
    } else {
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(GA::P + GB::P) : "memory");
      if constexpr (IN == E4M3 && MI == 16) {
        static_assert(GA::P == GB::P, "copies by A's count");
        Frags8 f;
        each<TJ>([&](auto t) __attribute__((always_inline)) { read_b8(f, B0, decltype(t)::value); });
        each<TI / 2>([&](auto t) __attribute__((always_inline)) { read_a8(f, 0, decltype(t)::value); });
        each<TI>([&](auto i) __attribute__((always_inline)) { settle(acc[decltype(i)::value]); });
        for (; s < nsteps; ++s) step8(std::integral_constant<bool, EVEN>{}, f, s);
        each<TI>([&](auto i) __attribute__((always_inline)) { settle(acc[decltype(i)::value]); });
        return;
      }
#pragma unroll
      for (int u = 0; u < READS; ++u) read(f0, smem, smem + B0, 0, u);
      if constexpr (MI == 16) {  // one loop, so that the accumulators have one place
        each<TI>([&](auto i) __attribute__((always_inline)) { settle(acc[decltype(i)::value]); });
        for (; s < nsteps; ++s) step(std::integral_constant<bool, EVEN>{}, s);
        each<TI>([&](auto i) __attribute__((always_inline)) { settle(acc[decltype(i)::value]); });
      } else {
        for (; s + 2 < whole; ++s) step(inside, s);
        for (; s < nsteps; ++s) step(any, s);
      }
    }
  };
  contract(any);
  if constexpr (IN == F32) {
    // Sums that are not finite are formed again, with infinities split so that they give infinity.
    float bad = 0.f;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = not_finite(bad, acc[i][j][r]);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (the slots are free: the vote's place)
    int* votes = reinterpret_cast<int*>(smem);
    if (lane == 0) votes[wave] = 0;
    if (bad != bad) votes[wave] = 1;
    __syncthreads();
    const int again = votes[0] | votes[1] | votes[2] | votes[3];
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(again)) contract(inside);
  }
  if (!EARLY) fetch();
  // no copy in flight, no wave still reading: the slots become the epilogue's strips
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // A wave's 32 rows of its columns at a time through LDS, so that a lane gets eight consecutive
  // columns and up to 256 bytes of a row are stored together.  One wave a SIMD hides no
  // latency: the rows of a pass are in flight together, the residual's next pass with them.
  char* strip = smem + wave * (32 * G::PITCH);
  static_assert(4 * 32 * G::PITCH <= G::LDS, "the strips fit the slots");
  char* mine = strip + (lane / LPR) * G::PITCH + cl * 4;
#pragma unroll 1
  for (int i = 0; i < GA::OWN / 32; ++i) {
    each<GA::OWN / 32>([&](auto tile) {
      constexpr int I = decltype(tile)::value;
      if (i != I) return;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        if constexpr (MI == 32) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4 v = {acc[I][j][4 * q], acc[I][j][4 * q + 1], acc[I][j][4 * q + 2], acc[I][j][4 * q + 3]};
            if constexpr (IN == E4M3) v = v * sa[I];
            *reinterpret_cast<f32x4*>(strip + (lane & 31) * G::PITCH + (32 * j + 8 * q + 4 * (lane >> 5)) * 4) = v;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            f32x4 v = acc[2 * I + q][j];
            if constexpr (IN == E4M3) v = v * sa[2 * I + q];
            *reinterpret_cast<f32x4*>(strip + (16 * q + (lane & 15)) * G::PITCH + (16 * j + 4 * (lane >> 4)) * 4) = v;
          }
        }
      }
    });
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int64_t m = m0 + wm * GA::OWN + 32 * i + lane / LPR;
    if (split) {
      float* p = a.part + (static_cast<int64_t>(item) * TM + (m - m0)) * TN + (n - n0);
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const f32x4 v0 = *reinterpret_cast<const f32x4*>(mine + u * RS * G::PITCH);
        const f32x4 v1 = *reinterpret_cast<const f32x4*>(mine + u * RS * G::PITCH + 16);
        if (m + u * RS >= a.M || n >= a.N) continue;
        *reinterpret_cast<f32x4*>(p + u * RS * TN) = v0;
        *reinterpret_cast<f32x4*>(p + u * RS * TN + 4) = v1;
      }
    } else {
      const int have = a.N - n;
      auto rows = [&](auto all) __attribute__((always_inline)) {
        constexpr bool ALL = decltype(all)::value;
        if (OUT == F32 && a.e.res && i > 0) fetch_residual(all, i);
        Raw8<OUT> now[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) now[u] = res[u];
        if (OUT != F32 && a.e.res && i + 1 < GA::OWN / 32) fetch_residual(all, i + 1);
        if (!ALL && have < 8) return;
        with_act(a.e.act, [&](auto act) {
#pragma unroll
          for (int u = 0; u < ROWS; ++u) {
            float x[8];
            if constexpr (ALL) {
              const f32x4* at = reinterpret_cast<const f32x4*>(mine + u * RS * G::PITCH);
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = at[k / 4][k % 4];
            } else {
              const float* at = reinterpret_cast<const float*>(mine + u * RS * G::PITCH);
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = at[k];
            }
            if (ALL || m + u * RS < a.M) finish8<OUT, decltype(act)::value>(a.e, m + u * RS, n, a.N, 8, x, bias, sb, now[u]);
          }
        });
      };
      if (inner) {
        rows(inside);
      } else {
        rows(any);
        if (have > 0 && have < 8) {  // (a wave's only columns)
#pragma unroll 1
          for (int u = 0; u < ROWS && m + u * RS < a.M; ++u) {
            const f32x4* at = reinterpret_cast<const f32x4*>(mine + u * RS * G::PITCH);
            float x[8] = {at[0][0], at[0][1], at[0][2], at[0][3], at[1][0], at[1][1], at[1][2], at[1][3]};
            finish_edge<OUT>(a.e, m + u * RS, n, a.N, x, bias, sb);
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Sums of the parts of the split tiles, in a fixed order, and the epilogue: a thread has eight columns of
// every LANES-th part, a block 2048 / LANES values.
template <int OUT, int TM, int TN, bool SCALED, int LANES>
__global__ __launch_bounds__(256) void gemm_sum_kernel(GemmArgs a) {
  constexpr int G = 256 / LANES, PER = TM * TN / 8 / G;
  __shared__ float sums[LANES > 1 ? LANES - 1 : 1][LANES > 1 ? G : 1][9];
  const unsigned of_tail = blockIdx.x / PER, at = (blockIdx.x % PER) * G + threadIdx.x % G;
  const int sub = threadIdx.x / G;
  int m0, n0;
  tile_at<TM, TN>(a.full + of_tail, (a.M + TM - 1) / TM, (a.N + TN - 1) / TN, m0, n0);
  const int r = at / (TN / 8), c = at % (TN / 8) * 8;
  const bool mine = m0 + r < a.M && n0 + c < a.N;
  float bias[8], sb[8], v[8] = {};
  if (mine) {
    columns8<OUT, SCALED>(a.e, n0 + c, a.N, bias, sb);
    const int64_t each = static_cast<int64_t>(a.tail) * TM * TN;
    const float* p = a.part + (static_cast<int64_t>(of_tail) * TM + r) * TN + c;
#pragma unroll 4
    for (int s = sub; s < a.splits; s += LANES) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * each), y = *reinterpret_cast<const f32x4*>(p + s * each + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k], v[4 + k] += y[k];
    }
  }
  if constexpr (LANES > 1) {
    if (sub > 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[sub - 1][threadIdx.x % G][k] = v[k];
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int l = 0; l + 1 < LANES; ++l)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += sums[l][threadIdx.x][k];
  }
  if (mine) finish_edge<OUT>(a.e, m0 + r, n0 + c, a.N, v, bias, sb);
}

// tile: rows of C; below 128 only where both operands' rows run along the contraction, 256 not in fp32
template <int IN, int OUT, bool TRA, bool TRB>
void launch_gemm(const GemmArgs& a, int tile, void* stream) {
  const unsigned grid = ((a.full + 7) & ~7) + ((a.tail * a.splits + 7) & ~7);
  const unsigned sums = a.tail * (tile * (tile == 256 ? 256 : 128) / 2048);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define MALOQ_GEMM(TM, TN, EVEN)                                                                  \
  if (tile == TM) {                                                                            \
    gemm_kernel<IN, OUT, TM, TN, TRA, TRB, EVEN><<<grid, 256, 0, st>>>(a);                           \
    if (a.tail > 0 && a.splits <= 16) gemm_sum_kernel<OUT, TM, TN, IN == E4M3, 1><<<sums, 256, 0, st>>>(a); \
    if (a.tail > 0 && a.splits > 16) gemm_sum_kernel<OUT, TM, TN, IN == E4M3, 8><<<8 * sums, 256, 0, st>>>(a); \
  }
  if constexpr (IN == BF16 || IN == F16) {
    if (a.K % 64 == 0) {
      MALOQ_GEMM(256, 256, true)
    } else {
      MALOQ_GEMM(256, 256, false)
    }
  }
  if constexpr (IN == E4M3) {
    if (a.K % 128 == 0) {
      MALOQ_GEMM(256, 256, true)
    } else {
      MALOQ_GEMM(256, 256, false)
    }
  }
  MALOQ_GEMM(128, 128, false)
  if constexpr (!TRA && !TRB) {
    MALOQ_GEMM(64, 128, false)
    MALOQ_GEMM(32, 128, false)
  }
#undef MALOQ_GEMM
}
constexpr int FEW_ROWS = 16;  // of x at most, for the kernel of a few rows
void launch_few(int in, int out, const GemmArgs& a, void* stream);  // dense_few.hip
void launch_nt(int in, const GemmArgs& a, int tile, void* stream);    // dense_nt16.hip
void launch_nt8(int out, const GemmArgs& a, int tile, void* stream);  // dense_nt8.hip
void launch_nn(int in, const GemmArgs& a, int tile, void* stream);    // dense_bwd.hip
void launch_tn(int in, const GemmArgs& a, int tile, void* stream);

}  // namespace dense
}  // namespace maloq
