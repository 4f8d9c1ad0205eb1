#pragma once
// Tiled matrix products of the dense layers (dense.hip): C[m][n] = sum_k A(m, k) B(n, k), with the
// epilogue y = act(C [sa_m sb_n] + bias_n) + residual_mn.
//
// A workgroup of four waves owns a T x T tile of C, a wave a quarter of it in 32 x 32 MFMA tiles.
// Both operands are copied global -> LDS by DMA into a ring of four stages, three in flight, 64
// bytes of the contraction a stage for an operand whose rows run along it (N), 32 rows of it for one
// whose rows run across it (TR: the weights of an input gradient, both operands of a weight
// gradient), which is read back transposed (ds_read_b64_tr_b16).  One barrier per stage.
//
// What the operands must fulfil (the host sees to it): bases and row strides multiples of 16 bytes,
// the contiguous extent a multiple of 16 bytes.  Rows past the last are the last again (what they
// give is not stored); what lies past the contraction's end comes from a page of zeros.
#include "common.h"
#include "split_bf16.h"

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

// Types of operands and of results.  F32 operands are three bf16 planes (split_bf16.h).
enum { F32 = 0, BF16 = 1, F16 = 2, E4M3 = 3 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

__host__ __device__ constexpr int size_of(int type) { return type == F32 ? 4 : (type == E4M3 ? 1 : 2); }

// ------------------------------------------------------------- activations
// fp32 results need more than the hardware's exponential and reciprocal (1 ulp each, the
// exponential's argument rounded too) give; for 16 bits these are four digits more than enough.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (EXACT) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
template <bool EXACT>
__device__ __forceinline__ float act_fwd(float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;  // (NaN stays)
  if (act == ACT_SILU) return z * sigmoid<EXACT>(z);
  if (act == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
template <bool EXACT>
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if (act == ACT_SILU) {
    const float p = sigmoid<EXACT>(z);
    return p * (1.f + z * (1.f - p));
  }
  if (act == ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
           z * (EXACT ? expf(-0.5f * z * z) : __expf(-0.5f * z * z)) * 0.39894228040143268f;
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
// Eight at once, 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (TYPE == F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
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
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (TYPE == F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
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
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
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
  int vec;                // out, res and z take 16-byte accesses at columns that are multiples of 8
};

// Eight columns from n on of row m.  `bias` and `sb`: the lane's columns (zeros and ones where there are none).
template <int OUT>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t m, int n, int N, float (&v)[8],
                                        const float (&bias)[8], const float (&sb)[8]) {
  if (e.sa) {
    const float s = e.sa[m];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= s * sb[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += bias[k];
  const bool whole = e.vec && n + 8 <= N;
  if (e.z) {
    if (whole) {
      store8<OUT>(e.z, m * N + n, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < N) store1<OUT>(e.z, m * N + n + k, v[k]);
    }
  }
  if (e.act != ACT_NONE) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = act_fwd<OUT == F32>(v[k], e.act);
  }
  if (whole) {
    if (e.res) {
      float r[8];
      load8<OUT>(e.res, m * e.ldr + n, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += r[k];
    }
    store8<OUT>(e.out, m * e.ldo + n, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (n + k < N) store1<OUT>(e.out, m * e.ldo + n + k, e.res ? v[k] + load1<OUT>(e.res, m * e.ldr + n + k) : v[k]);
  }
}
template <int OUT>
__device__ __forceinline__ void columns8(const Epilogue& e, int n, int N, float (&bias)[8], float (&sb)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    bias[k] = e.bias && n + k < N ? load1<OUT>(e.bias, n + k) : 0.f;
    sb[k] = e.sb && n + k < N ? e.sb[n + k] : 1.f;
  }
}

// ----------------------------------------------------------------- kernel
struct GemmArgs {
  const char *a, *b;
  int64_t lda, ldb;     // bytes from one row to the next
  int64_t pa, pb;       // F32: bytes from one plane to the next
  int M, N, K;          // K: elements
  int splits;           // parts of the contraction
  int steps;            // K steps of a part
  float* part;          // splits > 1: [splits][M][N]
  Epilogue e;
};

static __device__ __constant__ uint4 zero_page[4] = {};

template <int T, int WAVES>
struct Geo {
  static constexpr int NS = 4;                 // stages
  static constexpr int OP = T * 64;            // bytes of one operand in a stage
  static constexpr int STAGE = 2 * OP;
  static constexpr int P = OP / 1024 / WAVES;  // 1 KB pieces that a wave copies of an operand
  static constexpr int TI = T / 64;            // MFMA tiles of a wave, each way
  static constexpr int PITCH = T / 2 * 4 + 16; // bytes of a row of the epilogue's strip
};

template <int IN>
__device__ __forceinline__ f32x16 mfma16(const s16x8& a, const s16x8& b, const f32x16& c) {
  if constexpr (IN == F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// One operand: how this lane copies it into a stage and reads it back.
template <int IN, int T, bool TR>
struct Operand {
  using G = Geo<T, 4>;
  static constexpr int ES = IN == E4M3 ? 1 : 2, KE = 64 / ES;
  static_assert(!TR || ES == 2, "transposed reads are of 16-bit elements");
  const char* base;     // the tile's first row (TR: column) at the contraction's start
  int64_t kstep, plane;
  unsigned off[G::P];   // from base + the step's offset
  int kel[G::P];        // element of the step's contraction that the piece's 16 bytes start at
  int rd[G::TI];        // where a lane's fragments of MFMA tile t lie in a stage

  // rows: the operand's extent across the contraction; r0: the tile's first
  __device__ __forceinline__ void init(const char* p, int64_t ld, int64_t plane_, int rows, int r0, int wave, int lane,
                                       int half) {
    plane = plane_;
    if constexpr (!TR) {
      // a row's four 16-byte chunks of the stage lie XORed with (row / 4) % 4: the reads of
      // any 16 consecutive rows then hit all banks once
      base = uniform(p + static_cast<int64_t>(r0) * ld);
      kstep = 64;
#pragma unroll
      for (int j = 0; j < G::P; ++j) {
        int r = (wave * G::P + j) * 16 + (lane >> 2);
        const int c = (lane & 3) ^ ((lane >> 4) & 3);
        kel[j] = c * (16 / ES);
        r = r0 + r < rows ? r : rows - 1 - r0;
        off[j] = static_cast<unsigned>(r * ld + c * 16);
      }
#pragma unroll
      for (int t = 0; t < G::TI; ++t) rd[t] = (half * (T / 2) + 32 * t + (lane & 31)) * 64;
    } else {
      // chunk c of contraction row r lies at c ^ 4 (r % 4): the four rows that a transposed
      // read of 16 lanes takes lie in different banks
      base = uniform(p + static_cast<int64_t>(r0) * ES);
      kstep = KE * ld;
      const int last = ((rows - r0) * ES + 15) / 16 - 1;  // of the row's chunks
#pragma unroll
      for (int j = 0; j < G::P; ++j) {
        const int at = (wave * G::P + j) * 64 + lane;
        constexpr int CH = T * ES / 16;  // chunks of a row
        const int r = at / CH;
        int c = (at % CH) ^ ((r & 3) << 2);
        c = c < last ? c : last;
        kel[j] = r;
        off[j] = static_cast<unsigned>(r * ld + c * 16);
      }
      const int g = lane >> 4, aa = lane & 3, kk = (lane >> 2) & 3;
#pragma unroll
      for (int t = 0; t < G::TI; ++t)
        rd[t] = (8 * (g >> 1) + kk) * (T * ES) + (2 * (g & 1) + (aa >> 1)) * 16 + (aa & 1) * 8 +
                64 * ((half * G::TI + t) ^ kk);
    }
  }
  // K step `step` of plane `pl` into the operand's part of a stage at LDS address `lds`; left: the
  // elements of the contraction from the step's first on.
  __device__ __forceinline__ void copy(unsigned lds, int wave, int step, int pl, int left) const {
    const char* p = base + step * kstep + pl * plane;
    if (left >= KE) {
#pragma unroll
      for (int j = 0; j < G::P; ++j)
        asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[j]), "s"(p),
                     "s"(__builtin_amdgcn_readfirstlane(lds + (wave * G::P + j) * 1024))
                     : "memory", "m0");
    } else {
#pragma unroll
      for (int j = 0; j < G::P; ++j) {
        const char* q = kel[j] < left ? p + off[j] : reinterpret_cast<const char*>(&zero_page[0]);
        asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(q),
                     "s"(__builtin_amdgcn_readfirstlane(lds + (wave * G::P + j) * 1024))
                     : "memory", "m0");
      }
    }
  }
  // 16-bit fragment: 8 elements of the contraction from 16 ks + 8 (lane / 32) on
  __device__ __forceinline__ s16x8 frag(const char* stage, int t, int ks, int lane) const {
    if constexpr (TR) {
      const s16x4 a = read_tr(stage + rd[t] + (16 * ks) * (T * ES)), b = read_tr(stage + rd[t] + (16 * ks + 4) * (T * ES));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const s16x8*>(stage + rd[t] + (((2 * ks + (lane >> 5)) ^ ((lane >> 2) & 3)) << 4));
    }
  }
  // 8-bit fragment: chunks lane / 32 and 2 + lane / 32 (the same elements of both operands, in the same order)
  __device__ __forceinline__ i32x8 frag8(const char* stage, int t, int lane) const {
    const i32x4 a = *reinterpret_cast<const i32x4*>(stage + rd[t] + (((lane >> 5) ^ ((lane >> 2) & 3)) << 4));
    const i32x4 b = *reinterpret_cast<const i32x4*>(stage + rd[t] + (((2 + (lane >> 5)) ^ ((lane >> 2) & 3)) << 4));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <int IN, int OUT, int T, bool TRA, bool TRB>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void gemm_kernel(GemmArgs a) {
  using G = Geo<T, 4>;
  using A = Operand<IN, T, TRA>;
  using B = Operand<IN, T, TRB>;
  constexpr int KE = A::KE, TI = G::TI;
  constexpr int PASSES = IN == F32 ? SPLIT_PRODUCTS : 1;
  __shared__ alignas(1024) char smem[G::NS * G::STAGE];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;

  // Tiles in an order in which the workgroups that run at the same time on one XCD (they are dealt
  // out over the eight in turn) share rows and columns: runs of 8 tiles down, then across.
  const int mt = (a.M + T - 1) / T, nt = (a.N + T - 1) / T;
  const unsigned tiles = static_cast<unsigned>(mt) * nt, per = gridDim.x >> 3;
  const unsigned wid = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (wid >= tiles * a.splits) return;  // whole workgroup, before any barrier
  const unsigned split = wid / tiles, id = wid - split * tiles;
  constexpr unsigned GM = 8;
  const unsigned group = id / (GM * nt), first = group * GM;
  const unsigned high = mt - first < GM ? mt - first : GM;
  const unsigned in_group = id - group * (GM * nt);
  const int m0 = __builtin_amdgcn_readfirstlane(first + in_group % high) * T;
  const int n0 = __builtin_amdgcn_readfirstlane(in_group / high) * T;

  const int ksteps = (a.K + KE - 1) / KE;
  const int kb = __builtin_amdgcn_readfirstlane(split * a.steps);
  const int kn = kb + a.steps < ksteps ? a.steps : (ksteps > kb ? ksteps - kb : 0);
  const int nsteps = __builtin_amdgcn_readfirstlane(kn * PASSES);

  const int wm = wave >> 1, wn = wave & 1;
  A oa;
  B ob;
  oa.init(a.a, a.lda, a.pa, a.M, m0, wave, lane, wm);
  ob.init(a.b, a.ldb, a.pb, a.N, n0, wave, lane, wn);
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) char*)smem));

  auto copy = [&](int stage, int s) {
    s = s < nsteps ? s : nsteps - 1;  // past the end: the last again, not read
    const int k = kb + s / PASSES, p = PASSES == 1 ? 0 : s % PASSES;
    const int left = a.K - k * KE;
    // the order of split_a and split_b
    const int pa = PASSES == 1 ? 0 : (0x021010 >> (4 * (5 - p))) & 3, pb = PASSES == 1 ? 0 : (0x201100 >> (4 * (5 - p))) & 3;
    oa.copy(lds0 + stage * G::STAGE, wave, k, pa, left);
    ob.copy(lds0 + stage * G::STAGE + G::OP, wave, k, pb, left);
  };

  f32x16 acc[TI][TI];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // (B's tile is the MFMA's first operand: a lane then holds four consecutive columns of a row of C)
  auto step = [&](int stage) {
    const char *sa = smem + stage * G::STAGE, *sb = sa + G::OP;
    if constexpr (IN == E4M3) {
      i32x8 fa[TI], fb[TI];
#pragma unroll
      for (int t = 0; t < TI; ++t) {
        fa[t] = oa.frag8(sa, t, lane);
        fb[t] = ob.frag8(sb, t, lane);
      }
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j)  // (unit block scales)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, 0, 0x7f7f7f7f, 0,
                                                                       0x7f7f7f7f);
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        s16x8 fa[TI], fb[TI];
#pragma unroll
        for (int t = 0; t < TI; ++t) {
          fa[t] = oa.frag(sa, t, ks, lane);
          fb[t] = ob.frag(sb, t, ks, lane);
        }
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int j = 0; j < TI; ++j) acc[i][j] = mfma16<IN>(fb[j], fa[i], acc[i][j]);
      }
    }
  };

  if (nsteps > 0) {
    copy(0, 0);
    copy(1, 1);
    copy(2, 2);
    for (int s = 0; s < nsteps; ++s) {
      // each step: this wave's copies of it done (two later steps' in flight), then all waves'
      // (barrier); the stage refilled was read one step earlier
      if constexpr (T == 256)
        asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      copy((s + 3) & 3, s + 3);
      step(s & 3);
    }
  }
  // no copy in flight, no wave still reading: the stages become the epilogue's strips
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // A wave's 32 rows of T / 2 columns at a time through LDS, so that a lane gets eight consecutive
  // columns and 256 (T = 128: 128) bytes of a row are stored together.
  constexpr int LPR = T / 2 / 8;  // lanes of a row
  char* strip = smem + wave * (32 * G::PITCH);
  static_assert(4 * 32 * G::PITCH <= G::NS * G::STAGE, "the strips fit the stages");
  const int cl = (lane % LPR) * 8, n = n0 + wn * (T / 2) + cl;
  float bias[8], sb[8];
  if (a.splits == 1) columns8<OUT>(a.e, n, a.N, bias, sb);
#pragma unroll
  for (int i = 0; i < TI; ++i) {
#pragma unroll
    for (int j = 0; j < TI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        *reinterpret_cast<f32x4*>(strip + (lane & 31) * G::PITCH + (32 * j + 8 * q + 4 * (lane >> 5)) * 4) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 2
    for (int r = lane / LPR; r < 32; r += 64 / LPR) {
      const int64_t m = m0 + wm * (T / 2) + 32 * i + r;
      const f32x4 v0 = *reinterpret_cast<const f32x4*>(strip + r * G::PITCH + cl * 4);
      const f32x4 v1 = *reinterpret_cast<const f32x4*>(strip + r * G::PITCH + cl * 4 + 16);
      float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
      if (m >= a.M || n >= a.N) continue;
      if (a.splits > 1) {
        float* p = a.part + (static_cast<int64_t>(split) * a.M + m) * a.N + n;
        if (a.N % 4 == 0 && n + 8 <= a.N) {
          *reinterpret_cast<f32x4*>(p) = v0;
          *reinterpret_cast<f32x4*>(p + 4) = v1;
        } else {
          for (int k = 0; k < 8; ++k)
            if (n + k < a.N) p[k] = v[k];
        }
      } else {
        finish8<OUT>(a.e, m, n, a.N, v, bias, sb);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Sums of the parts of a split contraction, in their order, and the epilogue.
template <int OUT>
__global__ __launch_bounds__(256) void gemm_sum_kernel(GemmArgs a) {
  const int groups = (a.N + 7) / 8;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= static_cast<int64_t>(a.M) * groups) return;
  const int64_t m = id / groups;
  const int n = static_cast<int>(id - m * groups) * 8;
  float bias[8], sb[8], v[8] = {};
  columns8<OUT>(a.e, n, a.N, bias, sb);
  const int64_t mn = static_cast<int64_t>(a.M) * a.N;
  const float* p = a.part + m * a.N + n;
  if (a.N % 4 == 0 && n + 8 <= a.N) {
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * mn), y = *reinterpret_cast<const f32x4*>(p + s * mn + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k], v[4 + k] += y[k];
    }
  } else {
    for (int s = 0; s < a.splits; ++s)
      for (int k = 0; k < 8; ++k)
        if (n + k < a.N) v[k] += p[s * mn + k];
  }
  finish8<OUT>(a.e, m, n, a.N, v, bias, sb);
}

// Launches: layouts 0 (x W^T), 1 (dz W: B across its rows), 2 (dz^T x: both across)
template <int IN, int OUT, bool TRA, bool TRB>
void launch_gemm(const GemmArgs& a, int tile, void* stream) {
  const int64_t tiles = static_cast<int64_t>((a.M + tile - 1) / tile) * ((a.N + tile - 1) / tile) * a.splits;
  const unsigned grid = static_cast<unsigned>((tiles + 7) / 8 * 8);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (tile == 256)
    gemm_kernel<IN, OUT, 256, TRA, TRB><<<grid, 256, 0, st>>>(a);
  else
    gemm_kernel<IN, OUT, 128, TRA, TRB><<<grid, 256, 0, st>>>(a);
}
void launch_nt(int in, const GemmArgs& a, int tile, void* stream);    // dense_nt16.hip
void launch_nt8(int out, const GemmArgs& a, int tile, void* stream);  // dense_nt8.hip
void launch_nn(int in, const GemmArgs& a, int tile, void* stream);    // dense_bwd.hip
void launch_tn(int in, const GemmArgs& a, int tile, void* stream);

}  // namespace dense
}  // namespace maloq
