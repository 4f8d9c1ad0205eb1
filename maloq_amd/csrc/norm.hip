// Root-mean-square norm with the residual's addition (maloq_rms_norm_*), and rows in 8 bits with
// one scale each (maloq_quantize_rows):
//
//   h = x + r;  rstd = (mean_k h_k^2 + eps)^-1/2;  y_k = h_k rstd w_k           (fp32, rounded once)
//   8 bits: a = max_k |y_k|, s = max(a, 2^-100) / 448, q_k = e4m3(y_k / s)
//   backward, u = g w:  dh = rstd (u - h rstd^2 mean(u h)) + g_h,  dw_k = sum_rows g_k h_k rstd
//
// The backward starts from h as it was stored, in the tensors' type: an fp32 copy would be 6 bytes a value more than the
// 14 that a 16-bit training step moves (a bf16 step's gradients are off by 2.5e-3 in norm from those of the unrounded h, one
// rounding being 1.7e-3).  Or, where the type does not hold every h (fp16: sums beyond 65504 are
// stored as infinities), from n = h rstd, of at most sqrt(width) <= 128, stored times 256, so that its least
// values are off by no more of the type's than h's are:  dh = rstd (u - n mean(u n)) + g_h,  dw_k = sum_rows g_k n_k.
//
// Memory bound: every value is read once and held in registers between the row's sums and its
// outputs.  TPR threads have a row, V values each in runs of 8 (16 bytes of 16-bit values, at any
// address), a row's last run perhaps shorter: within a wave the sums are shuffles, beyond it one
// exchange through LDS.  8191 x 4096 bf16 48 us (5.6 TB/s; a large copy 4.8), its 8-bit form from memory 62
// (3.8); 4093 x 8192 forward 45 us (6.0), backward 55 (4.9; 69 without the next row on its way); 32 000 x
// 128 fp32 13.6 and 14.6.  A step
// of 4093 x 8192 107 us in bf16, 119 in fp16, which writes the normed row too.
#include "dense_gemm.h"
#include "../../include/maloq_hip.h"

namespace maloq {
int sum_parts(int type, const float* part, int64_t blocks, int n, void* out, void* stream);  // dense.hip

namespace norm {

using dense::BF16;
using dense::F16;
using dense::F32;
using dense::MAX_THREADS;

struct NormArgs {
  const void *x, *r, *w;
  int64_t ldx, ldr, rows;
  int n;
  float eps;
  void *h, *y;
  float* rstd;
  uint8_t* q;
  float* scale;
  int quantize_only;  // q of x itself
  void* unit;         // UNIT h rstd
  int64_t first;      // row of this launch
  int int8;           // q: integers of -127 to 127 rather than e4m3
};
constexpr float UNIT = 256.f;  // a power of two

// Sum (or maximum) over the TPR threads of a row; TPR > 64: through LDS, `lds` a row of 16 floats
// that no other exchange uses until the next barrier.
template <int TPR, bool MAX>
__device__ __forceinline__ float across(float v, float* lds) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int k = 1; k < W; ++k) v = MAX ? fmaxf(v, lds[k]) : v + lds[k];
  }
  return v;
}

// The integer nearest to 127 v / m (|v| <= m, ties to the even one), t = v (127 / m) being that within 2^-15.  Beside a half,
// which side of it the quotient lies on is settled by 127 v - q m, which is exact in two floats there.  (Both are divided by
// 2^8: 127 v must not pass the floats' range.)
__device__ __forceinline__ int nearest127(float v, float m, float t) {
  float q = rintf(t);
  if (__builtin_expect(fabsf(t - q) > 0.4999f, 0)) {
    const float x = v * 0x1p-8f, y = m * 0x1p-8f, half = 0.5f * y;
    const float p = 127.f * x, e = fmaf(127.f, x, -p), r = fmaf(-q, y, p);
    const float above = (r - half) + e, below = (r + half) + e;
    const bool odd = static_cast<int>(q) & 1;
    q += above > 0.f || (above == 0.f && odd) ? 1.f : 0.f;
    q -= below < 0.f || (below == 0.f && odd) ? 1.f : 0.f;
  }
  return static_cast<int>(q);
}

template <int TYPE, int TPR, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_fwd_kernel(NormArgs a) {
  constexpr int RUNS = V / 8, NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  __shared__ float lds[3][16];
  const int t = threadIdx.x % TPR;
  const int64_t row = a.first + static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  if (TPR <= 64 && row >= a.rows) return;  // (TPR > 64: one row a block, never past the last)
  float h[RUNS][8];
  dense::Raw8<TYPE> x[RUNS], r[RUNS];
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    const int c = (i * TPR + t) * 8;
    x[i] = r[i] = {};
    if (c < a.n) x[i] = dense::load_part8<TYPE>(a.x, row * a.ldx + c, a.n - c);
    if (c < a.n && a.r) r[i] = dense::load_part8<TYPE>(a.r, row * a.ldr + c, a.n - c);
  }
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    const int c = (i * TPR + t) * 8;
    float e[8];
    dense::unpack8<TYPE>(x[i], h[i]);
    dense::unpack8<TYPE>(r[i], e);
    if (a.r) {
#pragma unroll
      for (int k = 0; k < 8; ++k) h[i][k] += e[k];
    }
    if (a.h && c < a.n) dense::store_part8<TYPE>(a.h, row * a.n + c, h[i], a.n - c);
  }
  if (!a.quantize_only) {
    float s[4] = {};
#pragma unroll
    for (int k = 0; k < V; ++k) s[k & 3] = fmaf(h[k / 8][k % 8], h[k / 8][k % 8], s[k & 3]);
    const float sum = across<TPR, false>((s[0] + s[1]) + (s[2] + s[3]), lds[0]);
    const float rstd = 1.f / sqrtf(sum / a.n + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rstd;
    if (a.unit) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const int c = (i * TPR + t) * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = h[i][k] * rstd * UNIT;
        if (c < a.n) dense::store_part8<TYPE>(a.unit, row * a.n + c, v, a.n - c);
      }
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c < a.n) {
        float w[8];
        dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.w, c, a.n - c), w);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i][k] *= rstd * w[k];
        if (a.y) dense::store_part8<TYPE>(a.y, row * a.n + c, h[i], a.n - c);
      }
    }
  }
  if (a.q) {
    float m = 0.f, bad = 0.f;  // bad: NaN if a value is not finite (the maximum passes over NaN)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      m = fmaxf(m, fabsf(h[k / 8][k % 8]));
      bad = fmaf(h[k / 8][k % 8], 0.f, bad);
    }
    m = across<TPR, true>(m, lds[1]);
    bad = across<TPR, false>(bad, lds[2]);
    m = fmaxf(m, 0x1p-100f);
    const float most = a.int8 ? 127.f : 448.f, inv = most / m;
    if (t == 0) a.scale[row] = m / most + bad;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c >= a.n) continue;
      union {
        uint32_t w[2];
        uint8_t b[8];
      } p;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float* v = h[i] + 4 * k;
        if (a.int8) {
          p.w[k] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) p.w[k] |= static_cast<uint32_t>(nearest127(v[j], m, v[j] * inv) & 255) << (8 * j);
          continue;
        }
        int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
        p.w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, u, true);
      }
      uint8_t* q = a.q + row * a.n + c;
      if (c + 8 <= a.n) {
        struct __attribute__((packed, aligned(1))) Eight {
          uint32_t w[2];
        };
        *reinterpret_cast<Eight*>(q) = {{p.w[0], p.w[1]}};
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < a.n) q[k] = p.b[k];
      }
    }
  }
}

// -------------------------------------------------------------- backward
struct NormBwdArgs {
  const void *g, *gh, *h, *w;
  int64_t ldg, ldgh, ldh, rows;
  int n;
  const float* rstd;
  float* part;  // [blocks][n], or null
  void* dx;
  int unit;     // h is UNIT h rstd
};

// A workgroup takes every gridDim-th group of RPB rows, the next group's values on their way while it
// has this one's; each thread keeps its columns' sums of dw over all of them, and the workgroup
// writes one row of partial sums.
template <int TYPE, int TPR, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_bwd_kernel(NormBwdArgs a) {
  constexpr int RUNS = V / 8, NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  constexpr bool AHEAD = TPR < 1024;  // (a workgroup of 16 waves has no registers for it, and other waves instead)
  __shared__ float lds[2][16];
  __shared__ float sums[RPB > 1 ? RPB : 1][RPB > 1 ? TPR : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float w[RUNS][8], dw[RUNS][8];
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    const int c = (i * TPR + t) * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) w[i][k] = dw[i][k] = 0.f;
    if (c < a.n) dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.w, c, a.n - c), w[i]);
  }
  dense::Raw8<TYPE> ng[RUNS], nh[RUNS];
  float nr = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    nr = a.rstd[row];
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c >= a.n) continue;
      ng[i] = dense::load_part8<TYPE>(a.g, row * a.ldg + c, a.n - c);
      nh[i] = dense::load_part8<TYPE>(a.h, row * a.ldh + c, a.n - c);
    }
  };
#pragma unroll
  for (int i = 0; i < RUNS; ++i) ng[i] = nh[i] = {};
  const int64_t stride = static_cast<int64_t>(gridDim.x) * RPB;
  if (AHEAD) fetch(static_cast<int64_t>(blockIdx.x) * RPB + sub);
  int turn = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += stride) {
    const int64_t row = r0 + sub;
    if (TPR <= 64 && row >= a.rows) break;
    if (!AHEAD) fetch(row);
    float g[RUNS][8], h[RUNS][8];
    dense::Raw8<TYPE> e[RUNS];
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * TPR + t) * 8;
      dense::unpack8<TYPE>(ng[i], g[i]);
      dense::unpack8<TYPE>(nh[i], h[i]);
      if (a.gh && a.dx && c < a.n) e[i] = dense::load_part8<TYPE>(a.gh, row * a.ldgh + c, a.n - c);
    }
    const float rstd = nr, to_n = a.unit ? 1.f / UNIT : rstd;  // h to_n = n
    if (AHEAD) fetch(row + stride);
    float s[4] = {};
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float u = g[k / 8][k % 8], v = h[k / 8][k % 8];
      s[k & 3] = fmaf(u * w[k / 8][k % 8], v, s[k & 3]);
      dw[k / 8][k % 8] = fmaf(u, v * to_n, dw[k / 8][k % 8]);
    }
    const float dot = across<TPR, false>((s[0] + s[1]) + (s[2] + s[3]), lds[turn]);
    turn ^= 1;  // (the next row's exchange must not overwrite what a slower wave still reads)
    const float f = dot / a.n * to_n * to_n;
    if (!a.dx) continue;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c >= a.n) continue;
      float o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = rstd * (g[i][k] * w[i][k] - h[i][k] * f);
      if (a.gh) {
        float u[8];
        dense::unpack8<TYPE>(e[i], u);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += u[k];
      }
      dense::store_part8<TYPE>(a.dx, row * a.n + c, o, a.n - c);
    }
  }
  if (!a.part) return;
  float* p = a.part + static_cast<int64_t>(blockIdx.x) * a.n;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k / 8 * TPR + t) * 8 + k % 8;
    if constexpr (RPB > 1) {
      __syncthreads();
      sums[sub][t] = dw[k / 8][k % 8];
      __syncthreads();
      if (sub == 0 && c < a.n) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < RPB; ++j) s += sums[j][t];
        p[c] = s;
      }
    } else if (c < a.n) {
      p[c] = dw[k / 8][k % 8];
    }
  }
}

// ------------------------------------------------------------------ host
constexpr int MAX_WIDTH = 16384;

// Threads a row and values a thread: at most 16 values (the backward has up to seven arrays of them),
// and several rows a wave where rows are short.
struct Pick {
  int tpr, v;
};
static Pick pick(int n) {
  if (n <= 256) return {16, 16};
  if (n <= 512) return {64, 8};
  if (n <= 1024) return {64, 16};
  if (n <= 2048) return {256, 8};
  if (n <= 4096) return {256, 16};
  if (n <= 8192) return {512, 16};
  return {1024, 16};
}
static int rows_of_block(const Pick& p) { return p.tpr >= 256 ? 1 : 256 / p.tpr; }

// (as many launches as it takes: one has fewer than 2^32 threads, 2^28 rows of up to 256 values or 2^22 of 16384)
template <int TYPE>
static void launch_fwd(NormArgs a, hipStream_t st) {
  const Pick p = pick(a.n);
  const int64_t most = MAX_THREADS / (p.tpr > 256 ? p.tpr : 256) * rows_of_block(p);
  for (a.first = 0; a.first < a.rows; a.first += most) {
    const int64_t rows = a.rows - a.first < most ? a.rows - a.first : most;
    const unsigned grid = static_cast<unsigned>((rows + rows_of_block(p) - 1) / rows_of_block(p));
#define MALOQ_NORM(TPR, V) \
  if (p.tpr == TPR && p.v == V) rms_norm_fwd_kernel<TYPE, TPR, V><<<grid, TPR > 256 ? TPR : 256, 0, st>>>(a);
    MALOQ_NORM(16, 16)
    MALOQ_NORM(64, 8) MALOQ_NORM(64, 16)
    MALOQ_NORM(256, 8) MALOQ_NORM(256, 16)
    MALOQ_NORM(512, 16) MALOQ_NORM(1024, 16)
#undef MALOQ_NORM
  }
}

static unsigned bwd_blocks(int64_t rows, const Pick& p) {
  const int64_t groups = (rows + rows_of_block(p) - 1) / rows_of_block(p), most = 2 * device_cus();
  return static_cast<unsigned>(groups < most ? groups : most);
}
template <int TYPE>
static void launch_bwd(const NormBwdArgs& a, hipStream_t st) {
  const Pick p = pick(a.n);
  const unsigned grid = bwd_blocks(a.rows, p);
#define MALOQ_NORM(TPR, V) \
  if (p.tpr == TPR && p.v == V) rms_norm_bwd_kernel<TYPE, TPR, V><<<grid, TPR > 256 ? TPR : 256, 0, st>>>(a);
  MALOQ_NORM(16, 16)
  MALOQ_NORM(64, 8) MALOQ_NORM(64, 16)
  MALOQ_NORM(256, 8) MALOQ_NORM(256, 16)
  MALOQ_NORM(512, 16) MALOQ_NORM(1024, 16)
#undef MALOQ_NORM
}

static int check(int dtype, int64_t rows, int64_t width) {
  MALOQ_REQUIRE(dtype >= F32 && dtype <= F16, "unsupported dtype code %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  MALOQ_REQUIRE(width >= 1 && width <= MAX_WIDTH, "rows of %lld values: 1 to %d", (long long)width, MAX_WIDTH);
  MALOQ_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "%lld rows out of range", (long long)rows);
  return MALOQ_OK;
}

static int forward(int dtype, const NormArgs& a, void* stream) {
  if (int rc = check(dtype, a.rows, a.n)) return rc;
  MALOQ_REQUIRE(!a.q || a.scale || a.rows == 0, "8-bit rows need a place for their scales");
  if (a.rows == 0) return MALOQ_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == F32) launch_fwd<F32>(a, st);
  if (dtype == BF16) launch_fwd<BF16>(a, st);
  if (dtype == F16) launch_fwd<F16>(a, st);
  return check_launch("maloq_rms_norm_fwd");
}

}  // namespace norm
}  // namespace maloq

using namespace maloq;
using namespace maloq::norm;

extern "C" int maloq_rms_norm_fwd(int dtype, const void* x, int64_t ld_x, const void* residual, int64_t ld_res,
                                  const void* weight, int64_t rows, int64_t width, float eps, void* h, void* y, float* rstd,
                                  void* q, float* scale, void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  const NormArgs a{x, residual, weight, ld_x, ld_res, rows, static_cast<int>(width), eps, h, y, rstd,
                   static_cast<uint8_t*>(q), scale, 0, nullptr, 0, 0};
  return forward(dtype, a, stream);
}

extern "C" int maloq_rms_norm_unit_fwd(int dtype, const void* x, int64_t ld_x, const void* residual, int64_t ld_res,
                                       const void* weight, int64_t rows, int64_t width, float eps, void* h, void* y, float* rstd,
                                       void* unit, void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  const NormArgs a{x, residual, weight, ld_x, ld_res, rows, static_cast<int>(width), eps, h, y, rstd, nullptr, nullptr, 0, unit, 0, 0};
  return forward(dtype, a, stream);
}

extern "C" int maloq_quantize_rows(int dtype, const void* x, int64_t ld_x, int64_t rows, int64_t width, void* q, float* scale,
                                   void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  const NormArgs a{x, nullptr, nullptr, ld_x, 0, rows, static_cast<int>(width), 0.f, nullptr, nullptr, nullptr,
                   static_cast<uint8_t*>(q), scale, 1, nullptr, 0, 0};
  return forward(dtype, a, stream);
}

extern "C" int maloq_rms_norm_int8_fwd(int dtype, const void* x, int64_t ld_x, const void* residual, int64_t ld_res,
                                       const void* weight, int64_t rows, int64_t width, float eps, void* h, void* q, float* scale,
                                       void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  const NormArgs a{x, residual, weight, ld_x, ld_res, rows, static_cast<int>(width), eps, h, nullptr, nullptr,
                   static_cast<uint8_t*>(q), scale, 0, nullptr, 0, 1};
  return forward(dtype, a, stream);
}

extern "C" int maloq_quantize_rows_int8(int dtype, const void* x, int64_t ld_x, int64_t rows, int64_t width, void* q, float* scale,
                                        void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  const NormArgs a{x, nullptr, nullptr, ld_x, 0, rows, static_cast<int>(width), 0.f, nullptr, nullptr, nullptr,
                   static_cast<uint8_t*>(q), scale, 1, nullptr, 0, 1};
  return forward(dtype, a, stream);
}

extern "C" int64_t maloq_rms_norm_bwd_partials_floats(int64_t rows, int64_t width) {
  if (rows < 0 || width < 1 || width > MAX_WIDTH) return -1;
  return static_cast<int64_t>(bwd_blocks(rows, pick(static_cast<int>(width)))) * width;
}

static int backward(int dtype, const void* g, int64_t ld_g, const void* g_h, int64_t ld_gh, const void* h, int64_t ld_h,
                    const void* weight, const float* rstd, int64_t rows, int64_t width, float* partials, void* dx, void* dw,
                    int unit, void* stream) {
  if (int rc = check(dtype, rows, width)) return rc;
  MALOQ_REQUIRE(!dw || partials, "the weight's gradient needs its partial sums");
  const int n = static_cast<int>(width);
  const NormBwdArgs a{g, g_h, h, weight, ld_g, ld_gh, ld_h, rows, n, rstd, dw ? partials : nullptr, dx, unit};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    if (dtype == F32) launch_bwd<F32>(a, st);
    if (dtype == BF16) launch_bwd<BF16>(a, st);
    if (dtype == F16) launch_bwd<F16>(a, st);
    if (int rc = check_launch("maloq_rms_norm_bwd")) return rc;
  }
  if (!dw) return MALOQ_OK;
  return sum_parts(dtype, partials, rows > 0 ? bwd_blocks(rows, pick(n)) : 0, n, dw, stream);
}

extern "C" int maloq_rms_norm_bwd(int dtype, const void* g, int64_t ld_g, const void* g_h, int64_t ld_gh, const void* h,
                                  int64_t ld_h, const void* weight, const float* rstd, int64_t rows, int64_t width,
                                  float* partials, void* dx, void* dw, void* stream) {
  return backward(dtype, g, ld_g, g_h, ld_gh, h, ld_h, weight, rstd, rows, width, partials, dx, dw, 0, stream);
}

extern "C" int maloq_rms_norm_unit_bwd(int dtype, const void* g, int64_t ld_g, const void* g_h, int64_t ld_gh, const void* unit,
                                       int64_t ld_unit, const void* weight, const float* rstd, int64_t rows, int64_t width,
                                       float* partials, void* dx, void* dw, void* stream) {
  return backward(dtype, g, ld_g, g_h, ld_gh, unit, ld_unit, weight, rstd, rows, width, partials, dx, dw, 1, stream);
}
