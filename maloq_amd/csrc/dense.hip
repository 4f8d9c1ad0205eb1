// Dense layers (maloq_linear_*): y = act(x W^T + b) + r and its gradients, and the same of 8-bit
// operands with scales.  The products are dense_gemm.h's; here are the choice of tiles, what brings
// operands into the form that the products need, and the activation's gradient.
#include "dense_gemm.h"
#include "../../include/maloq_hip.h"

namespace maloq {
namespace dense {

// --------------------------------------------------------- operands' form
// Rows of `cols` elements to rows of ldp, a multiple of 16 bytes, the rest zero; up to two matrices a launch.
struct PadJob {
  const void* src;
  void* dst;
  int64_t ld, rows;
  int cols, ldp;
  int64_t first, left;  // 16 bytes of the result: done before this launch, and after that to do
  unsigned blocks;
};
template <class E>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadJob a, PadJob b) {
  constexpr int V = 16 / sizeof(E);
  const bool second = blockIdx.x >= a.blocks;
  const PadJob& j = second ? b : a;
  const int per = j.ldp / V;
  const int64_t id = j.first + static_cast<int64_t>(blockIdx.x - (second ? a.blocks : 0)) * 256 + threadIdx.x;
  if (id >= j.rows * per) return;
  const int64_t r = id / per;
  const int c = static_cast<int>(id - r * per) * V;
  const E* src = static_cast<const E*>(j.src) + r * j.ld + c;
  union {
    E e[V];
    uint4 q;
  } v;
  if (c + V <= j.cols) {
    v.q = load_loose(src);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v.e[k] = c + k < j.cols ? src[k] : E(0);
  }
  *reinterpret_cast<uint4*>(static_cast<E*>(j.dst) + r * j.ldp + c) = v.q;
}
static int pad_rows(int es, PadJob a, PadJob b, hipStream_t st) {
  constexpr int64_t MOST = MAX_THREADS / 256;
  for (PadJob* j : {&a, &b}) j->first = 0, j->left = j->rows * (j->ldp / (16 / es));
  if (a.left + b.left == 0) return MALOQ_OK;
  while (a.left + b.left > 0) {
    int64_t grid = 0;
    for (PadJob* j : {&a, &b}) {
      const int64_t blocks = (j->left + 255) / 256, now = blocks < MOST - grid ? blocks : MOST - grid;
      j->blocks = static_cast<unsigned>(now);
      j->left -= now < blocks ? now * 256 : j->left;
      grid += now;
    }
    if (es == 4)
      pad_rows_kernel<uint32_t><<<static_cast<unsigned>(grid), 256, 0, st>>>(a, b);
    else if (es == 2)
      pad_rows_kernel<uint16_t><<<static_cast<unsigned>(grid), 256, 0, st>>>(a, b);
    else
      pad_rows_kernel<uint8_t><<<static_cast<unsigned>(grid), 256, 0, st>>>(a, b);
    for (PadJob* j : {&a, &b}) j->first += static_cast<int64_t>(j->blocks) * 256;
  }
  return check_launch("pad_rows");
}

// ---------------------------------------------------- activation's gradient
// dz = g act'(z) (rows of ldz, zero past n), and its column sums by blocks of `rows` rows: a block has
// 128 columns, 16 lanes of 8, and 16 rows at a time.  Memory bound: 4133 x 4096 bf16 21.6 us, 4.7 TB/s.
// z comes, and dz goes, in the tensors' type: the products take 16-bit operands, and an fp32 z would be twice the bytes here and in
// the forward.  That makes a bf16 step's gradients 2.4e-3 off in norm, where one rounding of the result is 1.7e-3 (fp16 3.0e-4 and
// 2.1e-4).  db sums dz before it is rounded.
template <int TYPE, int ACT>
__global__ __launch_bounds__(256) void act_bwd_kernel(const void* g, int64_t ldg, const void* z, int64_t m, int n, void* dz,
                                                      int64_t ldz, float* part, int rows, unsigned columns) {
  __shared__ float sums[16][129];
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const unsigned by = blockIdx.x / columns, bx = blockIdx.x - by * columns;
  const int c = bx * 128 + cx * 8;
  const int64_t r0 = static_cast<int64_t>(by) * rows;
  float s[8] = {};
#pragma unroll 4
  for (int i = 0; i < rows; i += 16) {
    const int64_t r = r0 + i + ry;
    if (r >= m) break;
    float v[8];
    unpack8<TYPE>(load_part8<TYPE>(g, r * ldg + c, n - c), v);
    if constexpr (ACT != ACT_NONE) {
      float y[8];
      unpack8<TYPE>(load_part8<TYPE>(z, r * n + c, n - c), y);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= c + k < n ? act_slope<TYPE == F32, ACT>(y[k]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] += v[k];
    if (dz && c < ldz) store_part8<TYPE>(dz, r * ldz + c, v, static_cast<int>(ldz - c < 8 ? ldz - c : 8));
  }
  if (!part) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) sums[ry][cx * 8 + k] = s[k];
  __syncthreads();
  const int col = threadIdx.x;
  if (col < 128 && bx * 128 + col < n) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += sums[k][col];
    part[static_cast<int64_t>(by) * n + bx * 128 + col] = t;
  }
}

}  // namespace dense

// Sums of the rows of part [blocks][n], in a fixed order, to n values of a type: a block has 32 columns,
// each by 32 threads that take every 32nd row.
template <int TYPE>
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* part, int64_t blocks, int n, void* out) {
  __shared__ float sums[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  float s = 0.f;
  if (c < n) {
    int64_t b = ry;
    for (; b + 7 * 32 < blocks; b += 8 * 32) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(b + 32 * k) * n + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
#pragma unroll 4
    for (; b < blocks; b += 32) s += part[b * n + c];
  }
  sums[ry][cx] = s;
  __syncthreads();
  if (ry == 0 && c < n) {
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sums[k][cx];
    dense::store1<TYPE>(out, c, s);
  }
}
int sum_parts(int type, const float* part, int64_t blocks, int n, void* out, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int grid = (n + 31) / 32;
  if (type == dense::F32) sum_parts_kernel<dense::F32><<<grid, 1024, 0, st>>>(part, blocks, n, out);
  if (type == dense::BF16) sum_parts_kernel<dense::BF16><<<grid, 1024, 0, st>>>(part, blocks, n, out);
  if (type == dense::F16) sum_parts_kernel<dense::F16><<<grid, 1024, 0, st>>>(part, blocks, n, out);
  return check_launch("sum_parts");
}

namespace dense {

// ------------------------------------------------------------------- host
constexpr int64_t MAX_DIM = int64_t(1) << 24;  // of a product: offsets within a tile stay below 2^32 bytes

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Shape {
  int in, layout;      // layout: 0 x W^T, 1 dz W, 2 dz^T x
  int64_t m, n, k;
  int es, vec;         // operand bytes, elements of 16 bytes
  int64_t ext[2], rows[2];  // contiguous extent and rows of A and B in memory
  bool few;            // the kernel for a few rows: operands as they are
  int tile, full, tail, splits, steps;
};

// The tile, and how many tiles, the last ones, are split along the contraction so that they fill the chip:
// what takes the least time by this model, in microseconds.  Whole tiles are dealt to the CUs first, either as
// many as all can hold at a time or, where that leaves most of a round empty, one to each; parts join them.  A K
// step takes `one` where a workgroup is alone on its CU and `all` where as many are there as fit; the first
// one's start and epilogue take `ends`, each further one's `more`; partial sums are written and read
// back, and a kernel adds them.  Fitted to the times that 131 products of 17 .. 40000 x 64 .. 16384 x 64 .. 16384 values
// took with every tile and 1 to 16 parts (1463 times; off by 8 % rms); its choices take 2 % longer than the
// best of these on average, 14 % at most; of 172 gradients' products, to which it was not fitted, 2 % too, 21 %
// at most.  (777 x 1240 x 1531 bf16: whole tiles of 128 16.6 us, in three parts 20.2; 256 x 4096 x 1024: 24.4
// whole, 14.0 in four parts; fp32 2100 x 1024 x 2048, 272 tiles of 128: whole 82.8, the last 16 in four parts
// 60.3; bf16 9000 x 256 x 1000: tiles of 256 23.5, of 128 18.7.)
struct TileTimes {
  uint32_t tile, fit;  // rows; workgroups a CU
  double one, all, ends, more;
};
constexpr TileTimes TIMES_16[] = {{256, 1, 1.01, 1.01, 11.0, 4.1}, {128, 2, 0.38, 0.795, 6.1, 0.3}, {64, 2, 0.227, 0.41, 5.5, 1.9}, {32, 3, 0.224, 0.67, 4.9, 0.9}};
constexpr TileTimes TIMES_32[] = {{128, 2, 1.05, 2.12, 8.7, 0}, {64, 2, 0.77, 1.36, 7.4, 1.0}, {32, 3, 0.50, 0.83, 7.1, 1.5}};
struct SumTimes {
  double value, ends, part;  // a partial sum's way to memory and back; their kernel, and for each part, sixteen at most
};
constexpr SumTimes SUM_16 = {1.19e-6, 0.89, 0.036}, SUM_32 = {1.46e-6, 0, 0.074};

static Shape shape_of(int in, int layout, int64_t m, int64_t n, int64_t k) {
  Shape s{in, layout, m, n, k, size_of(in), 16 / size_of(in), {}, {}, false, 0, 0, 0, 1, 0};
  s.ext[0] = layout == 2 ? m : k, s.rows[0] = layout == 2 ? k : m;
  s.ext[1] = layout == 0 ? k : n, s.rows[1] = layout == 0 ? n : k;
  s.few = layout == 0 && in != F32 && m <= FEW_ROWS;
  if (s.few) return s;
  if (m == 0 || n == 0) return s;
  // (32-bit divisions: this runs in every call, on the host)
  const uint32_t cus = static_cast<uint32_t>(device_cus()), steps = static_cast<uint32_t>((k * s.es + 127) / 128);
  double best = 0;
  const SumTimes& sum = in == F32 ? SUM_32 : SUM_16;
  const TileTimes* const first_of = in == F32 ? TIMES_32 : TIMES_16;
  for (const TileTimes* c = first_of; c != first_of + (in == F32 ? 3 : 4); ++c) {
    const uint32_t tile = c->tile, wide = tile == 256 ? 256 : 128;
    if (tile < 128 && (layout != 0 || m > tile)) continue;
    const uint32_t mt = static_cast<uint32_t>((m + tile - 1) / tile), nt = static_cast<uint32_t>((n + wide - 1) / wide), tiles = mt * nt;
    // whole tiles that are dealt to each CU at a time (1 of few tiles: the same parts again)
    for (uint32_t deal = c->fit; deal > 0; deal = deal > 1 && tiles > cus ? 1 : 0) {
      const uint32_t slots = deal * cus, full = tiles / slots * slots, tail = tiles - full;
      // rows of the tail's tiles that exist (they are the last rows of tiles)
      const uint32_t first = tail >= nt ? mt - (tail + nt - 1) / nt : mt - 1;
      const double rows = static_cast<double>(m - static_cast<int64_t>(first) * tile), high = rows < tile ? rows : tile;
      for (const uint32_t p : {1u, 2u, 3u, 4u, 6u, 8u, 12u, 16u, tail ? cus / tail : 0, tail ? slots / tail : 0, tail ? 2 * slots / tail : 0}) {
        if (p == 0 || (p > 1 && (p * 2 > steps || tail == 0))) continue;
        const uint32_t each = (steps + p - 1) / p, parts = each > 0 ? (steps + each - 1) / each : 1;
        // of the CU that has the most: whole tiles and parts, their steps, the longest's, and how many are there at a time
        const uint32_t whole = parts > 1 ? full / cus : (tiles + cus - 1) / cus, pieces = parts > 1 ? (tail * parts + cus - 1) / cus : 0;
        const double work = static_cast<double>(whole) * steps + pieces * each, longest = whole ? steps : each;
        const double fit = c->fit, there = work > fit * longest ? fit : (work > longest ? work / longest : 1.0);
        const double step = c->fit > 1 ? c->one + (c->all - c->one) * (there - 1) / (c->fit - 1) : c->one;
        double t = work / there * step + c->ends + c->more * (whole + pieces - 1);
        if (parts > 1) t += sum.value * tail * parts * wide * high + sum.ends + sum.part * (parts < 16 ? parts : 16);
        if (s.tile == 0 || t < best) {
          best = t;
          s.tile = static_cast<int>(tile);
          s.splits = static_cast<int>(parts);
          s.steps = static_cast<int>(parts > 1 ? each : steps);
          s.full = static_cast<int>(parts > 1 ? full : tiles);
          s.tail = static_cast<int>(tiles - s.full);
        }
      }
    }
  }
  return s;
}

static bool copied(const Shape& s, int op) { return !s.few && s.ext[op] % s.vec; }
static int64_t copy_bytes(const Shape& s, int op) { return copied(s, op) ? up(s.rows[op] * up(s.ext[op], s.vec) * s.es, 256) : 0; }
static int64_t part_bytes(const Shape& s) { return 4 * static_cast<int64_t>(s.splits) * s.tail * s.tile * (s.tile == 256 ? 256 : 128); }
static int64_t workspace(const Shape& s) { return copy_bytes(s, 0) + copy_bytes(s, 1) + part_bytes(s); }

// ready: bit op set: the operand's rows reach to the next multiple of 16 bytes already, with zeros, and start at such.
static int run(int in, int out, int layout, const void* a, int64_t lda, const void* b, int64_t ldb, int64_t m, int64_t n,
               int64_t k, Epilogue e, int ready, void* ws, void* stream) {
  MALOQ_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m < MAX_DIM * 64 && n < MAX_DIM && k < MAX_DIM * 64,
                "product of sizes %lld x %lld x %lld out of range", (long long)m, (long long)n, (long long)k);
  if (m == 0 || n == 0) return MALOQ_OK;
  const Shape s = shape_of(in, layout, m, n, k);
  MALOQ_REQUIRE(s.rows[0] < (int64_t(1) << 31) && s.rows[1] < (int64_t(1) << 31) && s.ext[0] < MAX_DIM && s.ext[1] < MAX_DIM,
                "product of sizes %lld x %lld x %lld out of range", (long long)m, (long long)n, (long long)k);
  hipStream_t st = static_cast<hipStream_t>(stream);
  GemmArgs g{};
  g.M = static_cast<int>(m), g.N = static_cast<int>(n), g.K = static_cast<int>(k);
  const void* p[2] = {a, b};
  int64_t ld[2] = {lda, ldb};
  char* w = static_cast<char*>(ws);
  PadJob jobs[2] = {};
  for (int op = 0; op < 2 && k > 0; ++op) {
    if (copied(s, op) && !(ready >> op & 1)) {
      MALOQ_REQUIRE(w, "an operand of %lld rows needs a workspace", (long long)s.rows[op]);
      const int64_t ldp = up(s.ext[op], s.vec);
      jobs[op] = {p[op], w, ld[op], s.rows[op], static_cast<int>(s.ext[op]), static_cast<int>(ldp), 0, 0, 0};
      p[op] = w, ld[op] = ldp;
    }
    w += copy_bytes(s, op);
    ld[op] *= s.es;
    MALOQ_REQUIRE(s.few || (reinterpret_cast<uint64_t>(p[op]) | ld[op]) % 16 == 0, "operand rows must start at multiples of 16 bytes");
    MALOQ_REQUIRE(ld[op] >= 0 && ld[op] < (int64_t(1) << 24), "row stride of an operand too large");
  }
  if (int rc = pad_rows(s.es, jobs[0], jobs[1], st)) return rc;
  g.a = static_cast<const char*>(p[0]), g.b = static_cast<const char*>(p[1]);
  g.lda = ld[0], g.ldb = ld[1];
  g.full = s.full, g.tail = s.tail, g.splits = s.splits, g.steps = s.steps;
  g.part = reinterpret_cast<float*>(w);
  MALOQ_REQUIRE(s.tail == 0 || ws, "a split product needs a workspace");
  g.e = e;
  if (s.few)
    launch_few(in, out, g, stream);
  else if (in == E4M3)
    launch_nt8(out, g, s.tile, stream);
  else if (layout == 0)
    launch_nt(in, g, s.tile, stream);
  else if (layout == 1)
    launch_nn(in, g, s.tile, stream);
  else
    launch_tn(in, g, s.tile, stream);
  return check_launch("maloq_linear");
}

static int check_types(int dtype, int act) {
  MALOQ_REQUIRE(dtype >= F32 && dtype <= F16, "unsupported dtype code %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  MALOQ_REQUIRE(act >= ACT_NONE && act <= ACT_GELU, "unknown activation %d", act);
  return MALOQ_OK;
}

}  // namespace dense
}  // namespace maloq

using namespace maloq;
using namespace maloq::dense;

extern "C" int64_t maloq_linear_workspace_bytes(int dtype, int product, int64_t m, int64_t k, int64_t n) {
  if (dtype < F32 || dtype > E4M3 || product < 0 || product > 2 || m < 0 || k < 0 || n < 0) return -1;
  // product 1: [m, n] x [n, k], 2: [n, m] x [m, k]
  return product == 0   ? workspace(shape_of(dtype, 0, m, n, k))
         : product == 1 ? workspace(shape_of(dtype, 1, m, k, n))
                        : workspace(shape_of(dtype, 2, n, k, m));
}

extern "C" int maloq_linear_plan(int dtype, int product, int64_t m, int64_t k, int64_t n, int64_t* plan) {
  MALOQ_REQUIRE(dtype >= F32 && dtype <= E4M3 && product >= 0 && product <= (dtype == E4M3 ? 0 : 2) && m >= 0 && k >= 0 && n >= 0 && plan,
                "no product %d of dtype code %d", product, dtype);
  const Shape s = product == 0   ? shape_of(dtype, 0, m, n, k)
                  : product == 1 ? shape_of(dtype, 1, m, k, n)
                                 : shape_of(dtype, 2, n, k, m);
  plan[0] = s.tile, plan[1] = s.full, plan[2] = s.tail, plan[3] = s.splits;
  return MALOQ_OK;
}

extern "C" int maloq_linear_pad(int dtype, const void* x, int64_t ld_x, int64_t m, const void* w, int64_t ld_w, int64_t n,
                                int64_t k, void* x_out, void* w_out, void* stream) {
  if (int rc = check_types(dtype, 0)) return rc;
  MALOQ_REQUIRE(m >= 0 && n >= 0 && k >= 0 && k < MAX_DIM, "sizes out of range");
  const int es = size_of(dtype), kp = static_cast<int>(up(k, 16 / es));
  return pad_rows(es, {x, x_out, ld_x, m, static_cast<int>(k), kp, 0, 0, 0}, {w, w_out, ld_w, n, static_cast<int>(k), kp, 0, 0, 0},
                  static_cast<hipStream_t>(stream));
}

extern "C" int maloq_linear_fwd(int dtype, const void* x, int64_t ld_x, const void* w, int64_t ld_w, const void* bias,
                                const void* residual, int64_t ld_res, int act, int64_t m, int64_t k, int64_t n, void* ws,
                                void* z, void* y, void* stream) {
  if (int rc = check_types(dtype, act)) return rc;
  Epilogue e{nullptr, nullptr, bias, residual, ld_res, y, n, z, act};
  return run(dtype, dtype, 0, x, ld_x, w, ld_w, m, n, k, e, 0, ws, stream);
}

extern "C" int maloq_linear_quantized(int out_dtype, const void* q, int64_t ld_q, const float* scale, const void* wq,
                                      int64_t ld_w, const float* w_scale, const void* bias, const void* residual,
                                      int64_t ld_res, int act, int64_t m, int64_t k, int64_t n, void* ws, void* y,
                                      void* stream) {
  if (int rc = check_types(out_dtype, act)) return rc;
  MALOQ_REQUIRE((scale && w_scale) || m == 0 || n == 0, "8-bit operands need their scales");
  Epilogue e{scale, w_scale, bias, residual, ld_res, y, n, nullptr, act};
  return run(E4M3, out_dtype, 0, q, ld_q, wq, ld_w, m, n, k, e, 0, ws, stream);
}

extern "C" int maloq_linear_dx(int dtype, const void* dz, int64_t ld_dz, const void* w, int64_t ld_w, int padded, int64_t m,
                               int64_t k, int64_t n, void* ws, void* dx, void* stream) {
  if (int rc = check_types(dtype, 0)) return rc;
  Epilogue e{nullptr, nullptr, nullptr, nullptr, 0, dx, k, nullptr, ACT_NONE};
  return run(dtype, dtype, 1, dz, ld_dz, w, ld_w, m, k, n, e, padded ? 3 : 1, ws, stream);
}

extern "C" int maloq_linear_dw(int dtype, const void* dz, int64_t ld_dz, const void* x, int64_t ld_x, int padded, int64_t m,
                               int64_t k, int64_t n, void* ws, void* dw, void* stream) {
  if (int rc = check_types(dtype, 0)) return rc;
  Epilogue e{nullptr, nullptr, nullptr, nullptr, 0, dw, k, nullptr, ACT_NONE};
  return run(dtype, dtype, 2, dz, ld_dz, x, ld_x, n, k, m, e, padded ? 3 : 1, ws, stream);
}

// Rows of a block of the activation's gradient: 128, fewer until there are four blocks a CU.
static int act_bwd_rows(int64_t m, int64_t n) {
  int64_t rows = 128;
  while (rows > 16 && (m + rows - 1) / rows * ((n + 127) / 128) < 4 * device_cus()) rows /= 2;
  return static_cast<int>(rows);
}

extern "C" int64_t maloq_linear_act_bwd_partials_floats(int64_t m, int64_t n) {
  if (m < 0 || n < 0) return -1;
  const int rows = act_bwd_rows(m, n);
  return (m + rows - 1) / rows * n;
}

extern "C" int maloq_linear_act_bwd(int dtype, const void* g, int64_t ld_g, const void* z, int act, int64_t m, int64_t n,
                                    void* dz, int64_t ld_dz, float* partials, void* db, void* stream) {
  if (int rc = check_types(dtype, act)) return rc;
  MALOQ_REQUIRE(act == ACT_NONE || z || m == 0 || n == 0, "the gradient of an activation needs what it was given");
  MALOQ_REQUIRE(!dz || ld_dz >= n, "ld_dz %lld < n", (long long)ld_dz);
  const int rows = act_bwd_rows(m, n);
  const int64_t blocks = (m + rows - 1) / rows, wide = dz && ld_dz > n ? ld_dz : n;
  MALOQ_REQUIRE(m >= 0 && n >= 0 && wide < MAX_DIM && blocks * ((wide + 127) / 128) <= MAX_THREADS / 256, "%lld x %lld values are too many", (long long)m, (long long)n);
  if (n == 0) return MALOQ_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!db) partials = nullptr;
  const unsigned columns = static_cast<unsigned>((wide + 127) / 128), grid = columns * static_cast<unsigned>(blocks);
  if (blocks > 0) {
#define MALOQ_ACT_BWD(TYPE, ACT)                                                                                        \
  if (dtype == TYPE && act == ACT)                                                                                       \
    act_bwd_kernel<TYPE, ACT><<<grid, 256, 0, st>>>(g, ld_g, z, m, static_cast<int>(n), dz, ld_dz, partials, rows, columns);
#define MALOQ_ACT_BWD4(TYPE) \
  MALOQ_ACT_BWD(TYPE, ACT_NONE) MALOQ_ACT_BWD(TYPE, ACT_RELU) MALOQ_ACT_BWD(TYPE, ACT_SILU) MALOQ_ACT_BWD(TYPE, ACT_GELU)
    MALOQ_ACT_BWD4(F32)
    MALOQ_ACT_BWD4(BF16)
    MALOQ_ACT_BWD4(F16)
#undef MALOQ_ACT_BWD4
#undef MALOQ_ACT_BWD
  }
  if (int rc = check_launch("maloq_linear_act_bwd")) return rc;
  return db ? sum_parts(dtype, partials, blocks, static_cast<int>(n), db, stream) : MALOQ_OK;
}
