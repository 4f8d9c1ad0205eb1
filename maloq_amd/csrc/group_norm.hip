// Group norm with an activation, channels last (maloq_group_norm_*): x [samples][places][channels], a group is c = channels /
// groups consecutive channels of all places of a sample:
//
//   mean, var over places x c;  rstd = (var + eps)^-1/2;  n = (x - mean) rstd;  z = n w + b;  y = act(z)
//   backward, u = g act'(z):  db = sum u,  dw = sum u n,  dx = rstd (u w - mean(u w) - n mean(u w n))
//
// Everything between load and store is fp32.  The variance is of differences from the mean: of a thread's values from their
// own mean first, then of the means (sums of squares would lose what a mean beside a small deviation leaves).
//
// Memory bound.  Where some groups' values of a sample fit the registers of a workgroup (up to 65536 values, the backward
// with its two arrays 16384), one launch reads and writes everything once; else one launch sums parts of each group and one
// reads the values again.
//
// A thread has eight consecutive channels (16 bytes of 16-bit values, at any address), `wp` threads, a power of two, the
// workgroup's columns of a place; further threads the places that follow.
//
// What bounds it: 4 x 16384 x 512 bf16 in 32 groups (67 MB), with silu: sums of parts 25 to 27 us, result 25 to 26 (its second read from the
// caches), gradients' parts 36 (134 MB), dx 38 (201 MB, 5.3 TB/s, the rate of a large copy); a step moves 536 MB where 268 are
// its arrays.  Held: 8 x 4096 x 512 24 us for 67 MB, one workgroup a CU, whose load, two exchanges and stores follow each other;
// 32 x 1000 x 128 fp32 15 us and its gradient 21.  Vector units: 17 instructions a value for silu (two of them at a quarter of the
// rate), 45 for its gradient.  A batch of places ahead in the loops of parts was no faster (27 and 39 us: registers).  Of the kernels
// that hold eight places with 1024 threads those for groups of any channels spill, 9 registers in fp32 and 2 in bf16.
#include "dense_gemm.h"
#include "../../include/maloq_hip.h"

namespace maloq {
int sum_parts(int type, const float* part, int64_t blocks, int n, void* out, void* stream);  // dense.hip

namespace group {

using dense::BF16;
using dense::F16;
using dense::F32;
using dense::MAX_THREADS;

struct GroupArgs {
  const void *x, *g, *w, *b;  // w, b: or null
  int64_t ldx, ldg;
  int samples, places, channels, groups, c;
  int act;
  float eps;
  void* out;     // y, or dx (or null)
  float* stats;  // [samples][groups][2]: mean, rstd
  float* part;   // partial sums
  void* dwb;     // [2][channels]: dw, db
  int wp, gpt, tiles;   // threads of a place; groups of a tile, tiles of a place
  int sub, subcols;     // tiles of a group of more columns than a tile has, and their columns (sub = 1: none)
  int parts, rows;      // parts of a sample's places, and their places
  int slots;            // workgroups of a tile, each every slots-th sample (of two launches: every slots-th part, in the backward's first)
  int span;             // threads of a sample: all of a workgroup's, or up to a wave's, others having the samples that follow
};

// The columns of tile t
struct Columns {
  int col0, cols, group0, groups, c;  // c: columns of a group that are here
};
__device__ __forceinline__ Columns columns_of(const GroupArgs& a, int t) {
  if (a.sub > 1) {
    const int g = t / a.sub, first = (t - g * a.sub) * a.subcols, cols = a.c - first < a.subcols ? a.c - first : a.subcols;
    return {g * a.c + first, cols, g, 1, cols};
  }
  const int g0 = t * a.gpt, n = a.groups - g0 < a.gpt ? a.groups - g0 : a.gpt;
  return {g0 * a.c, n * a.c, g0, n, a.c};
}

// EIGHTS, in all that follows: groups of a multiple of eight channels, so that a thread's columns are of one group, whose numbers
// it holds once (of() is the place of column k's in such an array).
template <bool EIGHTS>
constexpr int OF = EIGHTS ? 1 : 8;
template <bool EIGHTS>
__device__ __forceinline__ constexpr int of(int k) { return EIGHTS ? 0 : k; }

// A thread's eight columns.  A tile's last eight overlap those before, [lo, 8) being its own; a tile of fewer has [0, hi).
struct Lane {
  int first, lo, hi;  // first: in the tile
  __device__ __forceinline__ Lane(const Columns& t, int u) {
    first = u * 8 + 8 <= t.cols || t.cols < 8 ? u * 8 : t.cols - 8;
    lo = u * 8 - first < 8 ? u * 8 - first : 8;
    hi = t.cols - first < 8 ? t.cols - first : 8;
    if (u * 8 >= t.cols) first = lo = hi = 0;
  }
  __device__ __forceinline__ bool any() const { return hi > lo; }
};

// Sums over the columns of each of the tile's groups, of Q numbers for each of a thread's eight columns: over the lanes of
// a wave that have the same columns, then through LDS.  sums: [Q][samples of the workgroup][groups], where the caller finds
// them after it returns.  lds: [Q][rows][8 wp], rows = samples where there are several, else waves, or NT / wp where a place
// takes more than a wave.
__host__ __device__ constexpr int lds_rows(int nt, int wp, int span) { return span < nt ? nt / span : wp < 64 ? nt / 64 : nt / wp; }
template <int NT, int Q, bool EIGHTS>
__device__ __forceinline__ void group_sums(float (&v)[Q][8], int wp, int span, const Columns& t, const Lane& l, float* lds, float* sums) {
  const int tid = threadIdx.x, per = NT / span, wave = span < 64 ? span : 64;  // wave: lanes that add their numbers
  const int rows = per > 1 ? per : wp < 64 ? NT / 64 : NT / wp, row = per > 1 ? tid / span : wp < 64 ? tid >> 6 : tid / wp;
  const bool writes = wp >= 64 || (tid & (wave - 1)) < wp;
  const int c = EIGHTS ? t.c / 8 : t.c, pitch = EIGHTS ? wp : wp * 8;
  if constexpr (EIGHTS) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float s = ((v[q][0] + v[q][1]) + (v[q][2] + v[q][3])) + ((v[q][4] + v[q][5]) + (v[q][6] + v[q][7]));
      for (int o = wp; o < wave; o *= 2) s += __shfl_xor(s, o);
      if (writes) lds[(q * rows + row) * pitch + (tid & (wp - 1))] = s;
    }
  } else {
    for (int o = wp; o < wave; o *= 2) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[q][k] += __shfl_xor(v[q][k], o);
    }
    if (writes) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k >= l.lo && k < l.hi) lds[(q * rows + row) * pitch + l.first + k] = v[q][k];
    }
  }
  __syncthreads();
  const int all = per * t.groups;
  int tpg = 64;
  while (tpg > 1 && tpg * all > NT) tpg /= 2;
  const int j = tid & (tpg - 1);
  for (int i = tid / tpg; i < all; i += NT / tpg) {
    const int of_sample = per > 1 ? i / t.groups : 0, g = i - of_sample * t.groups, end = per > 1 ? of_sample + 1 : rows;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float s = 0.f;
      for (int r = of_sample; r < end; ++r)
        for (int ch = j; ch < c; ch += tpg) s += lds[(q * rows + r) * pitch + g * c + ch];
      for (int o = tpg / 2; o > 0; o /= 2) s += __shfl_xor(s, o);
      if (j == 0) sums[q * all + i] = s;
    }
  }
  __syncthreads();
}
// f(column of the eight, group of the tile that it is in); EIGHTS: f(0, the eight's group)
template <bool EIGHTS, class F>
__device__ __forceinline__ void each_column(const Columns& t, const Lane& l, const F& f) {
  int g = l.first / t.c, left = (g + 1) * t.c - l.first;
  if constexpr (EIGHTS) {
    f(0, g < t.groups ? g : t.groups - 1);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (left == 0) ++g, left = t.c;
    --left;
    f(k, g < t.groups ? g : t.groups - 1);
  }
}

// Eight columns of w (or ones) and b (or zeros)
template <int TYPE>
__device__ __forceinline__ void load_affine(const GroupArgs& a, int col, const Lane& l, float (&w)[8], float (&b)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = 1.f, b[k] = 0.f;
  if (!l.any()) return;
  if (a.w) dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.w, col, l.hi), w);
  if (a.b) dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.b, col, l.hi), b);
}
// Eight columns of R places from row r on, every step-th, as far as `places`; the others zero.
template <int TYPE, bool EIGHTS, int R>
__device__ __forceinline__ void load_places(dense::Raw8<TYPE> (&x)[R], const void* p, int64_t ld, int64_t row0, int col, int r, int step,
                                            int places, const Columns& t, const Lane& l) {
#pragma unroll
  for (int i = 0; i < R; ++i) x[i] = {};
  if (!l.any()) return;
  if (EIGHTS || t.cols >= 8) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (r + i * step < places) x[i] = dense::load_raw8<TYPE>(p, (row0 + r + i * step) * ld + col);
  } else {
#pragma unroll 1
    for (int i = 0; i < R; ++i) {
      if (r + i * step >= places) break;
      const dense::Raw8<TYPE> v = dense::load_part8<TYPE>(p, (row0 + r + i * step) * ld + col, l.hi);
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (k == i) x[k] = v;
    }
  }
}
template <int TYPE, bool EIGHTS>
__device__ __forceinline__ void store_place(const GroupArgs& a, int64_t row, int col, const Columns& t, const Lane& l, const float (&v)[8]) {
  if (EIGHTS || t.cols >= 8)
    dense::store8<TYPE>(a.out, row * a.channels + col, v);  // (columns that two threads have are the same from both)
  else
    dense::store_part8<TYPE>(a.out, row * a.channels + col, v, l.hi);
}
// f(activation as a constant), one of them
template <class F>
__device__ __forceinline__ void with_act(int act, const F& f) {
  if (act == dense::ACT_NONE)
    f(std::integral_constant<int, dense::ACT_NONE>{});
  else if (act == dense::ACT_RELU)
    f(std::integral_constant<int, dense::ACT_RELU>{});
  else if (act == dense::ACT_SILU)
    f(std::integral_constant<int, dense::ACT_SILU>{});
  else
    f(std::integral_constant<int, dense::ACT_GELU>{});
}
// n and u of eight columns, from x and g
template <int TYPE, int ACT, bool EIGHTS>
__device__ __forceinline__ void slopes(float (&x)[8], float (&g)[8], const float (&mean)[OF<EIGHTS>], const float (&rstd)[OF<EIGHTS>],
                                       const float (&w)[8], const float (&b)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[k] = (x[k] - mean[of<EIGHTS>(k)]) * rstd[of<EIGHTS>(k)];
    g[k] *= dense::act_slope<TYPE == F32, ACT>(fmaf(x[k], w[k], b[k]));
  }
}

// ------------------------------------------------- values held in registers
// A workgroup has one tile of one sample, or of several where a wave or less has all places of one; a thread R places of
// eight columns.
template <int TYPE, int NT, int R, bool EIGHTS>
__global__ __launch_bounds__(NT) void group_fwd_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x, per = NT / a.span, sample = tid / a.span, rt = (tid - sample * a.span) / a.wp, nr = a.span / a.wp;
  const unsigned items = static_cast<unsigned>((a.samples + per - 1) / per) * a.tiles, item = dense::dealt(blockIdx.x, items);
  if (item >= items) return;
  const int n0 = item / a.tiles * per, n = n0 + sample, places = n < a.samples ? a.places : 0;
  const Columns t = columns_of(a, item % a.tiles);
  const Lane l(t, tid & (a.wp - 1));
  float* sums = lds + lds_rows(NT, a.wp, a.span) * a.wp * 8;  // [2][samples][groups]
  const int col = t.col0 + l.first, all = per * t.groups, mine = sample * t.groups;
  const int64_t row0 = static_cast<int64_t>(n) * a.places;

  dense::Raw8<TYPE> raw[R];
  load_places<TYPE, EIGHTS, R>(raw, a.x, a.ldx, row0, col, rt, nr, places, t, l);
  float x[R][8], v[1][8], mean[OF<EIGHTS>], rstd[OF<EIGHTS>], scale[8], b[8];
  load_affine<TYPE>(a, col, l, scale, b);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    dense::unpack8<TYPE>(raw[i], x[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] += x[i][k];
  }
  group_sums<NT, 1, EIGHTS>(v, a.wp, a.span, t, l, lds, sums);
  const float count = static_cast<float>(a.places) * a.c;  // (divided by: a group of one value has that mean)
  each_column<EIGHTS>(t, l, [&](int k, int g) { mean[k] = sums[mine + g] / count; });
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[i][k] -= mean[of<EIGHTS>(k)];
    if (rt + i * nr < places) {  // (a thread without columns: numbers that nobody reads)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[0][k] = fmaf(x[i][k], x[i][k], v[0][k]);
    }
  }
  group_sums<NT, 1, EIGHTS>(v, a.wp, a.span, t, l, lds, sums + all);
  if (a.stats) {
    for (int i = tid; i < all; i += NT) {
      const int of_sample = i / t.groups, g = i - of_sample * t.groups;
      if (n0 + of_sample >= a.samples) break;
      float* s = a.stats + (static_cast<int64_t>(n0 + of_sample) * a.groups + t.group0 + g) * 2;
      s[0] = sums[i] / count;
      s[1] = 1.f / sqrtf(sums[all + i] / count + a.eps);
    }
  }
  if (!l.any()) return;
  each_column<EIGHTS>(t, l, [&](int k, int g) { rstd[k] = 1.f / sqrtf(sums[all + mine + g] / count + a.eps); });
#pragma unroll
  for (int k = 0; k < 8; ++k) scale[k] *= rstd[of<EIGHTS>(k)];
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i * nr + rt >= places) break;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[i][k] = dense::act_fwd<TYPE == F32, decltype(act)::value>(fmaf(x[i][k], scale[k], b[k]));
      store_place<TYPE, EIGHTS>(a, row0 + i * nr + rt, col, t, l, x[i]);
    }
  });
}

// Sums over the places of a workgroup, of eight columns a thread: put(0 or 1, column of the tile, sum).
template <int NT, class F>
__device__ __forceinline__ void column_sums(float (&v)[2][8], int wp, const Columns& t, const Lane& l, float* lds, const F& put) {
  const int tid = threadIdx.x, rows = wp < 64 ? NT / 64 : NT / wp, pitch = wp * 8;
  for (int o = wp; o < 64; o *= 2) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[q][k] += __shfl_xor(v[q][k], o);
  }
  if (wp >= 64 || (tid & 63) < wp) {
    const int row = wp < 64 ? tid >> 6 : tid / wp;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k >= l.lo && k < l.hi) lds[(q * rows + row) * pitch + l.first + k] = v[q][k];
  }
  __syncthreads();
  for (int i = tid; i < 2 * t.cols; i += NT) {
    const int q = i < t.cols ? 0 : 1, ch = q ? i - t.cols : i;
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += lds[(q * rows + r) * pitch + ch];
    put(q, ch, s);
  }
}

// .. and every slots-th sample; dw and db are summed over them.
template <int TYPE, int NT, int R, bool EIGHTS>
__global__ __launch_bounds__(NT) void group_bwd_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x, per = NT / a.span, sample = tid / a.span, rt = (tid - sample * a.span) / a.wp, nr = a.span / a.wp;
  const unsigned item = dense::dealt(blockIdx.x, static_cast<unsigned>(a.slots) * a.tiles);
  if (item >= static_cast<unsigned>(a.slots) * a.tiles) return;
  const int slot = item / a.tiles;
  const Columns t = columns_of(a, item - slot * a.tiles);
  const Lane l(t, tid & (a.wp - 1));
  float* sums = lds + 2 * lds_rows(NT, a.wp, a.span) * a.wp * 8;  // [2][samples][groups]
  const int col = t.col0 + l.first, all = per * t.groups, of_sample = sample * t.groups;
  const float count = 1.f / (static_cast<float>(a.places) * a.c);
  float w[8], b[8], total[2][8];
  load_affine<TYPE>(a, col, l, w, b);
#pragma unroll
  for (int k = 0; k < 8; ++k) total[0][k] = total[1][k] = 0.f;
  for (int64_t n0 = static_cast<int64_t>(slot) * per; n0 < a.samples; n0 += static_cast<int64_t>(a.slots) * per) {
    const int64_t n = n0 + sample < a.samples ? n0 + sample : a.samples - 1, row0 = n * a.places;
    const int mine = n0 + sample < a.samples && l.any() ? a.places : 0;
    dense::Raw8<TYPE> x[R], g[R];
    load_places<TYPE, EIGHTS, R>(x, a.x, a.ldx, row0, col, rt, nr, mine, t, l);
    load_places<TYPE, EIGHTS, R>(g, a.g, a.ldg, row0, col, rt, nr, mine, t, l);
    float mean[OF<EIGHTS>], rstd[OF<EIGHTS>], u[R][8], v[2][8];
    const float* stats = a.stats + (n * a.groups + t.group0) * 2;
    each_column<EIGHTS>(t, l, [&](int k, int gr) { mean[k] = stats[2 * gr], rstd[k] = stats[2 * gr + 1]; });
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] = v[1][k] = 0.f;
    with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
        dense::unpack8<TYPE>(g[i], u[i]);
        slopes<TYPE, decltype(act)::value, EIGHTS>(e, u[i], mean, rstd, w, b);
        if (rt + i * nr < mine) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            v[0][k] = fmaf(u[i][k], e[k], v[0][k]);
            v[1][k] += u[i][k];
          }
        }
      }
    });
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 8; ++k) total[q][k] += v[q][k], v[q][k] *= w[k];
    if (!a.out) continue;
    group_sums<NT, 2, EIGHTS>(v, a.wp, a.span, t, l, lds, sums);
    float m0[OF<EIGHTS>], m1[OF<EIGHTS>];
    each_column<EIGHTS>(t, l, [&](int k, int gr) { m1[k] = sums[of_sample + gr] * count, m0[k] = sums[all + of_sample + gr] * count; });
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (rt + i * nr >= mine) break;
      float e[8];
      dense::unpack8<TYPE>(x[i], e);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int o = of<EIGHTS>(k);
        e[k] = rstd[o] * (fmaf(u[i][k], w[k], -m0[o]) - (e[k] - mean[o]) * rstd[o] * m1[o]);
      }
      store_place<TYPE, EIGHTS>(a, row0 + i * nr + rt, col, t, l, e);
    }
  }
  if (!a.part && !a.dwb) return;
  __syncthreads();  // (the last sample's sums have been read)
  column_sums<NT>(total, a.wp, t, l, lds, [&](int q, int ch, float s) {
    const int64_t at = static_cast<int64_t>(q) * a.channels + t.col0 + ch;
    if (a.dwb)  // (one workgroup a tile)
      dense::store1<TYPE>(a.dwb, at, s);
    else
      a.part[static_cast<int64_t>(slot) * 2 * a.channels + at] = s;
  });
}

// ------------------------------------------------------------- two launches
// The first sums parts of each group, the second adds a group's parts, in every workgroup that needs it, and reads the
// values again.
constexpr int WIDE = 256;      // threads
constexpr int MAX_COLS = 512;  // of a tile

// The places of a part
__device__ __forceinline__ int places_of(const GroupArgs& a, int part) {
  const int left = a.places - part * a.rows;
  return left < a.rows ? left : a.rows;
}
// workgroup -> tile, part, sample; tiles of the same places next to each other
struct Where {
  int tile, part, n;
};
__device__ __forceinline__ bool where(const GroupArgs& a, unsigned block, Where& w) {
  const unsigned all = static_cast<unsigned>(a.samples) * a.parts * a.tiles, item = dense::dealt(block, all);
  if (item >= all) return false;
  const unsigned sp = item / a.tiles;
  w = {static_cast<int>(item - sp * a.tiles), static_cast<int>(sp % a.parts), static_cast<int>(sp / a.parts)};
  return true;
}
// The parts of group g (of the tile) of a sample: pairs of numbers
__device__ __forceinline__ float2* pairs_of(const GroupArgs& a, int n, int g) {
  return reinterpret_cast<float2*>(a.part) + (static_cast<int64_t>(n) * a.groups + g) * a.parts * a.sub;
}
__device__ __forceinline__ int pair_of(const GroupArgs& a, const Where& at) { return at.part * a.sub + (a.sub > 1 ? at.tile % a.sub : 0); }

// Mean and sum of squared differences from it, of each of the tile's groups in a part.
constexpr int BATCH = 8;  // places of a thread at a time
template <int TYPE, bool EIGHTS>
__global__ __launch_bounds__(WIDE) void group_parts_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  Where at;
  if (!where(a, blockIdx.x, at)) return;
  const int tid = threadIdx.x, rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const Lane l(t, tid & (a.wp - 1));
  float* sums = lds + (a.wp < 64 ? WIDE / 64 : WIDE / a.wp) * a.wp * 8;
  const int col = t.col0 + l.first, places = places_of(a, at.part);
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  float mean[8], m2[8], n = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) mean[k] = m2[k] = 0.f;
  for (int r0 = rt; r0 < places && l.any(); r0 += BATCH * nr) {
    dense::Raw8<TYPE> raw[BATCH];
    load_places<TYPE, EIGHTS, BATCH>(raw, a.x, a.ldx, row0, col, r0, nr, places, t, l);
    const int some = (places - r0 + nr - 1) / nr, m = some < BATCH ? some : BATCH;
    float x[BATCH][8], s[8], d[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = d[k] = 0.f;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      dense::unpack8<TYPE>(raw[i], x[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += x[i][k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = m == BATCH ? s[k] * (1.f / BATCH) : s[k] / m;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (i < m) {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = fmaf(x[i][k] - s[k], x[i][k] - s[k], d[k]);
      }
    }
    const float all = n + m, f = m / all, h = n * f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float apart = s[k] - mean[k];
      mean[k] = fmaf(apart, f, mean[k]);
      m2[k] += fmaf(apart * apart, h, d[k]);
    }
    n = all;
  }
  float v[1][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = n * mean[k];
  group_sums<WIDE, 1, EIGHTS>(v, a.wp, WIDE, t, l, lds, sums);
  const float count = static_cast<float>(places) * t.c;
  float of_group[OF<EIGHTS>];
  each_column<EIGHTS>(t, l, [&](int k, int g) { of_group[k] = sums[g] / count; });
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float apart = mean[k] - of_group[of<EIGHTS>(k)];
    v[0][k] = fmaf(apart * apart, n, m2[k]);
  }
  group_sums<WIDE, 1, EIGHTS>(v, a.wp, WIDE, t, l, lds, sums + t.groups);
  for (int g = tid; g < t.groups; g += WIDE) pairs_of(a, at.n, t.group0 + g)[pair_of(a, at)] = make_float2(sums[g] / count, sums[t.groups + g]);
}
// Mean and rstd of the tile's groups from their parts, to stats[2][groups].
template <class F>
__device__ __forceinline__ void each_group(const Columns& t, const F& f) {
  int tpg = 64;
  while (tpg > 1 && tpg * t.groups > WIDE) tpg /= 2;
  const int j = threadIdx.x & (tpg - 1);
  for (int g = threadIdx.x / tpg; g < t.groups; g += WIDE / tpg) f(g, j, tpg);
  __syncthreads();
}
__device__ __forceinline__ void merge_parts(const GroupArgs& a, int n, const Columns& t, float* stats) {
  const int all = a.parts * a.sub;
  const float values = static_cast<float>(a.places) * a.c, share = 1.f / values;
  auto count = [&](int i) {
    if (a.sub == 1) return static_cast<float>(places_of(a, i)) * a.c;
    const int of = i % a.sub, left = a.c - of * a.subcols;
    return static_cast<float>(places_of(a, i / a.sub)) * (left < a.subcols ? left : a.subcols);
  };
  each_group(t, [&](int g, int j, int tpg) {
    const float2* p = pairs_of(a, n, t.group0 + g);
    const float first = p[0].x;  // (differences from it: parts of one mean have that mean)
    float s = 0.f, m2 = 0.f;
    for (int i = j; i < all; i += tpg) s = fmaf(p[i].x - first, count(i) * share, s);
    for (int o = tpg / 2; o > 0; o /= 2) s += __shfl_xor(s, o);
    s += first;
    for (int i = j; i < all; i += tpg) {
      const float2 v = p[i];
      m2 += fmaf((v.x - s) * (v.x - s), count(i), v.y);
    }
    for (int o = tpg / 2; o > 0; o /= 2) m2 += __shfl_xor(m2, o);
    if (j == 0) stats[g] = s, stats[t.groups + g] = 1.f / sqrtf(m2 * share + a.eps);
  });
}
template <int TYPE, bool EIGHTS>
__global__ __launch_bounds__(WIDE) void group_apply_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  Where at;
  if (!where(a, blockIdx.x, at)) return;
  const int tid = threadIdx.x, rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const Lane l(t, tid & (a.wp - 1));
  const int col = t.col0 + l.first, places = places_of(a, at.part);
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  dense::Raw8<TYPE> x[BATCH];
  load_places<TYPE, EIGHTS, BATCH>(x, a.x, a.ldx, row0, col, rt, nr, places, t, l);
  float mean[OF<EIGHTS>], rstd[OF<EIGHTS>], scale[8], b[8];
  load_affine<TYPE>(a, col, l, scale, b);
  merge_parts(a, at.n, t, lds);
  if (a.stats && at.part == 0 && (a.sub == 1 || at.tile % a.sub == 0)) {
    for (int g = tid; g < t.groups; g += WIDE) {
      float* s = a.stats + (static_cast<int64_t>(at.n) * a.groups + t.group0 + g) * 2;
      s[0] = lds[g], s[1] = lds[t.groups + g];
    }
  }
  if (!l.any()) return;
  each_column<EIGHTS>(t, l, [&](int k, int g) { mean[k] = lds[g], rstd[k] = lds[t.groups + g]; });
#pragma unroll
  for (int k = 0; k < 8; ++k) scale[k] *= rstd[of<EIGHTS>(k)];
  for (int r0 = rt; r0 < places;) {
    with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (r0 + i * nr >= places) break;
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = dense::act_fwd<TYPE == F32, decltype(act)::value>(fmaf(e[k] - mean[of<EIGHTS>(k)], scale[k], b[k]));
        store_place<TYPE, EIGHTS>(a, row0 + r0 + i * nr, col, t, l, e);
      }
    });
    r0 += BATCH * nr;
    if (r0 < places) load_places<TYPE, EIGHTS, BATCH>(x, a.x, a.ldx, row0, col, r0, nr, places, t, l);
  }
}

// Of a part: the sums of u w n and u w of each group; and columns[slots][2][channels] (for dw and db; or null), the sums of u n
// and u of each column.  MANY: of every slots-th part; else each part has its row of columns, which for many samples of few
// places would be more bytes than x (100000 x 1 x 8192 bf16: 6.6 GB beside 1.6), but whose kernel has three waves a SIMD for two.
constexpr int BATCH_BWD = 4;
template <int TYPE, bool EIGHTS, bool MANY>
__global__ __launch_bounds__(WIDE) void group_bwd_parts_kernel(GroupArgs a, float* columns) {
  extern __shared__ float lds[];
  Where at;
  unsigned slot = 0;
  if constexpr (MANY) {
    const unsigned all = static_cast<unsigned>(a.slots) * a.tiles, item = dense::dealt(blockIdx.x, all);
    if (item >= all) return;
    slot = item / a.tiles;
    at.tile = static_cast<int>(item - slot * a.tiles);
  } else if (!where(a, blockIdx.x, at)) {
    return;
  }
  const int tid = threadIdx.x, rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const Lane l(t, tid & (a.wp - 1));
  float* sums = lds + 2 * (a.wp < 64 ? WIDE / 64 : WIDE / a.wp) * a.wp * 8;
  const int col = t.col0 + l.first;
  float v[2][8];
  const auto part = [&]() __attribute__((always_inline)) {
    const int places = places_of(a, at.part);
    const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
    float mean[OF<EIGHTS>], rstd[OF<EIGHTS>], w[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] = v[1][k] = 0.f;
    load_affine<TYPE>(a, col, l, w, b);
    const float* stats = a.stats + (static_cast<int64_t>(at.n) * a.groups + t.group0) * 2;
    each_column<EIGHTS>(t, l, [&](int k, int g) { mean[k] = stats[2 * g], rstd[k] = stats[2 * g + 1]; });
    for (int r0 = rt; r0 < places && l.any(); r0 += BATCH_BWD * nr) {
      dense::Raw8<TYPE> x[BATCH_BWD], g[BATCH_BWD];
      load_places<TYPE, EIGHTS, BATCH_BWD>(x, a.x, a.ldx, row0, col, r0, nr, places, t, l);
      load_places<TYPE, EIGHTS, BATCH_BWD>(g, a.g, a.ldg, row0, col, r0, nr, places, t, l);
      with_act(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < BATCH_BWD; ++i) {
          if (r0 + i * nr >= places) break;
          float e[8], u[8];
          dense::unpack8<TYPE>(x[i], e);
          dense::unpack8<TYPE>(g[i], u);
          slopes<TYPE, decltype(act)::value, EIGHTS>(e, u, mean, rstd, w, b);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            v[0][k] = fmaf(u[k], e[k], v[0][k]);
            v[1][k] += u[k];
          }
        }
      });
    }
    float uw[2][8];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 8; ++k) uw[q][k] = v[q][k] * w[k];
    group_sums<WIDE, 2, EIGHTS>(uw, a.wp, WIDE, t, l, lds, sums);
    for (int g = tid; g < t.groups; g += WIDE) pairs_of(a, at.n, t.group0 + g)[pair_of(a, at)] = make_float2(sums[g], sums[t.groups + g]);
  };
  if constexpr (MANY) {
    float total[2][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) total[0][k] = total[1][k] = 0.f;
    const unsigned parts = static_cast<unsigned>(a.samples) * a.parts;
    for (unsigned i = slot; i < parts; i += a.slots) {
      at.part = static_cast<int>(i % a.parts), at.n = static_cast<int>(i / a.parts);
      part();
#pragma unroll
      for (int k = 0; k < 8; ++k) total[0][k] += v[0][k], total[1][k] += v[1][k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] = total[0][k], v[1][k] = total[1][k];
  } else {
    part();
  }
  if (!columns) return;
  float* to = columns + (MANY ? static_cast<int64_t>(slot) : static_cast<int64_t>(at.n) * a.parts + at.part) * 2 * a.channels + t.col0;
  column_sums<WIDE>(v, a.wp, t, l, lds, [&](int q, int ch, float s) { to[static_cast<int64_t>(q) * a.channels + ch] = s; });
}
// dx; and the first `adders` workgroups add the rows of columns to dw and db.
constexpr int ADD = 32;  // columns of a workgroup, each by 8 threads
template <int TYPE, bool EIGHTS>
__global__ __launch_bounds__(WIDE) void group_bwd_apply_kernel(GroupArgs a, const float* columns, unsigned adders) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x;
  if (blockIdx.x < adders) {
    const int c = blockIdx.x * ADD + tid % ADD, lane = tid / ADD;
    const int64_t all = a.slots, wide = 2 * static_cast<int64_t>(a.channels);
    float s[8] = {};
    if (c < wide) {
      int64_t i = lane;
      for (; i + 7 * 8 < all; i += 8 * 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += columns[(i + 8 * k) * wide + c];
      }
      for (; i < all; i += 8) s[0] += columns[i * wide + c];
    }
    lds[tid] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (lane > 0 || c >= wide) return;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += lds[k * ADD + tid];
    dense::store1<TYPE>(a.dwb, c, sum);
    return;
  }
  Where at;
  if (!where(a, blockIdx.x - adders, at)) return;
  const int rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const Lane l(t, tid & (a.wp - 1));
  const int col = t.col0 + l.first, places = places_of(a, at.part);
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  dense::Raw8<TYPE> x[BATCH_BWD], g[BATCH_BWD];
  load_places<TYPE, EIGHTS, BATCH_BWD>(x, a.x, a.ldx, row0, col, rt, nr, places, t, l);
  load_places<TYPE, EIGHTS, BATCH_BWD>(g, a.g, a.ldg, row0, col, rt, nr, places, t, l);
  float mean[OF<EIGHTS>], rstd[OF<EIGHTS>], w[8], b[8], m0[OF<EIGHTS>], m1[OF<EIGHTS>];
  load_affine<TYPE>(a, col, l, w, b);
  const float* stats = a.stats + (static_cast<int64_t>(at.n) * a.groups + t.group0) * 2;
  each_column<EIGHTS>(t, l, [&](int k, int gr) { mean[k] = stats[2 * gr], rstd[k] = stats[2 * gr + 1]; });
  const float share = 1.f / (static_cast<float>(a.places) * a.c);
  each_group(t, [&](int gr, int j, int tpg) {
    const float2* p = pairs_of(a, at.n, t.group0 + gr);
    float s0 = 0.f, s1 = 0.f;
    for (int i = j; i < a.parts * a.sub; i += tpg) s0 += p[i].x, s1 += p[i].y;
    for (int o = tpg / 2; o > 0; o /= 2) s0 += __shfl_xor(s0, o), s1 += __shfl_xor(s1, o);
    if (j == 0) lds[gr] = s0 * share, lds[t.groups + gr] = s1 * share;
  });
  if (!l.any()) return;
  each_column<EIGHTS>(t, l, [&](int k, int gr) { m1[k] = lds[gr], m0[k] = lds[t.groups + gr]; });
  for (int r0 = rt; r0 < places;) {
    with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < BATCH_BWD; ++i) {
        if (r0 + i * nr >= places) break;
        float e[8], u[8];
        dense::unpack8<TYPE>(x[i], e);
        dense::unpack8<TYPE>(g[i], u);
        slopes<TYPE, decltype(act)::value, EIGHTS>(e, u, mean, rstd, w, b);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = rstd[of<EIGHTS>(k)] * (fmaf(u[k], w[k], -m0[of<EIGHTS>(k)]) - e[k] * m1[of<EIGHTS>(k)]);
        store_place<TYPE, EIGHTS>(a, row0 + r0 + i * nr, col, t, l, e);
      }
    });
    r0 += BATCH_BWD * nr;
    if (r0 < places) {
      load_places<TYPE, EIGHTS, BATCH_BWD>(x, a.x, a.ldx, row0, col, r0, nr, places, t, l);
      load_places<TYPE, EIGHTS, BATCH_BWD>(g, a.g, a.ldg, row0, col, r0, nr, places, t, l);
    }
  }
}

// ------------------------------------------------------------------- host
constexpr int64_t MAX_CHANNELS = int64_t(1) << 24;
constexpr int64_t MOST_THREADS = MAX_THREADS - 8 * 1024;  // of a launch, whose grid is a multiple of eight workgroups

static int pow2(int64_t v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}

// Threads of a workgroup and places of a thread (threads 0: two launches), and the tiles.
struct Plan {
  int threads, places, wp, gpt, tiles, sub, subcols, parts, rows, slots, span;
};
constexpr int MAX_LDS = 64 * 1024;
// LDS of a workgroup of nt threads: Q numbers of each column that a wave (a place, a sample) has, and 2 of each group
static int64_t lds_of(int nt, int wp, int span, int64_t gpt, int q) {
  const int waves = wp < 64 ? nt / 64 : nt / wp, rows = lds_rows(nt, wp, span);  // (columns are summed over waves)
  return 4 * (q * static_cast<int64_t>(rows > waves ? rows : waves) * wp * 8 + 2 * gpt * (nt / span));
}
// Which way, in microseconds: a start, more for wider workgroups (parts: for a thousand pairs that a workgroup adds), for ten
// thousand values of the busiest CU (threads without a value count; held, groups of any channels 1.6 times as much, of less than
// eight 2.5), for each round of workgroups on the CUs, for a megabyte of x, and for one whose pieces of a place share cache lines.
// Fitted to 980 timings of 20 shapes (1 x 16 x 64 to 4 x 16384 x 512, 1 to 32 groups) with every tile, number of threads and part
// that they allow, 21 % off (rms).  Of 20 others, with gelu, the choices take 4.5 % longer than the best on average, 31 % at most.
// Added after that, from one or two shapes each: what groups of less than eight channels count, and `tiny` (5 x 1389 x 126 in 42 groups
// forward 21.8 us by the choice without them, 15.7 by this one).
// 32 x 1000 x 128 bf16 forward: held by 256 workgroups 10 us, in parts 14; 1 x 4096 x 512: held by 32 workgroups 14.5, parts 13.
struct Times {
  double start, wide, values, rounds, memory, pieces;
};
constexpr Times HELD[2] = {{3.6, 0.64, 1.27, 1.65, 0.069, 0.125}, {6.7, 1.23, 3.5, 0.69, 0.245, 0.326}};
constexpr Times PARTS[2] = {{5.2, 0.82, 1.58, 4.56, 0.334, 0.038}, {0.0, 0.56, 3.5, 11.7, 0.538, 0.06}};
static Plan plan_of(int dtype, int64_t samples, int64_t places, int64_t channels, int64_t groups, bool backward) {
  Plan best{};
  const int64_t c = channels / groups, cus = device_cus();
  const int es = dense::size_of(dtype), most = backward ? 4 : 8, most_threads = backward ? 512 : 1024;  // (two arrays: more registers)
  const Times& held = HELD[backward];
  const double mb = static_cast<double>(samples) * places * channels * es * 1e-6;
  // pieces of a place of less than 128 bytes share cache lines with other workgroups'
  const auto pieces = [&](int64_t gpt) { return gpt < groups && gpt * c * es < 128 ? mb * (128.0 / (gpt * c * es) - 1) : 0.0; };
  // (of less than 32 bytes they take a cache line a lane: 48 x 238 x 30 in 10 groups backward, 12 bytes 19.7 us, 30 bytes 14.0)
  const auto tiny = [&](int64_t gpt) { return gpt < groups && gpt * c * es < 32 ? 3.0 * (32.0 / (gpt * c * es) - 1) : 0.0; };
  const auto over = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  double least = 0;
  // (of the groups a tile that make as many tiles the fewest)
  const auto next = [&](int64_t gpt) { return gpt < groups ? (groups - 1) / (over(groups, gpt) - 1) + 1 : groups + 1; };
  for (int64_t gpt = 1; gpt <= groups && gpt * c <= 8 * most_threads; gpt = next(gpt)) {
    const int64_t units = (gpt * c + 7) / 8, tiles = over(groups, gpt);
    const int wp = pow2(units);
    for (const int nt : {64, 256, most_threads}) {
      // several samples side by side where a wave or less has one's places
      int span = nt;
      if (wp < 64 && places <= 64 / wp * (c % 8 == 0 ? 1 : 4)) span = pow2(c % 8 == 0 ? places : over(places, 4)) * wp;
      const int64_t need = wp <= nt ? over(places, span / wp) : most + 1, per = nt / span;
      if (need > most || lds_of(nt, wp, span, gpt, backward ? 2 : 1) > MAX_LDS) continue;
      const int r = c % 8 == 0 || need > 4 ? pow2(need) : 4;
      const int64_t items = over(samples, per) * tiles, fit = (backward ? 8 : 16) * 64 / nt;  // workgroups that a CU holds
      const double t = held.start + held.wide * nt / 256 + held.values * (c % 8 == 0 ? 1.0 : c < 8 ? 2.5 : 1.6) * 1e-4 * (over(items, cus) * nt * r * 8) +
                       held.rounds * over(items, cus * (fit > 0 ? fit : 1)) + held.memory * mb + held.pieces * pieces(gpt) + tiny(gpt);
      if (best.threads == 0 || t < least) {
        least = t;
        const int64_t slots = 2048 / nt * cus / tiles, turns = over(samples, per);
        best = {nt, r, wp, static_cast<int>(gpt), static_cast<int>(tiles), 1, 0, 1, static_cast<int>(places),
                static_cast<int>(turns < slots ? turns : (slots < 1 ? 1 : slots)), span};
      }
    }
  }

  Plan p{};
  p.sub = 1, p.span = WIDE;
  if (c > MAX_COLS) {
    p.sub = static_cast<int>(over(c, MAX_COLS));
    p.subcols = static_cast<int>(over(over(c, p.sub), 8) * 8);
    p.sub = static_cast<int>(over(c, p.subcols));
    p.gpt = 1, p.tiles = static_cast<int>(groups * p.sub), p.wp = pow2(p.subcols / 8);
  } else {
    // as few groups as fill 256 bytes of a place, or more where those leave lanes empty
    double most_full = 0;
    for (int64_t gpt = 1; gpt <= groups && gpt * c <= MAX_COLS; gpt = next(gpt)) {
      const int64_t units = (gpt * c + 7) / 8, bytes = gpt * c * es;
      const double full = static_cast<double>(gpt * c) / (8 * pow2(units)) * (gpt == groups || bytes >= 256 ? 1.0 : bytes / 256.0) * (bytes > 512 ? 0.9 : 1.0);
      if (full > most_full) most_full = full, p.gpt = static_cast<int>(gpt), p.wp = pow2(units);
    }
    p.tiles = static_cast<int>(over(groups, p.gpt));
  }
  // two workgroups a CU, each of whose threads has whole batches
  const int64_t step = (backward ? BATCH_BWD : BATCH) * (WIDE / p.wp), want = over(2 * cus, samples * p.tiles);
  const int64_t rows = over(over(places, want), step) * step;
  p.rows = static_cast<int>(rows < places ? rows : places);
  p.parts = static_cast<int>(over(places, p.rows));
  // the backward's rows of column sums: one a part; where that would be more than a quarter of x, as many as eight workgroups a CU
  // (of 8192 channels bf16: 100000 samples of one place 15.7 ms where a row a sample took 19.2, 5000 of four 0.96 and 1.11, 2000 of
  // sixteen 0.76 and 0.74)
  const int64_t every = samples * p.parts, some = 8 * cus > p.tiles ? 8 * cus / p.tiles : 1, all = MOST_THREADS / WIDE / p.tiles;
  const int64_t most_slots = p.rows * es < 32 ? some : every < all ? every : all;
  p.slots = static_cast<int>(over(every, over(every, most_slots)));
  if (best.threads == 0) return p;
  const Times& parts = PARTS[backward];
  const int64_t items = samples * p.tiles * p.parts;
  const double t = parts.start + parts.wide * 1e-3 * p.parts * p.gpt + parts.values * 1e-4 * (over(items, cus) * over(p.rows, step) * step * p.wp * 8) +
                   parts.rounds * over(items, 8 * cus) + parts.memory * mb + parts.pieces * pieces(p.gpt);
  return t < least ? p : best;
}

static int64_t workspace(const Plan& p, int64_t samples, int64_t channels, int64_t groups, bool backward) {
  if (p.threads) return backward && p.slots > 1 ? static_cast<int64_t>(p.slots) * 2 * channels : 0;
  return samples * p.parts * groups * p.sub * 2 + (backward ? p.slots * 2 * channels : 0);
}

static int check(int dtype, int act, int64_t samples, int64_t places, int64_t channels, int64_t groups) {
  MALOQ_REQUIRE(dtype >= F32 && dtype <= F16, "unsupported dtype code %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  MALOQ_REQUIRE(act >= dense::ACT_NONE && act <= dense::ACT_GELU, "unknown activation %d", act);
  MALOQ_REQUIRE(channels >= 1 && channels < MAX_CHANNELS && groups >= 1 && channels % groups == 0, "%lld channels in %lld groups",
                (long long)channels, (long long)groups);
  MALOQ_REQUIRE(samples >= 0 && places >= 0 && samples < (int64_t(1) << 30) && places < (int64_t(1) << 30),
                "%lld samples of %lld places out of range", (long long)samples, (long long)places);
  return MALOQ_OK;
}

static GroupArgs args_of(const Plan& p, int act, int64_t samples, int64_t places, int64_t channels, int64_t groups, float eps) {
  GroupArgs a{};
  a.samples = static_cast<int>(samples), a.places = static_cast<int>(places), a.channels = static_cast<int>(channels);
  a.groups = static_cast<int>(groups), a.c = a.channels / a.groups, a.act = act, a.eps = eps;
  a.wp = p.wp, a.gpt = p.gpt, a.tiles = p.tiles, a.sub = p.sub, a.subcols = p.subcols, a.parts = p.parts, a.rows = p.rows, a.slots = p.slots, a.span = p.span;
  return a;
}
static unsigned grid_of(int64_t items) { return static_cast<unsigned>((items + 7) / 8 * 8); }
// f(a launch's arguments, whether it is the first), until all samples have had one: as many a launch as have threads, of which
// `each` have `per` samples and `others` none.
template <int TYPE, class F>
static int by_launches(const GroupArgs& a, int64_t per, int64_t each, int64_t others, const F& f) {
  const int64_t most = (MOST_THREADS - others) / each * per;
  MALOQ_REQUIRE(most > 0, "%lld threads for a sample are too many", (long long)each);
  for (int64_t n0 = 0; n0 < a.samples; n0 += most) {
    GroupArgs now = a;
    const auto from = [&](const void* p, int64_t ld) { return p ? static_cast<const char*>(p) + n0 * a.places * ld * dense::size_of(TYPE) : nullptr; };
    now.x = from(a.x, a.ldx), now.g = from(a.g, a.ldg), now.out = const_cast<char*>(from(a.out, a.channels));
    if (a.stats) now.stats = a.stats + n0 * a.groups * 2;
    if (a.part) now.part = a.part + n0 * a.groups * a.parts * a.sub * 2;
    now.samples = static_cast<int>(a.samples - n0 < most ? a.samples - n0 : most);
    f(now, n0 == 0);
  }
  return MALOQ_OK;
}

template <int TYPE>
static int forward(const Plan& p, const GroupArgs& all, hipStream_t st) {
  const bool eights = all.c % 8 == 0 && all.subcols % 8 == 0;
  int rc = MALOQ_OK;
  if (p.threads) {
    const int64_t per = p.threads / p.span;
    rc = by_launches<TYPE>(all, per, static_cast<int64_t>(p.tiles) * p.threads, 0, [&](const GroupArgs& a, bool) {
      const unsigned lds = static_cast<unsigned>(lds_of(p.threads, p.wp, p.span, p.gpt, 1)), grid = grid_of((a.samples + per - 1) / per * a.tiles);
#define MALOQ_GROUP(NT, R, EIGHTS) \
  if (p.threads == NT && p.places == R && eights == EIGHTS) group_fwd_kernel<TYPE, NT, R, EIGHTS><<<grid, NT, lds, st>>>(a);
#define MALOQ_GROUP4(NT)                                                                              \
  MALOQ_GROUP(NT, 1, true) MALOQ_GROUP(NT, 2, true) MALOQ_GROUP(NT, 4, true) MALOQ_GROUP(NT, 8, true) \
  MALOQ_GROUP(NT, 4, false) MALOQ_GROUP(NT, 8, false)
      MALOQ_GROUP4(64)
      MALOQ_GROUP4(256)
      MALOQ_GROUP4(1024)
#undef MALOQ_GROUP4
#undef MALOQ_GROUP
    });
    return rc ? rc : check_launch("maloq_group_norm_fwd");
  }
  const auto launch = [&](auto is) {
    constexpr bool EIGHTS = decltype(is)::value;
    return by_launches<TYPE>(all, 1, static_cast<int64_t>(p.tiles) * p.parts * WIDE, 0, [&](const GroupArgs& a, bool) {
      const unsigned grid = grid_of(static_cast<int64_t>(a.samples) * p.tiles * p.parts);
      group_parts_kernel<TYPE, EIGHTS><<<grid, WIDE, lds_of(WIDE, p.wp, WIDE, p.gpt, 1), st>>>(a);
      group_apply_kernel<TYPE, EIGHTS><<<grid, WIDE, 8 * p.gpt, st>>>(a);
    });
  };
  rc = eights ? launch(std::true_type{}) : launch(std::false_type{});
  return rc ? rc : check_launch("maloq_group_norm_fwd");
}

template <int TYPE>
static int backward(const Plan& p, GroupArgs a, hipStream_t st) {
  const bool eights = a.c % 8 == 0 && a.subcols % 8 == 0;
  const int64_t items = static_cast<int64_t>(p.slots) * a.tiles;
  MALOQ_REQUIRE(items * (p.threads ? p.threads : WIDE) <= MOST_THREADS, "%lld tiles are too many", (long long)items);
  const unsigned grid = grid_of(items);
  if (p.threads) {
    const unsigned lds = static_cast<unsigned>(lds_of(p.threads, p.wp, p.span, p.gpt, 2));
    void* dwb = a.dwb;
    if (p.slots > 1) a.dwb = nullptr;
    if (!dwb || p.slots == 1) a.part = nullptr;
#define MALOQ_GROUP(NT, R, EIGHTS) \
  if (p.threads == NT && p.places == R && eights == EIGHTS) group_bwd_kernel<TYPE, NT, R, EIGHTS><<<grid, NT, lds, st>>>(a);
#define MALOQ_GROUP3(NT) MALOQ_GROUP(NT, 1, true) MALOQ_GROUP(NT, 2, true) MALOQ_GROUP(NT, 4, true) MALOQ_GROUP(NT, 4, false)
    MALOQ_GROUP3(64)
    MALOQ_GROUP3(256)
    MALOQ_GROUP3(512)
#undef MALOQ_GROUP3
#undef MALOQ_GROUP
    if (int rc = check_launch("maloq_group_norm_bwd")) return rc;
    return a.part ? sum_parts(TYPE, a.part, p.slots, 2 * a.channels, dwb, st) : MALOQ_OK;
  }
  const unsigned adders = a.dwb ? static_cast<unsigned>((2 * static_cast<int64_t>(a.channels) + ADD - 1) / ADD) : 0;
  float* columns = a.dwb ? a.part + static_cast<int64_t>(a.samples) * a.groups * a.parts * a.sub * 2 : nullptr;
  const auto launch = [&](auto is) -> int {
    constexpr bool EIGHTS = decltype(is)::value;
    const unsigned lds = static_cast<unsigned>(lds_of(WIDE, p.wp, WIDE, p.gpt, 2)), lds_apply = 8 * p.gpt > 1024 ? 8 * p.gpt : 1024;
    if (p.slots < static_cast<int64_t>(a.samples) * a.parts)
      group_bwd_parts_kernel<TYPE, EIGHTS, true><<<grid, WIDE, lds, st>>>(a, columns);
    else
      group_bwd_parts_kernel<TYPE, EIGHTS, false><<<grid, WIDE, lds, st>>>(a, columns);
    if (!a.out) {
      group_bwd_apply_kernel<TYPE, EIGHTS><<<adders, WIDE, lds_apply, st>>>(a, columns, adders);
      return MALOQ_OK;
    }
    return by_launches<TYPE>(a, 1, static_cast<int64_t>(p.tiles) * p.parts * WIDE, static_cast<int64_t>(adders) * WIDE, [&](const GroupArgs& now, bool first) {
      const unsigned others = first ? adders : 0;
      group_bwd_apply_kernel<TYPE, EIGHTS><<<grid_of(static_cast<int64_t>(now.samples) * p.tiles * p.parts) + others, WIDE, lds_apply, st>>>(now, columns, others);
    });
  };
  const int rc = eights ? launch(std::true_type{}) : launch(std::false_type{});
  return rc ? rc : check_launch("maloq_group_norm_bwd");
}

}  // namespace group
}  // namespace maloq

using namespace maloq;
using namespace maloq::group;

extern "C" int64_t maloq_group_norm_workspace_floats(int dtype, int64_t samples, int64_t places, int64_t channels, int64_t groups,
                                                     int backward) {
  if (check(dtype, 0, samples, places, channels, groups)) return -1;
  if (samples == 0 || places == 0) return 0;
  return workspace(plan_of(dtype, samples, places, channels, groups, backward), samples, channels, groups, backward);
}

extern "C" int maloq_group_norm_plan(int dtype, int64_t samples, int64_t places, int64_t channels, int64_t groups, int backward,
                                     int64_t* plan) {
  if (int rc = check(dtype, 0, samples, places, channels, groups)) return rc;
  MALOQ_REQUIRE(plan && samples > 0 && places > 0, "no plan without values");
  const Plan p = plan_of(dtype, samples, places, channels, groups, backward);
  plan[0] = p.threads, plan[1] = p.places, plan[2] = p.gpt, plan[3] = p.tiles, plan[4] = p.parts, plan[5] = p.sub, plan[6] = p.slots, plan[7] = p.span;
  return MALOQ_OK;
}

extern "C" int maloq_group_norm_fwd(int dtype, const void* x, int64_t ld_x, const void* weight, const void* bias, int act,
                                    int64_t samples, int64_t places, int64_t channels, int64_t groups, float eps, float* ws, void* y,
                                    float* stats, void* stream) {
  if (int rc = check(dtype, act, samples, places, channels, groups)) return rc;
  if (samples == 0 || places == 0) return MALOQ_OK;
  const Plan p = plan_of(dtype, samples, places, channels, groups, false);
  MALOQ_REQUIRE(y && (p.threads || ws), "the norm needs a place for its result and a workspace");
  GroupArgs a = args_of(p, act, samples, places, channels, groups, eps);
  a.x = x, a.ldx = ld_x, a.w = weight, a.b = bias, a.out = y, a.stats = stats, a.part = ws;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == F32 ? forward<F32>(p, a, st) : dtype == BF16 ? forward<BF16>(p, a, st) : forward<F16>(p, a, st);
}

extern "C" int maloq_group_norm_bwd(int dtype, const void* g, int64_t ld_g, const void* x, int64_t ld_x, const void* weight,
                                    const void* bias, const float* stats, int act, int64_t samples, int64_t places, int64_t channels,
                                    int64_t groups, float* ws, void* dx, void* dwb, void* stream) {
  if (int rc = check(dtype, act, samples, places, channels, groups)) return rc;
  if (samples == 0 || places == 0) return dwb ? sum_parts(dtype, nullptr, 0, static_cast<int>(2 * channels), dwb, stream) : MALOQ_OK;
  const Plan p = plan_of(dtype, samples, places, channels, groups, true);
  MALOQ_REQUIRE(stats && (ws || (p.threads && (!dwb || p.slots == 1))), "the norm's gradients need its statistics and a workspace");
  GroupArgs a = args_of(p, act, samples, places, channels, groups, 0.f);
  a.x = x, a.ldx = ld_x, a.g = g, a.ldg = ld_g, a.w = weight, a.b = bias, a.out = dx, a.stats = const_cast<float*>(stats);
  a.part = ws, a.dwb = dwb;
  if (!dx && !dwb) return MALOQ_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == F32 ? backward<F32>(p, a, st) : dtype == BF16 ? backward<BF16>(p, a, st) : backward<F16>(p, a, st);
}
