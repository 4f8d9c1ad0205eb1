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
// with its two arrays 32768), one launch reads and writes everything once; else a launch sums parts of each group, one adds
// the parts, and one reads the values again.
//
// A thread has eight consecutive channels (16 bytes of 16-bit values, at any address), `wp` threads, a power of two, the
// workgroup's columns of a place; further threads the places that follow.
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
  int wp, gpt, tiles;   // threads of a place; groups of a tile, tiles of a place
  int sub, subcols;     // tiles of a group of more columns than a tile has, and their columns (sub = 1: none)
  int parts, rows;      // parts of a sample's places, and their places
  int slots;            // workgroups of a tile, each every slots-th sample
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

// Sums over the columns of each of the tile's groups, of Q numbers for each of a thread's eight columns: over the lanes of
// a wave that have the same columns, then through LDS.  sums: [Q][groups], where the caller finds them after it returns.
// lds: [Q][rows][8 wp], rows = waves, or NT / wp where a place takes more than a wave.
template <int NT, int Q>
__device__ __forceinline__ void group_sums(float (&v)[Q][8], int wp, const Columns& t, float* lds, float* sums) {
  const int tid = threadIdx.x, u = tid & (wp - 1), rows = wp < 64 ? NT / 64 : NT / wp;
  const bool eights = t.c % 8 == 0;  // a thread's columns are of one group
  const int n = eights ? 1 : 8, c = eights ? t.c / 8 : t.c, pitch = wp * n;
  if (eights) {
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q][0] = ((v[q][0] + v[q][1]) + (v[q][2] + v[q][3])) + ((v[q][4] + v[q][5]) + (v[q][6] + v[q][7]));
  }
  for (int o = wp; o < 64; o *= 2) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      v[q][0] += __shfl_xor(v[q][0], o);
      if (!eights) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v[q][k] += __shfl_xor(v[q][k], o);
      }
    }
  }
  if (wp >= 64 || (tid & 63) < wp) {
    const int row = wp < 64 ? tid >> 6 : tid / wp;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float* p = lds + (q * rows + row) * pitch + u * n;
      p[0] = v[q][0];
      if (!eights) {
#pragma unroll
        for (int k = 1; k < 8; ++k) p[k] = v[q][k];
      }
    }
  }
  __syncthreads();
  int tpg = 64;
  while (tpg > 1 && tpg * t.groups > NT) tpg /= 2;
  const int j = tid & (tpg - 1);
  for (int g = tid / tpg; g < t.groups; g += NT / tpg) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float s = 0.f;
      for (int r = 0; r < rows; ++r)
        for (int ch = j; ch < c; ch += tpg) s += lds[(q * rows + r) * pitch + g * c + ch];
      for (int o = tpg / 2; o > 0; o /= 2) s += __shfl_xor(s, o);
      if (j == 0) sums[q * t.groups + g] = s;
    }
  }
  __syncthreads();
}
// f(column of the eight, group of the tile that it is in); past the last column the last group
template <class F>
__device__ __forceinline__ void each_column(const Columns& t, int u, const F& f) {
  int g = u * 8 / t.c, left = (g + 1) * t.c - u * 8;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (left == 0) ++g, left = t.c;
    --left;
    f(k, g < t.groups ? g : t.groups - 1);
  }
}

// Eight columns of w (or ones) and b (or zeros)
template <int TYPE>
__device__ __forceinline__ void load_affine(const GroupArgs& a, int col, int have, float (&w)[8], float (&b)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = 1.f, b[k] = 0.f;
  if (have <= 0) return;
  if (a.w) dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.w, col, have), w);
  if (a.b) dense::unpack8<TYPE>(dense::load_part8<TYPE>(a.b, col, have), b);
}
// y of eight columns
template <int TYPE, int ACT>
__device__ __forceinline__ void finish(float (&x)[8], const float (&mean)[8], const float (&scale)[8], const float (&b)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = dense::act_fwd<TYPE == F32, ACT>(fmaf(x[k] - mean[k], scale[k], b[k]));
}
// n and u of eight columns, from x and g
template <int TYPE, int ACT>
__device__ __forceinline__ void slopes(float (&x)[8], float (&g)[8], const float (&mean)[8], const float (&rstd)[8],
                                       const float (&w)[8], const float (&b)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[k] = (x[k] - mean[k]) * rstd[k];
    g[k] *= dense::act_slope<TYPE == F32, ACT>(fmaf(x[k], w[k], b[k]));
  }
}

// ------------------------------------------------- values held in registers
// A workgroup has one tile of one sample, a thread R places of eight columns.
template <int TYPE, int NT, int R>
__global__ __launch_bounds__(NT) void group_fwd_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = NT / a.wp;
  const unsigned item = dense::dealt(blockIdx.x, static_cast<unsigned>(a.samples) * a.tiles);
  if (item >= static_cast<unsigned>(a.samples) * a.tiles) return;
  const int n = item / a.tiles;
  const Columns t = columns_of(a, item - n * a.tiles);
  float* sums = lds + (a.wp < 64 ? NT / 64 : NT / a.wp) * a.wp * 8;  // [2][groups]
  const int have = t.cols - u * 8, col = t.col0 + u * 8;
  const int64_t row0 = static_cast<int64_t>(n) * a.places;

  dense::Raw8<TYPE> x[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = i * nr + rt;
    x[i] = {};
    if (have > 0 && r < a.places) x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
  }
  float v[1][8], mean[8], scale[8], b[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float e[8];
    dense::unpack8<TYPE>(x[i], e);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] += e[k];
  }
  group_sums<NT, 1>(v, a.wp, t, lds, sums);
  const float count = static_cast<float>(a.places) * a.c;
  each_column(t, u, [&](int k, int g) { mean[k] = sums[g] / count; });
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float e[8];
    dense::unpack8<TYPE>(x[i], e);
    if (i * nr + rt < a.places) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < have) v[0][k] = fmaf(e[k] - mean[k], e[k] - mean[k], v[0][k]);
    }
  }
  group_sums<NT, 1>(v, a.wp, t, lds, sums + t.groups);
  if (a.stats) {
    for (int g = tid; g < t.groups; g += NT) {
      float* s = a.stats + (static_cast<int64_t>(n) * a.groups + t.group0 + g) * 2;
      s[0] = sums[g] / count;
      s[1] = 1.f / sqrtf(sums[t.groups + g] / count + a.eps);
    }
  }
  if (have <= 0) return;
  load_affine<TYPE>(a, col, have, scale, b);
  each_column(t, u, [&](int k, int g) { scale[k] *= 1.f / sqrtf(sums[t.groups + g] / count + a.eps); });
  dense::with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = i * nr + rt;
      float e[8];
      dense::unpack8<TYPE>(x[i], e);
      finish<TYPE, decltype(act)::value>(e, mean, scale, b);
      if (r < a.places) dense::store_part8<TYPE>(a.out, (row0 + r) * a.channels + col, e, have);
    }
  });
}

// Sums over the places of a workgroup, of eight columns a thread, to part[0 .. cols) and part[channels ..).
template <int NT>
__device__ __forceinline__ void column_sums(float (&v)[2][8], int wp, int cols, float* lds, float* part, int64_t next) {
  const int tid = threadIdx.x, u = tid & (wp - 1), rows = wp < 64 ? NT / 64 : NT / wp, pitch = wp * 8;
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
      for (int k = 0; k < 8; ++k) lds[(q * rows + row) * pitch + u * 8 + k] = v[q][k];
  }
  __syncthreads();
  for (int i = tid; i < 2 * cols; i += NT) {
    const int q = i < cols ? 0 : 1, ch = q ? i - cols : i;
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += lds[(q * rows + r) * pitch + ch];
    part[q * next + ch] = s;
  }
}

// .. and every slots-th sample; dw and db are summed over them.
template <int TYPE, int NT, int R>
__global__ __launch_bounds__(NT) void group_bwd_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = NT / a.wp;
  const unsigned item = dense::dealt(blockIdx.x, static_cast<unsigned>(a.slots) * a.tiles);
  if (item >= static_cast<unsigned>(a.slots) * a.tiles) return;
  const int slot = item / a.tiles;
  const Columns t = columns_of(a, item - slot * a.tiles);
  float* sums = lds + 2 * (a.wp < 64 ? NT / 64 : NT / a.wp) * a.wp * 8;  // [2][groups]
  const int have = t.cols - u * 8, col = t.col0 + u * 8;
  const float count = static_cast<float>(a.places) * a.c;
  float w[8], b[8], total[2][8];
  load_affine<TYPE>(a, col, have, w, b);
#pragma unroll
  for (int k = 0; k < 8; ++k) total[0][k] = total[1][k] = 0.f;
  for (int n = slot; n < a.samples; n += a.slots) {
    const int64_t row0 = static_cast<int64_t>(n) * a.places;
    dense::Raw8<TYPE> x[R], g[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = i * nr + rt;
      x[i] = g[i] = {};
      if (have > 0 && r < a.places) {
        x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
        g[i] = dense::load_part8<TYPE>(a.g, (row0 + r) * a.ldg + col, have);
      }
    }
    float mean[8], rstd[8], uu[R][8], v[2][8];
    const float* stats = a.stats + (static_cast<int64_t>(n) * a.groups + t.group0) * 2;
    each_column(t, u, [&](int k, int gr) { mean[k] = stats[2 * gr], rstd[k] = stats[2 * gr + 1]; });
#pragma unroll
    for (int k = 0; k < 8; ++k) v[0][k] = v[1][k] = 0.f;
    dense::with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
        dense::unpack8<TYPE>(g[i], uu[i]);
        slopes<TYPE, decltype(act)::value>(e, uu[i], mean, rstd, w, b);
        const bool here = i * nr + rt < a.places;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (!here || k >= have) continue;
          v[0][k] += uu[i][k];
          v[1][k] = fmaf(uu[i][k], e[k], v[1][k]);
        }
      }
    });
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 8; ++k) total[q][k] += v[q][k], v[q][k] *= w[k];
    if (!a.out) continue;
    group_sums<NT, 2>(v, a.wp, t, lds, sums);
    float m0[8], m1[8];
    each_column(t, u, [&](int k, int gr) { m0[k] = sums[gr] / count, m1[k] = sums[t.groups + gr] / count; });
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = i * nr + rt;
      if (have <= 0 || r >= a.places) continue;
      float e[8];
      dense::unpack8<TYPE>(x[i], e);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = rstd[k] * (fmaf(uu[i][k], w[k], -m0[k]) - (e[k] - mean[k]) * rstd[k] * m1[k]);
      dense::store_part8<TYPE>(a.out, (row0 + r) * a.channels + col, e, have);
    }
  }
  if (!a.part) return;
  __syncthreads();  // (the last sample's sums have been read)
  // dw's sums (u n), then db's
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float s = total[0][k];
    total[0][k] = total[1][k], total[1][k] = s;
  }
  column_sums<NT>(total, a.wp, t.cols, lds, a.part + static_cast<int64_t>(slot) * 2 * a.channels + t.col0, a.channels);
}

// ------------------------------------------------------------ several launches
constexpr int WIDE = 256;      // threads
constexpr int BATCH = 8;       // places of a thread at a time
constexpr int MAX_COLS = 512;  // of a tile

// The places of a part
__device__ __forceinline__ int places_of(const GroupArgs& a, int part) {
  const int left = a.places - part * a.rows;
  return left < a.rows ? left : a.rows;
}
// blockIdx -> tile, part, sample; tiles of the same places next to each other
struct Where {
  int tile, part, n;
};
__device__ __forceinline__ bool where(const GroupArgs& a, Where& w) {
  const unsigned all = static_cast<unsigned>(a.samples) * a.parts * a.tiles, item = dense::dealt(blockIdx.x, all);
  if (item >= all) return false;
  const unsigned sp = item / a.tiles;
  w = {static_cast<int>(item - sp * a.tiles), static_cast<int>(sp % a.parts), static_cast<int>(sp / a.parts)};
  return true;
}

// Mean and sum of squared differences from it, of each of the tile's groups in a part: part[(n groups + g) parts sub + ..][2].
template <int TYPE>
__global__ __launch_bounds__(WIDE) void group_parts_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  Where at;
  if (!where(a, at)) return;
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  float* sums = lds + (a.wp < 64 ? WIDE / 64 : WIDE / a.wp) * a.wp * 8;
  const int have = t.cols - u * 8, col = t.col0 + u * 8, places = places_of(a, at.part);
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  float mean[8], m2[8], n = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) mean[k] = m2[k] = 0.f;
  if (have > 0) {
    for (int r0 = rt; r0 < places; r0 += BATCH * nr) {
      dense::Raw8<TYPE> x[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = r0 + i * nr;
        x[i] = {};
        if (r < places) x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
      }
      const int some = (places - r0 + nr - 1) / nr, m = some < BATCH ? some : BATCH;
      float s[8], d[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] = d[k] = 0.f;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += e[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] /= m;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
        if (i < m) {
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] = fmaf(e[k] - s[k], e[k] - s[k], d[k]);
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
  }
  float v[1][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = k < have ? n * mean[k] : 0.f;
  group_sums<WIDE, 1>(v, a.wp, t, lds, sums);
  const float count = static_cast<float>(places) * t.c;
  each_column(t, u, [&](int k, int g) {
    const float apart = mean[k] - sums[g] / count;
    v[0][k] = k < have ? fmaf(apart * apart, n, m2[k]) : 0.f;
  });
  group_sums<WIDE, 1>(v, a.wp, t, lds, sums + t.groups);
  for (int g = tid; g < t.groups; g += WIDE) {
    const int64_t of = (static_cast<int64_t>(at.n) * a.groups + t.group0 + g) * a.parts * a.sub;
    float* p = a.part + (of + static_cast<int64_t>(at.part) * a.sub + (a.sub > 1 ? at.tile % a.sub : 0)) * 2;
    p[0] = sums[g] / count;
    p[1] = sums[t.groups + g];
  }
}
// The parts of a group, a wave each: mean and rstd.
__global__ __launch_bounds__(64) void group_merge_kernel(GroupArgs a) {
  const int lane = threadIdx.x, all = a.parts * a.sub;
  const float* p = a.part + static_cast<int64_t>(blockIdx.x) * all * 2;
  auto count = [&](int i) {
    const int of = i % a.sub, cols = a.sub > 1 ? (a.c - of * a.subcols < a.subcols ? a.c - of * a.subcols : a.subcols) : a.c;
    return static_cast<float>(places_of(a, i / a.sub)) * cols;
  };
  const float n = static_cast<float>(a.places) * a.c;
  float s = 0.f, m2 = 0.f;
  const float first = p[0];  // (differences from it: parts of one mean have that mean)
  for (int i = lane; i < all; i += 64) s = fmaf(p[2 * i] - first, count(i) / n, s);
  for (int o = 32; o > 0; o /= 2) s += __shfl_xor(s, o);
  s += first;
  for (int i = lane; i < all; i += 64) {
    const float apart = p[2 * i] - s;
    m2 += fmaf(apart * apart, count(i), p[2 * i + 1]);
  }
  for (int o = 32; o > 0; o /= 2) m2 += __shfl_xor(m2, o);
  if (lane == 0) {
    a.stats[2 * static_cast<int64_t>(blockIdx.x)] = s;
    a.stats[2 * static_cast<int64_t>(blockIdx.x) + 1] = 1.f / sqrtf(m2 / n + a.eps);
  }
}
template <int TYPE>
__global__ __launch_bounds__(WIDE) void group_apply_kernel(GroupArgs a) {
  Where at;
  if (!where(a, at)) return;
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const int have = t.cols - u * 8, col = t.col0 + u * 8, places = places_of(a, at.part);
  if (have <= 0) return;
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  float mean[8], scale[8], b[8];
  load_affine<TYPE>(a, col, have, scale, b);
  const float* stats = a.stats + (static_cast<int64_t>(at.n) * a.groups + t.group0) * 2;
  each_column(t, u, [&](int k, int g) { mean[k] = stats[2 * g], scale[k] *= stats[2 * g + 1]; });
  for (int r0 = rt; r0 < places; r0 += BATCH * nr) {
    dense::Raw8<TYPE> x[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = r0 + i * nr;
      if (r < places) x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
    }
    dense::with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = r0 + i * nr;
        if (r >= places) break;
        float e[8];
        dense::unpack8<TYPE>(x[i], e);
        finish<TYPE, decltype(act)::value>(e, mean, scale, b);
        dense::store_part8<TYPE>(a.out, (row0 + r) * a.channels + col, e, have);
      }
    });
  }
}

// Sums of u n and u over a part's places, a column each: part[n][parts][2][channels].
constexpr int BATCH_BWD = 4;
template <int TYPE>
__global__ __launch_bounds__(WIDE) void group_bwd_parts_kernel(GroupArgs a) {
  extern __shared__ float lds[];
  Where at;
  if (!where(a, at)) return;
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const int have = t.cols - u * 8, col = t.col0 + u * 8, places = places_of(a, at.part);
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  float mean[8], rstd[8], w[8], b[8], v[2][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[0][k] = v[1][k] = 0.f;
  load_affine<TYPE>(a, col, have, w, b);
  const float* stats = a.stats + (static_cast<int64_t>(at.n) * a.groups + t.group0) * 2;
  each_column(t, u, [&](int k, int g) { mean[k] = stats[2 * g], rstd[k] = stats[2 * g + 1]; });
  if (have > 0) {
    for (int r0 = rt; r0 < places; r0 += BATCH_BWD * nr) {
      dense::Raw8<TYPE> x[BATCH_BWD], g[BATCH_BWD];
#pragma unroll
      for (int i = 0; i < BATCH_BWD; ++i) {
        const int r = r0 + i * nr;
        x[i] = g[i] = {};
        if (r < places) {
          x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
          g[i] = dense::load_part8<TYPE>(a.g, (row0 + r) * a.ldg + col, have);
        }
      }
      dense::with_act(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < BATCH_BWD; ++i) {
          float e[8], uu[8];
          dense::unpack8<TYPE>(x[i], e);
          dense::unpack8<TYPE>(g[i], uu);
          slopes<TYPE, decltype(act)::value>(e, uu, mean, rstd, w, b);
          if (r0 + i * nr < places) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              v[0][k] = fmaf(uu[k], e[k], v[0][k]);
              v[1][k] += uu[k];
            }
          }
        }
      });
    }
  }
  column_sums<WIDE>(v, a.wp, t.cols, lds, a.part + (static_cast<int64_t>(at.n) * a.parts + at.part) * 2 * a.channels + t.col0, a.channels);
}
// Of a sample's group: the columns' sums over the parts, to columns[n][2][channels], and the group's means of u w and u w n, to
// means[n][groups][2].  Threads: up to 256 columns, the rest parts.
__global__ __launch_bounds__(WIDE) void group_bwd_merge_kernel(GroupArgs a, int type, float* columns, float* means) {
  __shared__ float lds[2][WIDE];
  const int tid = threadIdx.x, n = blockIdx.x / a.groups, g = blockIdx.x - n * a.groups;
  int cp = 1;
  while (cp < a.c && cp < WIDE) cp *= 2;
  const int j = tid & (cp - 1), pl = tid / cp, np = WIDE / cp;
  float m0 = 0.f, m1 = 0.f;
  for (int c0 = 0; c0 < a.c; c0 += cp) {
    const int col = g * a.c + c0 + j;
    const bool here = c0 + j < a.c;
    float s[2] = {0.f, 0.f};
    if (here) {
      for (int p = pl; p < a.parts; p += np) {
        const float* at = a.part + (static_cast<int64_t>(n) * a.parts + p) * 2 * a.channels + col;
        s[0] += at[0];
        s[1] += at[a.channels];
      }
    }
    lds[0][tid] = s[0], lds[1][tid] = s[1];
    __syncthreads();
    if (pl == 0 && here) {
      for (int p = 1; p < np; ++p) s[0] += lds[0][p * cp + j], s[1] += lds[1][p * cp + j];
      float* to = columns + static_cast<int64_t>(n) * 2 * a.channels + col;
      to[0] = s[0], to[a.channels] = s[1];
      const float w = !a.w ? 1.f : type == F32 ? dense::load1<F32>(a.w, col) : type == BF16 ? dense::load1<BF16>(a.w, col) : dense::load1<F16>(a.w, col);
      m0 = fmaf(w, s[1], m0), m1 = fmaf(w, s[0], m1);
    }
    __syncthreads();
  }
  lds[0][tid] = m0, lds[1][tid] = m1;
  __syncthreads();
  for (int o = WIDE / 2; o > 0; o /= 2) {
    if (tid < o) lds[0][tid] += lds[0][tid + o], lds[1][tid] += lds[1][tid + o];
    __syncthreads();
  }
  const float count = static_cast<float>(a.places) * a.c;
  if (tid < 2) means[static_cast<int64_t>(blockIdx.x) * 2 + tid] = lds[tid][0] / count;
}
template <int TYPE>
__global__ __launch_bounds__(WIDE) void group_bwd_apply_kernel(GroupArgs a, const float* means) {
  Where at;
  if (!where(a, at)) return;
  const int tid = threadIdx.x, u = tid & (a.wp - 1), rt = tid / a.wp, nr = WIDE / a.wp;
  const Columns t = columns_of(a, at.tile);
  const int have = t.cols - u * 8, col = t.col0 + u * 8, places = places_of(a, at.part);
  if (have <= 0) return;
  const int64_t row0 = static_cast<int64_t>(at.n) * a.places + static_cast<int64_t>(at.part) * a.rows;
  const int64_t group0 = (static_cast<int64_t>(at.n) * a.groups + t.group0) * 2;
  float mean[8], rstd[8], w[8], b[8], m0[8], m1[8];
  load_affine<TYPE>(a, col, have, w, b);
  each_column(t, u, [&](int k, int g) {
    mean[k] = a.stats[group0 + 2 * g], rstd[k] = a.stats[group0 + 2 * g + 1];
    m0[k] = means[group0 + 2 * g], m1[k] = means[group0 + 2 * g + 1];
  });
  for (int r0 = rt; r0 < places; r0 += BATCH_BWD * nr) {
    dense::Raw8<TYPE> x[BATCH_BWD], g[BATCH_BWD];
#pragma unroll
    for (int i = 0; i < BATCH_BWD; ++i) {
      const int r = r0 + i * nr;
      if (r < places) {
        x[i] = dense::load_part8<TYPE>(a.x, (row0 + r) * a.ldx + col, have);
        g[i] = dense::load_part8<TYPE>(a.g, (row0 + r) * a.ldg + col, have);
      }
    }
    dense::with_act(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < BATCH_BWD; ++i) {
        const int r = r0 + i * nr;
        if (r >= places) break;
        float e[8], uu[8];
        dense::unpack8<TYPE>(x[i], e);
        dense::unpack8<TYPE>(g[i], uu);
        slopes<TYPE, decltype(act)::value>(e, uu, mean, rstd, w, b);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = rstd[k] * (fmaf(uu[k], w[k], -m0[k]) - e[k] * m1[k]);
        dense::store_part8<TYPE>(a.out, (row0 + r) * a.channels + col, e, have);
      }
    });
  }
}

// ------------------------------------------------------------------- host
constexpr int64_t MAX_CHANNELS = int64_t(1) << 24;

static int pow2(int64_t v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}

// Threads of a workgroup and places of a thread (threads 0: several launches), and the tiles.
struct Plan {
  int threads, places, wp, gpt, tiles, sub, subcols, parts, rows, slots;
};
// Held in registers where it fits: of the possible groups a workgroup and threads, what wastes the least: lanes without a
// value, pieces of a place of less than 128 bytes (whose cache lines several workgroups fetch), CUs without a workgroup.
static Plan plan_of(int dtype, int64_t samples, int64_t places, int64_t channels, int64_t groups, bool backward) {
  Plan best{};
  const int64_t c = channels / groups, cus = device_cus();
  const int es = dense::size_of(dtype), most_threads = backward ? 512 : 1024;  // (the backward's two arrays: 128 registers are too few)
  double least = 0;
  for (int64_t gpt = 1; gpt <= groups; ++gpt) {
    const int64_t units = (gpt * c + 7) / 8, tiles = (groups + gpt - 1) / gpt;
    if (units > most_threads) break;
    if ((groups + tiles - 1) / tiles != gpt) continue;  // (the same tiles from fewer groups each)
    const int wp = pow2(units);
    for (const int nt : {64, 256, most_threads}) {
      if (wp > nt) continue;
      const int64_t nr = nt / wp, need = (places + nr - 1) / nr;
      if (need > 8) continue;
      const int r = pow2(need);
      const double lanes = static_cast<double>(nt) * r * 8 / (static_cast<double>(places) * gpt * c);
      const double piece = tiles > 1 && gpt * c * es < 128 ? 128.0 / (gpt * c * es) : 1.0;
      const double items = static_cast<double>(samples) * tiles, busy = items * nt / 512 < cus ? cus / (items * nt / 512) : 1.0;
      const double cost = lanes * piece * busy * (1 + 0.02 * r);
      if (best.threads == 0 || cost < least) {
        least = cost;
        best = {nt, r, wp, static_cast<int>(gpt), static_cast<int>(tiles), 1, 0, 1, static_cast<int>(places), 1};
      }
    }
  }
  if (best.threads) {
    const int64_t fit = 2048 / best.threads * cus / best.tiles;  // workgroups that the chip holds, a tile
    best.slots = static_cast<int>(samples < fit ? samples : (fit < 1 ? 1 : fit));
    return best;
  }
  Plan p{};
  p.sub = 1;
  if (c > MAX_COLS) {
    p.sub = static_cast<int>((c + MAX_COLS - 1) / MAX_COLS);
    p.subcols = static_cast<int>(((c + p.sub - 1) / p.sub + 7) / 8 * 8);
    p.sub = static_cast<int>((c + p.subcols - 1) / p.subcols);
    p.gpt = 1, p.tiles = static_cast<int>(groups * p.sub), p.wp = pow2(p.subcols / 8);
  } else {
    // as many groups as fill a tile's threads
    double most_full = 0;
    for (int64_t gpt = 1; gpt <= groups && gpt * c <= MAX_COLS; ++gpt) {
      const int64_t units = (gpt * c + 7) / 8;
      const double full = static_cast<double>(gpt * c) / (8 * pow2(units)) * (gpt * c * es < 128 && gpt < groups ? gpt * c * es / 128.0 : 1.0);
      if (full >= most_full) most_full = full, p.gpt = static_cast<int>(gpt), p.wp = pow2(units);
    }
    p.tiles = static_cast<int>((groups + p.gpt - 1) / p.gpt);
  }
  // eight workgroups a CU, each of whose threads has whole batches
  const int64_t step = BATCH * (WIDE / p.wp), want = (8 * cus + samples * p.tiles - 1) / (samples * p.tiles);
  int64_t rows = (places + want - 1) / want;
  rows = (rows + step - 1) / step * step;
  p.rows = static_cast<int>(rows < places ? rows : places);
  p.parts = static_cast<int>((places + p.rows - 1) / p.rows);
  return p;
}

static int64_t workspace(const Plan& p, int64_t samples, int64_t channels, int64_t groups, bool backward) {
  if (p.threads) return backward ? static_cast<int64_t>(p.slots) * 2 * channels : 0;
  if (!backward) return samples * groups * p.parts * p.sub * 2;
  return samples * p.parts * 2 * channels + samples * 2 * channels + samples * groups * 2;
}

static int check(int dtype, int act, int64_t samples, int64_t places, int64_t channels, int64_t groups) {
  MALOQ_REQUIRE(dtype >= F32 && dtype <= F16, "unsupported dtype code %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  MALOQ_REQUIRE(act >= dense::ACT_NONE && act <= dense::ACT_GELU, "unknown activation %d", act);
  MALOQ_REQUIRE(channels >= 1 && channels < MAX_CHANNELS && groups >= 1 && channels % groups == 0, "%lld channels in %lld groups",
                (long long)channels, (long long)groups);
  MALOQ_REQUIRE(samples >= 0 && places >= 0 && samples < (int64_t(1) << 22) && places < (int64_t(1) << 30),
                "%lld samples of %lld places out of range", (long long)samples, (long long)places);
  return MALOQ_OK;
}

static GroupArgs args_of(const Plan& p, int act, int64_t samples, int64_t places, int64_t channels, int64_t groups, float eps) {
  GroupArgs a{};
  a.samples = static_cast<int>(samples), a.places = static_cast<int>(places), a.channels = static_cast<int>(channels);
  a.groups = static_cast<int>(groups), a.c = a.channels / a.groups, a.act = act, a.eps = eps;
  a.wp = p.wp, a.gpt = p.gpt, a.tiles = p.tiles, a.sub = p.sub, a.subcols = p.subcols, a.parts = p.parts, a.rows = p.rows, a.slots = p.slots;
  return a;
}
// LDS of a workgroup of nt threads: Q numbers of each column that a wave (a place) has, and 2 of each group
static unsigned lds_of(const Plan& p, int nt, int q) {
  const int rows = p.wp < 64 ? nt / 64 : nt / p.wp;
  return 4 * (q * rows * p.wp * 8 + 2 * p.gpt);
}
static unsigned grid_of(int64_t items) { return static_cast<unsigned>((items + 7) / 8 * 8); }

template <int TYPE>
static int forward(const Plan& p, const GroupArgs& a, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(a.samples) * a.tiles;
  if (p.threads) {
    MALOQ_REQUIRE(items * p.threads < MAX_THREADS - 8 * 1024, "%lld tiles are too many", (long long)items);
    const unsigned lds = lds_of(p, p.threads, 1), grid = grid_of(items);
#define MALOQ_GROUP(NT, R) \
  if (p.threads == NT && p.places == R) group_fwd_kernel<TYPE, NT, R><<<grid, NT, lds, st>>>(a);
#define MALOQ_GROUP4(NT) MALOQ_GROUP(NT, 1) MALOQ_GROUP(NT, 2) MALOQ_GROUP(NT, 4) MALOQ_GROUP(NT, 8)
    MALOQ_GROUP4(64)
    MALOQ_GROUP4(256)
    MALOQ_GROUP4(1024)
#undef MALOQ_GROUP4
#undef MALOQ_GROUP
    return check_launch("maloq_group_norm_fwd");
  }
  MALOQ_REQUIRE(items * a.parts * WIDE < MAX_THREADS - 8 * WIDE, "%lld tiles are too many", (long long)(items * a.parts));
  const unsigned grid = grid_of(items * a.parts);
  group_parts_kernel<TYPE><<<grid, WIDE, lds_of(p, WIDE, 1), st>>>(a);
  group_merge_kernel<<<static_cast<unsigned>(a.samples) * a.groups, 64, 0, st>>>(a);
  group_apply_kernel<TYPE><<<grid, WIDE, 0, st>>>(a);
  return check_launch("maloq_group_norm_fwd");
}

template <int TYPE>
static int backward(const Plan& p, const GroupArgs& a, void* dwb, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.threads ? p.slots : a.samples) * a.tiles;
  if (p.threads) {
    MALOQ_REQUIRE(items * p.threads < MAX_THREADS - 8 * 1024, "%lld tiles are too many", (long long)items);
    const unsigned lds = lds_of(p, p.threads, 2), grid = grid_of(items);
#define MALOQ_GROUP(NT, R) \
  if (p.threads == NT && p.places == R) group_bwd_kernel<TYPE, NT, R><<<grid, NT, lds, st>>>(a);
#define MALOQ_GROUP4(NT) MALOQ_GROUP(NT, 1) MALOQ_GROUP(NT, 2) MALOQ_GROUP(NT, 4) MALOQ_GROUP(NT, 8)
    MALOQ_GROUP4(64)
    MALOQ_GROUP4(256)
    MALOQ_GROUP4(512)
#undef MALOQ_GROUP4
#undef MALOQ_GROUP
    if (int rc = check_launch("maloq_group_norm_bwd")) return rc;
    return dwb ? sum_parts(TYPE, a.part, p.slots, 2 * a.channels, dwb, st) : MALOQ_OK;
  }
  MALOQ_REQUIRE(items * a.parts * WIDE < MAX_THREADS - 8 * WIDE, "%lld tiles are too many", (long long)(items * a.parts));
  const unsigned grid = grid_of(items * a.parts);
  float* columns = a.part + static_cast<int64_t>(a.samples) * a.parts * 2 * a.channels;
  float* means = columns + static_cast<int64_t>(a.samples) * 2 * a.channels;
  group_bwd_parts_kernel<TYPE><<<grid, WIDE, lds_of(p, WIDE, 2), st>>>(a);
  group_bwd_merge_kernel<<<static_cast<unsigned>(a.samples) * a.groups, WIDE, 0, st>>>(a, TYPE, columns, means);
  if (a.out) group_bwd_apply_kernel<TYPE><<<grid, WIDE, 0, st>>>(a, means);
  if (int rc = check_launch("maloq_group_norm_bwd")) return rc;
  return dwb ? sum_parts(TYPE, columns, a.samples, 2 * a.channels, dwb, st) : MALOQ_OK;
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
  plan[0] = p.threads, plan[1] = p.places, plan[2] = p.gpt, plan[3] = p.tiles, plan[4] = p.parts, plan[5] = p.sub, plan[6] = p.slots;
  return MALOQ_OK;
}

extern "C" int maloq_group_norm_fwd(int dtype, const void* x, int64_t ld_x, const void* weight, const void* bias, int act,
                                    int64_t samples, int64_t places, int64_t channels, int64_t groups, float eps, float* ws, void* y,
                                    float* stats, void* stream) {
  if (int rc = check(dtype, act, samples, places, channels, groups)) return rc;
  if (samples == 0 || places == 0) return MALOQ_OK;
  const Plan p = plan_of(dtype, samples, places, channels, groups, false);
  MALOQ_REQUIRE(y && (p.threads || (ws && stats)), "the norm needs a place for its result, a workspace and its statistics");
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
  MALOQ_REQUIRE(stats && (ws || (p.threads && !dwb)), "the norm's gradients need its statistics and a workspace");
  GroupArgs a = args_of(p, act, samples, places, channels, groups, 0.f);
  a.x = x, a.ldx = ld_x, a.g = g, a.ldg = ld_g, a.w = weight, a.b = bias, a.out = dx, a.stats = const_cast<float*>(stats);
  a.part = p.threads && !dwb ? nullptr : ws;
  if (!dx && !dwb) return MALOQ_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == F32 ? backward<F32>(p, a, dwb, st) : dtype == BF16 ? backward<BF16>(p, a, dwb, st) : backward<F16>(p, a, dwb, st);
}
